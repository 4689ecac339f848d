"""Host-side wrappers of the C ABI (include/acmil_hip.h) on torch CUDA tensors.

PyTorch is plumbing here: it owns device memory (caching allocator) and the stream; every numerical
step of the aggregation path runs in libacmil_hip.so.  Nothing in this file computes on the CPU and
there is no fallback: CPU tensors are rejected.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib

_DT = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
GA_DA = 128
MAX_BATCH = 64       # ACMIL_MAX_BATCH: bags per acmil_ga_forward_batch / _guarded launch
MAX_GROUP = 16       # GA_SEG_MAX: bags of one row-concatenated group (acmil_ga_train_step_group, acmil_ga_pool_group)


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _need_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("acmil_amd: the aggregation path runs only on an MI355X (got a %s tensor); "
                               "there is no CPU fallback" % t.device)


def mode_id(mode) -> int:
    if isinstance(mode, int):
        return mode
    return _lib.MODES[mode]


class GaDims:
    """Shape bundle of one gated-attention aggregator."""

    def __init__(self, D: int, Di: int, K: int, C: int, has_bag_head: bool = True, mode: int = 1):
        self.D, self.Di, self.K, self.C, self.has_bag_head = D, Di, K, C, bool(has_bag_head)
        self.mode = int(mode)      # arithmetic mode the weights were packed for (ACMIL_MODE_*); the backward follows it

    def args(self):
        return (self.D, self.Di, GA_DA, self.K, self.C)


def ga_pack_weights(W1, Wv, bv, Wu, bu, Ww, bw, Wc: Sequence[torch.Tensor], bc: Sequence[torch.Tensor],
                    Ws: Optional[torch.Tensor], bs: Optional[torch.Tensor], mode) -> Tuple[torch.Tensor, GaDims]:
    """acmil_ga_pack_weights: parameters (fp32, CUDA, contiguous) -> packed fragment stream (uint8 tensor)."""
    lib = _lib.load()
    mode = mode_id(mode)
    ts = [W1, Wv, bv, Wu, bu, Ww, bw] + list(Wc) + list(bc) + [t for t in (Ws, bs) if t is not None]
    _need_cuda(*ts)
    ts = [t.detach() for t in ts]
    for t in ts:
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError("acmil_amd: parameters must be contiguous fp32")
    Di, D = W1.shape
    K, C = Ww.shape[0], Wc[0].shape[0]
    if Wv.shape != (GA_DA, Di) or Wu.shape != (GA_DA, Di) or Ww.shape[1] != GA_DA or len(Wc) != K:
        raise RuntimeError("acmil_amd: unexpected parameter shapes")
    dims = GaDims(D, Di, K, C, has_bag_head=Ws is not None, mode=mode)
    nbytes = lib.acmil_ga_packed_bytes(*dims.args(), mode)
    if nbytes == 0:
        raise RuntimeError("acmil_amd: unsupported dimensions D=%d Di=%d K=%d C=%d" % (D, Di, K, C))
    packed = torch.empty(nbytes, dtype=torch.uint8, device=W1.device)
    wc_arr = (ctypes.c_void_p * K)(*[t.data_ptr() for t in Wc])
    bc_arr = (ctypes.c_void_p * K)(*[t.data_ptr() for t in bc])
    rc = lib.acmil_ga_pack_weights(W1.data_ptr(), Wv.data_ptr(), bv.data_ptr(), Wu.data_ptr(), bu.data_ptr(),
                                   Ww.data_ptr(), bw.data_ptr(), wc_arr, bc_arr, _ptr(Ws), _ptr(bs),
                                   *dims.args(), mode, packed.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_pack_weights")
    return packed, dims


_WS_CACHE: Dict[tuple, torch.Tensor] = {}


def _ws_bytes(nbytes: int, device) -> torch.Tensor:
    """Grow-only GA workspace per (device, stream).  The library's contract (csrc/ga_common.h): the first 256 bytes are a
    control block that is zero when the workspace is first used and that every launch leaves zero again (apart from the
    range status word of the most recent launch), so the buffer is zero-filled once here and then reused -- no memset between launches.  Calls are
    stream-ordered and a call's workspace contents are dead when it returns, so one buffer per stream is enough."""
    dev = torch.device(device)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), torch.cuda.current_stream(dev).cuda_stream)
    ws = _WS_CACHE.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _lib.check(_lib.load().acmil_ga_workspace_init(ws.data_ptr(), torch.cuda.current_stream(dev).cuda_stream), "acmil_ga_workspace_init")
        _WS_CACHE[key] = ws
    return ws


_SCRATCH_CACHE: Dict[tuple, torch.Tensor] = {}


def _repeat_scratch(nbytes: int, device) -> torch.Tensor:
    """Scratch of the device-predicated exact-fp32 repeats (ga_forward_guarded_wide, ga_rescore_fp32_cond): N * (D + D_inner + 256) * 4
    bytes that only a flagged bag ever touches.  One grow-only buffer per (device, stream) instead of an allocation per eval call (0.6 GB
    for a 100 000-patch fp16 bag at D = 1024, which the caching allocator then kept reserved per size class); calls on one
    stream are ordered, and the repeat's contents are dead when its merge + heads have run."""
    dev = torch.device(device)
    key = (dev.index if dev.index is not None else torch.cuda.current_device(), torch.cuda.current_stream(dev).cuda_stream)
    sc = _SCRATCH_CACHE.get(key)
    if sc is None or sc.numel() < nbytes:
        sc = None
        _SCRATCH_CACHE.pop(key, None)
        sc = _SCRATCH_CACHE[key] = torch.empty(max(int(nbytes * 1.25), 1 << 20), dtype=torch.uint8, device=dev)
    return sc


def _workspace(N: int, dims: GaDims, mode: int, device) -> torch.Tensor:
    return _ws_bytes(_lib.load().acmil_ga_workspace_bytes(N, dims.D, dims.Di, dims.K, dims.C, mode), device)


_BATCH_WS_NEED: Dict[tuple, int] = {}


def _batch_ws_need(lib, B: int, ns: Sequence[int], Ns, dims: "GaDims", mode: int) -> int:
    """acmil_ga_batch_workspace_bytes, remembered per (bag sizes, shape, mode): the per-slide eval loop asks the same question every call."""
    key = (tuple(ns), dims.D, dims.Di, dims.K, dims.C, mode)
    need = _BATCH_WS_NEED.get(key)
    if need is None:
        if len(_BATCH_WS_NEED) > 4096:
            _BATCH_WS_NEED.clear()
        need = _BATCH_WS_NEED[key] = lib.acmil_ga_batch_workspace_bytes(B, Ns, dims.D, dims.Di, dims.K, dims.C, mode)
    return need


def _range_status(ws: torch.Tensor) -> torch.Tensor:
    """Device view of the split-f16 range status word of a GA workspace (control block, word 1).  Non-zero = a projected
    feature left the f16 range or was not finite (which is also what a bag value outside the range causes: its hi half
    converts to inf): the f16x3 result is then not the fp32 result.  The word holds the result of the MOST RECENT split-f16 launch
    on this workspace (the last workgroup of a launch overwrites it; csrc/ga_common.h), so it must be read -- or copied with
    `status.clone()` -- before the next launch on the same stream's workspace.  Reading it (`int(...)`) synchronises; the
    modules do that (lagged, see architecture/transformer.py), the raw ops do not."""
    v = ws.__dict__.get("_acmil_status")      # one view per workspace tensor (slicing + view cost ~4 us of host time per call)
    if v is None:
        v = ws.__dict__["_acmil_status"] = ws[4:8].view(torch.int32)
    return v


def _check_x(x: torch.Tensor, dims: GaDims) -> None:
    _need_cuda(x)
    if x.dim() != 2 or x.shape[1] != dims.D or x.shape[0] < 1:
        raise RuntimeError("acmil_amd: bag must be [N>=1, %d], got %s" % (dims.D, tuple(x.shape)))
    if x.dtype not in _DT or not x.is_contiguous():
        raise RuntimeError("acmil_amd: bag must be contiguous fp32/fp16/bf16")


def ga_forward(x: torch.Tensor, packed: torch.Tensor, dims: GaDims, mode, want_scores: bool = True,
               want_preds: bool = True, want_afeat: bool = False, want_bag_feat: bool = False) -> Dict[str, torch.Tensor]:
    """acmil_ga_forward, fused eval path.  x [N,D] -> dict(A_out [K,N], sub_preds [K,C], slide_pred [C], ...)."""
    lib = _lib.load()
    mode = mode_id(mode)
    _check_x(x, dims)
    N, dev = x.shape[0], x.device
    f32 = dict(dtype=torch.float32, device=dev)
    out: Dict[str, torch.Tensor] = {}
    A = torch.empty(dims.K, N, **f32) if want_scores else None
    sub = torch.empty(dims.K, dims.C, **f32) if want_preds else None
    slide = torch.empty(dims.C, **f32) if (want_preds and dims.has_bag_head) else None
    af = torch.empty(dims.K, dims.Di, **f32) if want_afeat else None
    bf = torch.empty(dims.Di, **f32) if want_bag_feat else None
    ws = _workspace(N, dims, mode, dev)
    rc = lib.acmil_ga_forward(x.data_ptr(), _DT[x.dtype], N, packed.data_ptr(), *dims.args(), mode, _ptr(A), _ptr(sub),
                              _ptr(slide), _ptr(af), _ptr(bf), None, int(dims.has_bag_head), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_forward")
    for k, v in (("A_out", A), ("sub_preds", sub), ("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    out["range_status"] = _range_status(ws)
    return out


def ga_forward_batch(xs: Sequence[torch.Tensor], packed: torch.Tensor, dims: GaDims, mode, want_scores: bool = True,
                     want_afeat: bool = False, want_bag_feat: bool = False) -> Dict[str, object]:
    """acmil_ga_forward_batch: up to 64 bags (ACMIL_MAX_BATCH) [N_b, D] (same dtype) in one fused launch.
    Returns dict(A_out=list of [K,N_b], sub_preds [B,K,C], slide_pred [B,C], ...)."""
    lib = _lib.load()
    mode = mode_id(mode)
    B = len(xs)
    for x in xs:
        _check_x(x, dims)
        if x.dtype != xs[0].dtype:
            raise RuntimeError("acmil_amd: all bags of a batch must share one dtype")
    dev = xs[0].device
    f32 = dict(dtype=torch.float32, device=dev)
    Ns = (ctypes.c_int * B)(*[x.shape[0] for x in xs])
    xp = (ctypes.c_void_p * B)(*[x.data_ptr() for x in xs])
    A = [torch.empty(dims.K, x.shape[0], **f32) for x in xs] if want_scores else None
    Ap = (ctypes.c_void_p * B)(*[t.data_ptr() for t in A]) if want_scores else None
    sub = torch.empty(B, dims.K, dims.C, **f32)
    slide = torch.empty(B, dims.C, **f32) if dims.has_bag_head else None
    af = torch.empty(B, dims.K, dims.Di, **f32) if want_afeat else None
    bf = torch.empty(B, dims.Di, **f32) if want_bag_feat else None
    ws = _ws_bytes(lib.acmil_ga_batch_workspace_bytes(B, Ns, dims.D, dims.Di, dims.K, dims.C, mode), dev)
    rc = lib.acmil_ga_forward_batch(B, xp, Ns, _DT[xs[0].dtype], packed.data_ptr(), *dims.args(), mode, Ap, sub.data_ptr(),
                                    _ptr(slide), _ptr(af), _ptr(bf), int(dims.has_bag_head), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_forward_batch")
    out: Dict[str, object] = {"sub_preds": sub, "range_status": _range_status(ws)}
    for k, v in (("A_out", A), ("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    return out


def ga_forward_guarded(xs: Sequence[torch.Tensor], packed: torch.Tensor, packed_fp32: torch.Tensor, dims: GaDims,
                       fallback_count: Optional[torch.Tensor] = None, want_scores: bool = True, want_preds: bool = True,
                       want_afeat: bool = False, want_bag_feat: bool = False) -> Dict[str, object]:
    """acmil_ga_forward_guarded: the split-f16 fused forward of up to 64 bags followed, on the device, by its exact-fp32 repeat
    if (and only if) a bag left the f16 range -- no host read-back, the outputs are the fp32-parity result either way.
    Same returns as ga_forward_batch; fallback_count: device int32 [1] the library increments when the repeat ran."""
    lib = _lib.load()
    B = len(xs)
    for x in xs:
        _check_x(x, dims)
        if x.dtype != xs[0].dtype:
            raise RuntimeError("acmil_amd: all bags of a batch must share one dtype")
    _need_cuda(packed, packed_fp32, fallback_count)
    dev = xs[0].device
    ns = [x.shape[0] for x in xs]
    Ns = (ctypes.c_int * B)(*ns)
    xp = (ctypes.c_void_p * B)(*[x.data_ptr() for x in xs])
    A = [torch.empty(dims.K, n, dtype=torch.float32, device=dev) for n in ns] if want_scores else None
    Ap = (ctypes.c_void_p * B)(*[t.data_ptr() for t in A]) if want_scores else None
    sub = slide = None
    if want_preds:      # one allocation for the logits of all bags: [B][K*C] then [B][C]
        KC, Cc = dims.K * dims.C, dims.C
        buf = torch.empty(B * (KC + (Cc if dims.has_bag_head else 0)), dtype=torch.float32, device=dev)
        sub = buf[:B * KC].view(B, dims.K, dims.C)
        slide = buf[B * KC:].view(B, Cc) if dims.has_bag_head else None
    af = torch.empty(B, dims.K, dims.Di, dtype=torch.float32, device=dev) if want_afeat else None
    bf = torch.empty(B, dims.Di, dtype=torch.float32, device=dev) if want_bag_feat else None
    ws = _ws_bytes(_batch_ws_need(lib, B, ns, Ns, dims, _lib.MODE_F16X3), dev)
    rc = lib.acmil_ga_forward_guarded(B, xp, Ns, _DT[xs[0].dtype], packed.data_ptr(), packed_fp32.data_ptr(), *dims.args(), Ap,
                                      _ptr(sub), _ptr(slide), _ptr(af), _ptr(bf), int(dims.has_bag_head), _ptr(fallback_count),
                                      ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_forward_guarded")
    out: Dict[str, object] = {"range_status": _range_status(ws)}
    for k, v in (("A_out", A), ("sub_preds", sub), ("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    return out


def ga_forward_guarded_wide(x: torch.Tensor, packed: torch.Tensor, W1: torch.Tensor, dims: GaDims,
                            fallback_count: Optional[torch.Tensor] = None, want_scores: bool = True, want_preds: bool = True,
                            want_afeat: bool = False, want_bag_feat: bool = False) -> Dict[str, torch.Tensor]:
    """acmil_ga_forward_guarded_wide: the fused split-f16 forward of ONE bag at D_inner 384 / 512 followed, on the device, by its
    exact-fp32 repeat op by op if (and only if) the bag left the f16 range -- no host read-back.  W1 = dimreduction.fc1.weight (raw
    fp32, contiguous).  Same returns as ga_forward (unbatched)."""
    lib = _lib.load()
    _check_x(x, dims)
    _need_cuda(packed, W1, fallback_count)
    if W1.dtype != torch.float32 or not W1.is_contiguous() or tuple(W1.shape) != (dims.Di, dims.D):
        raise RuntimeError("acmil_amd: W1 must be the contiguous fp32 [D_inner, D_feat] projection weight")
    N, dev = x.shape[0], x.device
    f32 = dict(dtype=torch.float32, device=dev)
    A = torch.empty(dims.K, N, **f32) if want_scores else None
    sub = torch.empty(dims.K, dims.C, **f32) if want_preds else None
    slide = torch.empty(dims.C, **f32) if (want_preds and dims.has_bag_head) else None
    af = torch.empty(dims.K, dims.Di, **f32) if want_afeat else None
    bf = torch.empty(dims.Di, **f32) if want_bag_feat else None
    nsc = lib.acmil_ga_forward_guarded_wide_scratch_bytes(N, dims.D, dims.Di, dims.K, _DT[x.dtype], 0 if want_scores else 1)
    scratch = _repeat_scratch(nsc, dev)          # only ever touched by a flagged bag: ONE grow-only buffer per (device, stream)
    ws = _workspace(N, dims, _lib.MODE_F16X3, dev)
    rc = lib.acmil_ga_forward_guarded_wide(x.data_ptr(), _DT[x.dtype], N, packed.data_ptr(), W1.data_ptr(), *dims.args(), _ptr(A), _ptr(sub),
                                           _ptr(slide), _ptr(af), _ptr(bf), int(dims.has_bag_head), _ptr(fallback_count),
                                           scratch.data_ptr(), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_forward_guarded_wide")
    out: Dict[str, torch.Tensor] = {"range_status": _range_status(ws)}
    for k, v in (("A_out", A), ("sub_preds", sub), ("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    return out


def ga_rescore_fp32_cond(x: torch.Tensor, packed: torch.Tensor, W1: torch.Tensor, dims: GaDims, h: torch.Tensor, A: torch.Tensor,
                         status: torch.Tensor, fallback_count: Optional[torch.Tensor] = None) -> None:
    """acmil_ga_rescore_fp32_cond (composed path, eval): if the device word `status` (the range status a split-f16 projection launch
    left) is non-zero, h [N, Di] and A [K, N] are overwritten IN PLACE with their exact-fp32 values; nothing happens otherwise.  No
    host read-back: every launch of the repeat is predicated on the device."""
    lib = _lib.load()
    _check_x(x, dims)
    _need_cuda(packed, W1, h, A, status, fallback_count)
    N = x.shape[0]
    if tuple(h.shape) != (N, dims.Di) or tuple(A.shape) != (dims.K, N) or not h.is_contiguous() or not A.is_contiguous():
        raise RuntimeError("acmil_amd: h [N, D_inner] and A [K, N] of this bag, contiguous fp32")
    nsc = lib.acmil_ga_rescore_fp32_cond_scratch_bytes(N, dims.D, dims.Di, _DT[x.dtype])
    scratch = _repeat_scratch(nsc, x.device)
    rc = lib.acmil_ga_rescore_fp32_cond(x.data_ptr(), _DT[x.dtype], N, packed.data_ptr(), W1.data_ptr(), *dims.args(), dims.mode,
                                        h.data_ptr(), A.data_ptr(), status.data_ptr(), _ptr(fallback_count), scratch.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_rescore_fp32_cond")


def ga_scores(x: torch.Tensor, packed: torch.Tensor, dims: GaDims, mode, with_status: bool = False):
    """Score pass of a training step: raw scores A [K,N] and h [N,Di] (kept for pooling + backward);
    with_status: also the device view of the split-f16 range status (see _range_status)."""
    lib = _lib.load()
    mode = mode_id(mode)
    _check_x(x, dims)
    N, dev = x.shape[0], x.device
    A = torch.empty(dims.K, N, dtype=torch.float32, device=dev)
    h = torch.empty(N, dims.Di, dtype=torch.float32, device=dev)
    ws = _workspace(N, dims, mode, dev)        # tile counter + range status of the persistent kernel
    rc = lib.acmil_ga_forward(x.data_ptr(), _DT[x.dtype], N, packed.data_ptr(), *dims.args(), mode, A.data_ptr(), None,
                              None, None, None, h.data_ptr(), int(dims.has_bag_head), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_forward(score pass)")
    return (A, h, _range_status(ws)) if with_status else (A, h)


def stkim_select(scores: torch.Tensor, k: int, m: int, uniforms: Optional[torch.Tensor], rng: Optional[Tuple[int, int]] = None):
    """acmil_stkim_select(_rng): (topk_idx [K,k] int64 sorted by descending score, masked_idx [K,m] int64).
    uniforms [K,k]: the injected `torch.rand(K, k)` draw (parity tests); None + rng = (seed, offset): drawn on the device (Philox)."""
    lib = _lib.load()
    _need_cuda(scores)
    K, N = scores.shape
    dev = scores.device
    topk = torch.empty(K, k, dtype=torch.int64, device=dev)
    midx = torch.empty(K, m, dtype=torch.int64, device=dev)
    if m > 0 and uniforms is not None:
        if tuple(uniforms.shape) != (K, k):
            raise RuntimeError("acmil_amd: uniforms must be [K,k]")
        uniforms = uniforms.to(device=dev, dtype=torch.float32).contiguous()
    if m > 0 and uniforms is None and rng is None:
        raise RuntimeError("acmil_amd: STKIM needs either the uniforms [K,k] or rng = (seed, offset) for the device draw")
    seed, offset = rng if rng is not None else (0, 0)
    ws = torch.empty(lib.acmil_stkim_workspace_bytes(N, K, k), dtype=torch.uint8, device=dev)
    rc = lib.acmil_stkim_select_rng(scores.data_ptr(), N, K, k, m, _ptr(uniforms) if m > 0 else None, seed & (2 ** 64 - 1), offset & (2 ** 64 - 1),
                                    topk.data_ptr(), midx.data_ptr() if m > 0 else None, ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_stkim_select_rng")
    return topk, midx


def ga_pool(h: torch.Tensor, A: torch.Tensor, packed: torch.Tensor, dims: GaDims, mode,
            masked_idx: Optional[torch.Tensor], want_afeat: bool = False, want_bag_feat: bool = False):
    """acmil_ga_pool: masks A IN PLACE, then softmax / weighted sum / heads on the saved h."""
    lib = _lib.load()
    mode = mode_id(mode)
    _need_cuda(h, A)
    N, dev = h.shape[0], h.device
    f32 = dict(dtype=torch.float32, device=dev)
    sub = torch.empty(dims.K, dims.C, **f32)
    slide = torch.empty(dims.C, **f32) if dims.has_bag_head else None
    af = torch.empty(dims.K, dims.Di, **f32) if want_afeat else None
    bf = torch.empty(dims.Di, **f32) if want_bag_feat else None
    m = 0 if masked_idx is None else masked_idx.shape[1]
    ws = _workspace(N, dims, mode, dev)
    rc = lib.acmil_ga_pool(h.data_ptr(), A.data_ptr(), N, packed.data_ptr(), *dims.args(), mode,
                           _ptr(masked_idx) if m > 0 else None, m, sub.data_ptr(), _ptr(slide), _ptr(af), _ptr(bf),
                           int(dims.has_bag_head), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_pool")
    out = {"sub_preds": sub, "A_out": A}
    for k, v in (("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    return out


def ga_pool_group(h: torch.Tensor, A: torch.Tensor, rows: Sequence[int], packed: torch.Tensor, dims: GaDims, mode,
                  want_afeat: bool = False, want_bag_feat: bool = False):
    """acmil_ga_pool_group: unmasked softmax / weighted sum / heads per bag for up to 16 bags whose rows lie back to back in
    h [sum rows, Di] and A [K, sum rows] (A is not modified).  Outputs carry a leading bag axis."""
    lib = _lib.load()
    mode = mode_id(mode)
    _need_cuda(h, A)
    rows = [int(r) for r in rows]
    B, N, dev = len(rows), h.shape[0], h.device
    if B < 1 or B > MAX_GROUP or sum(rows) != N or A.shape != (dims.K, N) or not h.is_contiguous() or not A.is_contiguous():
        raise RuntimeError("acmil_amd.ga_pool_group: 1..%d bags, h [sum rows, Di] and A [K, sum rows] contiguous" % MAX_GROUP)
    f32 = dict(dtype=torch.float32, device=dev)
    sub = torch.empty(B, dims.K, dims.C, **f32)
    slide = torch.empty(B, dims.C, **f32) if dims.has_bag_head else None
    af = torch.empty(B, dims.K, dims.Di, **f32) if want_afeat else None
    bf = torch.empty(B, dims.Di, **f32) if want_bag_feat else None
    ws = _ws_bytes(lib.acmil_ga_pool_group_workspace_bytes(N, B, dims.Di, dims.K), dev)
    rc = lib.acmil_ga_pool_group(h.data_ptr(), A.data_ptr(), N, B, (ctypes.c_int * B)(*rows), packed.data_ptr(), *dims.args(), mode,
                                 sub.data_ptr(), _ptr(slide), _ptr(af), _ptr(bf), int(dims.has_bag_head), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_pool_group")
    out = {"sub_preds": sub, "A_out": A}
    for k, v in (("slide_pred", slide), ("afeat", af), ("bag_feat", bf)):
        if v is not None:
            out[k] = v
    return out


def gemm(a: torch.Tensor, b: torch.Tensor, trans_a: bool = False, trans_b: bool = False, alpha: float = 1.0,
         bias: Optional[torch.Tensor] = None, act: int = 0, out: Optional[torch.Tensor] = None, beta: float = 0.0,
         aux: Optional[torch.Tensor] = None, precision: str = "fp32") -> torch.Tensor:
    """acmil_gemm_f32 / acmil_gemm_f16x3 on 2-D (or batched 3-D) row-major tensors:
    out = act(alpha * op(a) @ op(b) + bias + beta*out).
    a fp32; b fp32/fp16/bf16; inner-most stride must be 1 (leading dimensions / batch strides are honoured).
    precision "fp32" = exact fp32 MFMA, "f16x3" / "bf16x3" = split-f16 / split-bf16 products (~1e-6 / ~1e-5 relative)."""
    if precision not in ("fp32", "f16x3", "bf16x3"):
        raise ValueError("acmil_amd.gemm: precision must be 'fp32', 'f16x3' or 'bf16x3'")
    lib = _lib.load()
    _need_cuda(a, b)
    if a.dim() == 2:
        a3, b3 = a.unsqueeze(0), b.unsqueeze(0)
    else:
        a3, b3 = a, b
    unit = lambda t: t.shape[-1] == 1 or t.stride(-1) == 1       # a size-1 inner dimension may carry any stride
    if not unit(a3) or not unit(b3) or a3.dtype != torch.float32 or b3.dtype not in _DT:
        raise RuntimeError("acmil_amd.gemm: operands must have unit inner stride; A fp32")
    batch = a3.shape[0]
    M, K = (a3.shape[2], a3.shape[1]) if trans_a else (a3.shape[1], a3.shape[2])
    K2, N = (b3.shape[2], b3.shape[1]) if trans_b else (b3.shape[1], b3.shape[2])
    if K != K2 or b3.shape[0] not in (1, batch):
        raise RuntimeError("acmil_amd.gemm: shape mismatch")
    if out is None:
        out = torch.empty((batch, M, N) if a.dim() == 3 else (M, N), dtype=torch.float32, device=a.device)
    o3 = out if out.dim() == 3 else out.unsqueeze(0)
    ws = torch.empty(lib.acmil_gemm_workspace_bytes(M, N, K, batch), dtype=torch.uint8, device=a.device)
    sb = 0 if b3.shape[0] == 1 else b3.stride(0)
    fn = {"fp32": lib.acmil_gemm_f32, "f16x3": lib.acmil_gemm_f16x3, "bf16x3": lib.acmil_gemm_bf16x3}[precision]
    rc = fn(int(trans_a), int(trans_b), M, N, K, float(alpha), a3.data_ptr(), a3.stride(1),
            a3.stride(0) if batch > 1 else 0, b3.data_ptr(), _DT[b3.dtype], b3.stride(1), sb, float(beta),
            o3.data_ptr(), o3.stride(1), o3.stride(0) if batch > 1 else 0, _ptr(bias), act, _ptr(aux),
            batch, ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_gemm")
    return out


def ga_backward(x: torch.Tensor, h: torch.Tensor, A_out: torch.Tensor, afeat: torch.Tensor, params: Sequence[torch.Tensor],
                dims: GaDims, d_sub: torch.Tensor, d_slide: Optional[torch.Tensor], d_A: Optional[torch.Tensor],
                grads_out: Optional[Sequence[torch.Tensor]] = None):
    """acmil_ga_backward.  params = [W1, Wv, bv, Wu, bu, Ww, bw, Wc_0..Wc_{K-1}, bc_0..bc_{K-1}, (Ws, bs)];
    returns the gradients in the same order."""
    lib = _lib.load()
    K, Cc, Di, D = dims.K, dims.C, dims.Di, dims.D
    W1, Wv, bv, Wu, bu, Ww, bw = params[:7]
    Wc = list(params[7:7 + K]); bc = list(params[7 + K:7 + 2 * K])
    Ws = params[7 + 2 * K] if dims.has_bag_head else None
    N, dev = x.shape[0], x.device
    grads = list(grads_out) if grads_out is not None else [torch.empty_like(p) for p in params]
    gW1, gWv, gbv, gWu, gbu, gWw, gbw = grads[:7]
    gWc, gbc = grads[7:7 + K], grads[7 + K:7 + 2 * K]
    gWs, gbs = (grads[7 + 2 * K], grads[8 + 2 * K]) if dims.has_bag_head else (None, None)
    f = lambda t: None if t is None else t.to(torch.float32).contiguous()
    d_sub, d_slide, d_A = f(d_sub), f(d_slide), f(d_A)
    if d_slide is not None:
        d_slide = d_slide.reshape(-1)
    if d_A is not None:
        d_A = d_A.reshape(K, N)
    arr = lambda ts: (ctypes.c_void_p * K)(*[t.data_ptr() for t in ts])
    ws = torch.empty(lib.acmil_ga_backward_workspace_bytes(N, D, Di, K, Cc), dtype=torch.uint8, device=dev)
    rc = lib.acmil_ga_backward(x.data_ptr(), _DT[x.dtype], N, h.data_ptr(), A_out.data_ptr(), afeat.data_ptr(),
                               Wv.data_ptr(), bv.data_ptr(), Wu.data_ptr(), bu.data_ptr(), Ww.data_ptr(), arr(Wc), _ptr(Ws),
                               d_sub.data_ptr(), _ptr(d_slide), _ptr(d_A), gW1.data_ptr(), gWv.data_ptr(), gbv.data_ptr(),
                               gWu.data_ptr(), gbu.data_ptr(), gWw.data_ptr(), gbw.data_ptr(), arr(gWc), arr(gbc),
                               _ptr(gWs), _ptr(gbs), D, Di, GA_DA, K, Cc, dims.mode, ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_backward")
    return grads


# validated (parameter, gradient) sets of ga_train_step: key -> the tensors themselves.  The strong references are the point: while an
# entry lives its tensors cannot be freed, so neither their id() nor their storage address can be taken over by a tensor of another
# dtype / shape (the kernels get raw pointers); `p.data = ...` / `set_` change data_ptr and miss the cache.  A few models per process.
_TRAIN_STEP_CHECKED: Dict[tuple, tuple] = {}
_TRAIN_STEP_CHECKED_MAX = 8


def ga_train_step(x: torch.Tensor, packed: torch.Tensor, dims: GaDims, mode, params: Sequence[torch.Tensor],
                  grads: Sequence[torch.Tensor], label: torch.Tensor, uniforms: Optional[torch.Tensor], k_top: int, m_mask: int,
                  repack: bool = True, guard_flag: Optional[torch.Tensor] = None, rng: Optional[Tuple[int, int]] = None,
                  adamw: Optional[tuple] = None):
    """acmil_ga_train_step: forward with STKIM masking + ACMIL loss + backward of one slide, enqueued by ONE library call.
    adamw (single-GPU runs): (flat_params, exp_avg, exp_avg_sq, lr, beta1, beta2, eps, weight_decay, step, skipped_dev, flag_report_ptr)
    of a FlatAdamW -- the call then goes to acmil_ga_train_step_adamw, whose last launch finishes the gradients, applies the update
    and rewrites `packed` for the new values (so the next call may pass repack=False).
    params / grads = [W1, Wv, bv, Wu, bu, Ww, bw, Wc_0.., bc_0.., (Ws, bs)] (gradients are overwritten).
    Returns a dict: losses [4] (loss0, loss1, diff, total), sub_preds [K,C], slide_pred [C] or None, A_out [K,N] (masked raw
    scores), topk_idx, masked_idx, range_status (device int32 view, see _range_status).
    guard_flag: a device float the step writes 1.0 / 0.0 into (range status != 0) without any host read-back."""
    lib = _lib.load()
    mode = mode_id(mode)
    _check_x(x, dims)
    K, Cc = dims.K, dims.C
    N, dev = x.shape[0], x.device
    # every pointer below is handed to the kernels raw: check what the op-by-op path checked in its wrappers.  The tensor-by-tensor
    # pass (~40 us of host time for 19 parameters) is remembered for the exact set of storages it was made on: a training loop hands
    # the same parameter / gradient tensors every step
    pp = [p.data_ptr() for p in params]
    gp = [g.data_ptr() for g in grads]
    seen = (dev, tuple(map(id, params)), tuple(pp), tuple(map(id, grads)), tuple(gp))
    if seen not in _TRAIN_STEP_CHECKED:
        _need_cuda(*params, *grads)
        n_par = 7 + 2 * K + (2 if dims.has_bag_head else 0)
        if len(params) != n_par or len(grads) != n_par:
            raise RuntimeError("acmil_amd.ga_train_step: expected %d parameters / gradients, got %d / %d" % (n_par, len(params), len(grads)))
        for p, g in zip(params, grads):
            if p.dtype != torch.float32 or g.dtype != torch.float32 or not p.is_contiguous() or not g.is_contiguous() or g.shape != p.shape \
                    or p.device != dev or g.device != dev:
                raise RuntimeError("acmil_amd.ga_train_step: parameters and gradients must be contiguous fp32 on the bag's device, same shapes")
        if len(_TRAIN_STEP_CHECKED) >= _TRAIN_STEP_CHECKED_MAX:
            _TRAIN_STEP_CHECKED.pop(next(iter(_TRAIN_STEP_CHECKED)))        # oldest entry (insertion order)
        _TRAIN_STEP_CHECKED[seen] = (tuple(params), tuple(grads))
    _need_cuda(label, guard_flag)
    if label.device != dev or label.numel() < 1:
        raise RuntimeError("acmil_amd.ga_train_step: label must be a [1] tensor on the bag's device")
    if label.dtype != torch.int64 or not label.is_contiguous():
        label = label.to(torch.int64).contiguous()
    if not (0 <= k_top <= N) or not (0 <= m_mask <= k_top):
        raise RuntimeError("acmil_amd.ga_train_step: need 0 <= m_mask <= k_top <= N (got k_top=%d m_mask=%d N=%d)" % (k_top, m_mask, N))
    if m_mask > 0 and uniforms is None and rng is None:
        raise RuntimeError("acmil_amd.ga_train_step: masking needs either the uniforms [K, k_top] or rng = (seed, offset) for the device draw")
    if m_mask > 0 and uniforms is not None:
        if tuple(uniforms.shape) != (K, k_top):       # the kernel reads row k at stride k_top
            raise RuntimeError("acmil_amd.ga_train_step: uniforms must be [K=%d, k_top=%d], got %s" % (K, k_top, tuple(uniforms.shape)))
        uniforms = uniforms.to(device=dev, dtype=torch.float32).contiguous()      # as acmil_stkim_select's wrapper does
    seed, offset = rng if rng is not None else (0, 0)
    if guard_flag is not None and (guard_flag.dtype != torch.float32 or guard_flag.device != dev or guard_flag.numel() < 1):
        raise RuntimeError("acmil_amd.ga_train_step: guard_flag must be a float32 device scalar")
    fbuf = torch.empty(4 + K * Cc + Cc + K * N, dtype=torch.float32, device=dev)
    losses, sub, slide, A = fbuf[:4], fbuf[4:4 + K * Cc].view(K, Cc), fbuf[4 + K * Cc:4 + K * Cc + Cc], fbuf[4 + K * Cc + Cc:].view(K, N)
    ibuf = torch.empty(K * (k_top + m_mask) + 1, dtype=torch.int64, device=dev)
    topk, midx = ibuf[:K * k_top].view(K, k_top), ibuf[K * k_top:K * (k_top + m_mask)].view(K, m_mask)
    ws = _ws_bytes(lib.acmil_ga_train_step_workspace_bytes(N, dims.D, dims.Di, K, Cc, k_top), dev)
    vpK = ctypes.c_void_p * K
    has_bag = dims.has_bag_head
    common = (
        x.data_ptr(), _DT[x.dtype], N, packed.data_ptr(), int(repack),
        *pp[:7], vpK(*pp[7:7 + K]), vpK(*pp[7 + K:7 + 2 * K]), pp[7 + 2 * K] if has_bag else None, pp[8 + 2 * K] if has_bag else None,
        *gp[:7], vpK(*gp[7:7 + K]), vpK(*gp[7 + K:7 + 2 * K]), gp[7 + 2 * K] if has_bag else None, gp[8 + 2 * K] if has_bag else None,
        *dims.args(), mode, label.data_ptr(), _ptr(uniforms) if m_mask > 0 else None, k_top, m_mask,
        losses.data_ptr(), sub.data_ptr(), slide.data_ptr() if has_bag else None, A.data_ptr(),
        topk.data_ptr() if k_top > 0 else None, midx.data_ptr() if m_mask > 0 else None, _ptr(guard_flag), ws.data_ptr(), _stream(),
        seed & (2 ** 64 - 1), offset & (2 ** 64 - 1))
    if adamw is None:
        rc = lib.acmil_ga_train_step_rng(*common)
        _lib.check(rc, "acmil_ga_train_step_rng")
    else:
        flat, m1, m2, lr, b1, b2, eps, wd, step, skipped, report = adamw
        rc = lib.acmil_ga_train_step_adamw(*common, flat.data_ptr(), flat.numel(), m1.data_ptr(), m2.data_ptr(), float(lr), float(b1),
                                           float(b2), float(eps), float(wd), int(step), skipped.data_ptr(), report)
        _lib.check(rc, "acmil_ga_train_step_adamw")
    return {"losses": losses, "sub_preds": sub, "slide_pred": slide if has_bag else None, "A_out": A,
            "topk_idx": topk if k_top > 0 else None, "masked_idx": midx if m_mask > 0 else None, "range_status": _range_status(ws)}




def ga_train_step_group(x: torch.Tensor, rows: Sequence[int], packed: torch.Tensor, dims: GaDims, mode, params: Sequence[torch.Tensor],
                        grads: Sequence[torch.Tensor], labels: torch.Tensor, uniforms: Optional[torch.Tensor], k_top: int, m_mask: int,
                        repack: bool = True, guard_flag: Optional[torch.Tensor] = None, rng: Optional[Tuple[int, int]] = None,
                        adamw: Optional[tuple] = None):
    """acmil_ga_train_step_group: ONE training step over a GROUP of bags (the single-GPU twin of slide-level data parallelism: the
    parameter gradients are the MEAN of the bags' per-slide gradients).  x [sum(rows), D]: the bags' rows back to back; rows: the
    bags' patch counts (host ints, 1 .. 16 bags); labels [G] int64 on the device; uniforms [G, K, k_top] or None (device draw).
    Returns a dict: losses [G,4], sub_preds [G,K,C], slide_pred [G,C] or None, A_out [K, sum(rows)] (bag b = columns
    offsets[b]:offsets[b+1]), topk_idx [G,K,k_top], masked_idx [G,K,m_mask] (bag-local indices), offsets, range_status."""
    lib = _lib.load()
    mode = mode_id(mode)
    _check_x(x, dims)
    rows = [int(r) for r in rows]
    G = len(rows)
    K, Cc = dims.K, dims.C
    N, dev = x.shape[0], x.device
    if not (1 <= G <= MAX_GROUP) or sum(rows) != N or min(rows) < max(1, k_top):
        raise RuntimeError("acmil_amd.ga_train_step_group: need 1..%d bags of >= max(1, k_top) rows that add up to x.shape[0] (got %s, N=%d, k_top=%d)"
                           % (MAX_GROUP, rows, N, k_top))
    if not x.is_contiguous():
        raise RuntimeError("acmil_amd.ga_train_step_group: x must be contiguous")
    pp = [p.data_ptr() for p in params]
    gp = [g.data_ptr() for g in grads]
    seen = (dev, tuple(map(id, params)), tuple(pp), tuple(map(id, grads)), tuple(gp))
    if seen not in _TRAIN_STEP_CHECKED:
        _need_cuda(*params, *grads)
        n_par = 7 + 2 * K + (2 if dims.has_bag_head else 0)
        if len(params) != n_par or len(grads) != n_par:
            raise RuntimeError("acmil_amd.ga_train_step_group: expected %d parameters / gradients, got %d / %d" % (n_par, len(params), len(grads)))
        for p, g in zip(params, grads):
            if p.dtype != torch.float32 or g.dtype != torch.float32 or not p.is_contiguous() or not g.is_contiguous() or g.shape != p.shape \
                    or p.device != dev or g.device != dev:
                raise RuntimeError("acmil_amd.ga_train_step_group: parameters and gradients must be contiguous fp32 on the bags' device, same shapes")
        if len(_TRAIN_STEP_CHECKED) >= _TRAIN_STEP_CHECKED_MAX:
            _TRAIN_STEP_CHECKED.pop(next(iter(_TRAIN_STEP_CHECKED)))
        _TRAIN_STEP_CHECKED[seen] = (tuple(params), tuple(grads))
    _need_cuda(labels, guard_flag)
    if labels.device != dev or labels.numel() != G:
        raise RuntimeError("acmil_amd.ga_train_step_group: labels must be a [%d] tensor on the bags' device" % G)
    if labels.dtype != torch.int64 or not labels.is_contiguous():
        labels = labels.to(torch.int64).contiguous()
    if not (0 <= m_mask <= k_top):
        raise RuntimeError("acmil_amd.ga_train_step_group: need 0 <= m_mask <= k_top")
    if m_mask > 0 and uniforms is None and rng is None:
        raise RuntimeError("acmil_amd.ga_train_step_group: masking needs either the uniforms [G, K, k_top] or rng = (seed, offset)")
    if m_mask > 0 and uniforms is not None:
        if tuple(uniforms.shape) != (G, K, k_top):
            raise RuntimeError("acmil_amd.ga_train_step_group: uniforms must be [G=%d, K=%d, k_top=%d], got %s" % (G, K, k_top, tuple(uniforms.shape)))
        uniforms = uniforms.to(device=dev, dtype=torch.float32).contiguous()
    seed, offset = rng if rng is not None else (0, 0)
    if guard_flag is not None and (guard_flag.dtype != torch.float32 or guard_flag.device != dev or guard_flag.numel() < 1):
        raise RuntimeError("acmil_amd.ga_train_step_group: guard_flag must be a float32 device scalar")
    n_l, n_s, n_b = 4 * G, G * K * Cc, G * Cc
    fbuf = torch.empty(n_l + n_s + n_b + K * N, dtype=torch.float32, device=dev)
    losses, sub, slide, A = fbuf[:n_l].view(G, 4), fbuf[n_l:n_l + n_s].view(G, K, Cc), fbuf[n_l + n_s:n_l + n_s + n_b].view(G, Cc), \
        fbuf[n_l + n_s + n_b:].view(K, N)
    ibuf = torch.empty(G * K * (k_top + m_mask) + 1, dtype=torch.int64, device=dev)
    topk, midx = ibuf[:G * K * k_top].view(G, K, k_top), ibuf[G * K * k_top:G * K * (k_top + m_mask)].view(G, K, m_mask)
    ws = _ws_bytes(lib.acmil_ga_train_step_group_workspace_bytes(G, N, dims.D, dims.Di, K, Cc, k_top), dev)
    vpK = ctypes.c_void_p * K
    has_bag = dims.has_bag_head
    rows_arr = (ctypes.c_int * G)(*rows)
    aw = None
    if adamw is not None:
        flat, m1, m2, lr, b1, b2, eps, wd, step, skipped, report = adamw
        aw = _lib.AdamwArgs(flat.data_ptr(), flat.numel(), m1.data_ptr(), m2.data_ptr(), float(lr), float(b1), float(b2), float(eps), float(wd),
                            int(step), skipped.data_ptr(), report)
    rc = lib.acmil_ga_train_step_group(
        x.data_ptr(), _DT[x.dtype], G, rows_arr, packed.data_ptr(), int(repack),
        *pp[:7], vpK(*pp[7:7 + K]), vpK(*pp[7 + K:7 + 2 * K]), pp[7 + 2 * K] if has_bag else None, pp[8 + 2 * K] if has_bag else None,
        *gp[:7], vpK(*gp[7:7 + K]), vpK(*gp[7 + K:7 + 2 * K]), gp[7 + 2 * K] if has_bag else None, gp[8 + 2 * K] if has_bag else None,
        *dims.args(), mode, labels.data_ptr(), _ptr(uniforms) if m_mask > 0 else None, k_top, m_mask,
        losses.data_ptr(), sub.data_ptr(), slide.data_ptr() if has_bag else None, A.data_ptr(),
        topk.data_ptr() if k_top > 0 else None, midx.data_ptr() if m_mask > 0 else None, _ptr(guard_flag), ws.data_ptr(), _stream(),
        seed & (2 ** 64 - 1), offset & (2 ** 64 - 1), ctypes.byref(aw) if aw is not None else None)
    _lib.check(rc, "acmil_ga_train_step_group")
    offs = [0]
    for r in rows:
        offs.append(offs[-1] + r)
    return {"losses": losses, "sub_preds": sub, "slide_pred": slide if has_bag else None, "A_out": A, "offsets": offs,
            "topk_idx": topk if k_top > 0 else None, "masked_idx": midx if m_mask > 0 else None, "range_status": _range_status(ws)}


def ga_adamw_supported(dims: GaDims, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], flat: torch.Tensor,
                       exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor) -> bool:
    """acmil_ga_adamw_supported: would acmil_ga_train_step_adamw / _group(adamw) / acmil_ga_adamw_pack accept this parameter set?
    Launches nothing."""
    lib = _lib.load()
    K = dims.K
    pp = [p.data_ptr() for p in params]
    gp = [g.data_ptr() for g in grads]
    vpK = ctypes.c_void_p * K
    has_bag = dims.has_bag_head
    rc = lib.acmil_ga_adamw_supported(
        *pp[:7], vpK(*pp[7:7 + K]), vpK(*pp[7 + K:7 + 2 * K]), pp[7 + 2 * K] if has_bag else None, pp[8 + 2 * K] if has_bag else None,
        gp[0], gp[1], gp[3], *dims.args(), mode_id("f16x3"), flat.data_ptr(), flat.numel(), exp_avg.data_ptr(), exp_avg_sq.data_ptr())
    return rc == 0


def ga_adamw_pack(packed: torch.Tensor, dims: GaDims, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], adamw: tuple,
                  skip_flag: Optional[torch.Tensor]):
    """acmil_ga_adamw_pack: AdamW over the module's flat parameter buffer + re-pack of the f16x3 packed buffer, one launch (final
    gradients: the data-parallel step).  params / grads as ga_train_step; adamw as there."""
    lib = _lib.load()
    K = dims.K
    pp = [p.data_ptr() for p in params]
    gp = [g.data_ptr() for g in grads]
    vpK = ctypes.c_void_p * K
    has_bag = dims.has_bag_head
    flat, m1, m2, lr, b1, b2, eps, wd, step, skipped, report = adamw
    rc = lib.acmil_ga_adamw_pack(
        *pp[:7], vpK(*pp[7:7 + K]), vpK(*pp[7 + K:7 + 2 * K]), pp[7 + 2 * K] if has_bag else None, pp[8 + 2 * K] if has_bag else None,
        *gp[:7], vpK(*gp[7:7 + K]), vpK(*gp[7 + K:7 + 2 * K]), gp[7 + 2 * K] if has_bag else None, gp[8 + 2 * K] if has_bag else None,
        *dims.args(), mode_id("f16x3"), packed.data_ptr(), flat.data_ptr(), flat.numel(), m1.data_ptr(), m2.data_ptr(), float(lr), float(b1),
        float(b2), float(eps), float(wd), int(step), _ptr(skip_flag), skipped.data_ptr(), report, _stream())
    _lib.check(rc, "acmil_ga_adamw_pack")


_TM_SIDE: Dict[tuple, tuple] = {}
_TM_SIDE_LOCK = threading.Lock()


def _transmil_side(dev: torch.device):
    """The (side stream, fork event, join event) triple acmil_transmil_forward_ex works with beside the current stream: owned HERE,
    by the caller of the library (one per device and compute stream, high priority, created at first use).  Nothing is created
    inside a graph capture: a capturing stream without a triple of its own (torch.cuda.graph captures on an internal stream) takes
    the device's spare triple, made together with the first eager one -- or runs serially if there has been no eager call yet.
    Returns raw handles, or (None, None, None)."""
    cur = torch.cuda.current_stream(dev)
    di = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (di, cur.cuda_stream)
    t = _TM_SIDE.get(key)
    if t is None:
        if torch.cuda.is_current_stream_capturing():
            t = _TM_SIDE.get((di, "capture"))
            if t is None:
                return None, None, None
        else:
            with _TM_SIDE_LOCK:
                t = _TM_SIDE.get(key)
                if t is None:
                    def make():
                        side = torch.cuda.Stream(device=dev, priority=-1)
                        fork, join = torch.cuda.Event(), torch.cuda.Event()
                        fork.record(cur); join.record(side)          # torch creates the hipEvent_t at the first record
                        return (side, fork, join)
                    t = _TM_SIDE[key] = make()
                    if (di, "capture") not in _TM_SIDE:
                        _TM_SIDE[(di, "capture")] = make()
    return t[0].cuda_stream, t[1].cuda_event, t[2].cuda_event


def transmil_forward(x: torch.Tensor, sd: Dict[str, torch.Tensor], n_class: int, debug: bool = False,
                     workspace: Optional[torch.Tensor] = None, side_stream: bool = True) -> Dict[str, torch.Tensor]:
    """acmil_transmil_forward_ex.  x [N,D] fp32 CUDA; sd: parameters under the reference's state_dict names
    (fp32, CUDA, contiguous).  Returns {'logits': [C]} plus 'h1','hp','h2' [(side^2+1), Di] when debug.
    workspace: a caller-owned uint8 CUDA buffer of at least acmil_transmil_workspace_bytes (tests: pre-filled scratch, canaries).
    side_stream=False: every launch on the current stream (the serial pipeline)."""
    lib = _lib.load()
    _need_cuda(x)
    if x.dtype != torch.float32:
        x = x.float()        # storage-format conversion only (fp16 bag -> fp32 operand of the fp32 MFMA GEMM)
    x = x.contiguous()
    N, D = x.shape
    Di = sd["_fc1.0.weight"].shape[0]
    c = lambda k: sd[k].detach().contiguous()
    keep = []

    def arr(keys):
        ts = [c(k) for k in keys]
        keep.extend(ts)
        return (ctypes.c_void_p * len(ts))(*[t.data_ptr() for t in ts])

    lay = lambda p: arr([p + ".norm.weight", p + ".norm.bias", p + ".attn.to_qkv.weight", p + ".attn.to_out.0.weight",
                         p + ".attn.to_out.0.bias", p + ".attn.res_conv.weight"])
    l1, l2 = lay("layer1"), lay("layer2")
    pp = arr(["pos_layer.proj.weight", "pos_layer.proj.bias", "pos_layer.proj1.weight", "pos_layer.proj1.bias",
              "pos_layer.proj2.weight", "pos_layer.proj2.bias"])
    small = [c(k) for k in ("_fc1.0.weight", "_fc1.0.bias", "cls_token", "norm.weight", "norm.bias", "_fc2.weight", "_fc2.bias")]
    nbytes = lib.acmil_transmil_workspace_bytes(N, D, Di, n_class)
    if nbytes == 0:
        raise RuntimeError("acmil_amd: unsupported TransMIL dimensions")
    if workspace is not None:
        if not workspace.is_cuda or workspace.dtype != torch.uint8 or workspace.numel() < nbytes or workspace.data_ptr() % 256 != 0:
            raise RuntimeError("acmil_amd: workspace must be a 256-byte aligned uint8 CUDA buffer of >= %d bytes" % nbytes)
        ws = workspace
    else:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    logits = torch.empty(n_class, dtype=torch.float32, device=x.device)
    import math
    side = int(math.ceil(math.sqrt(N)))
    dbg = [torch.empty(side * side + 1, Di, dtype=torch.float32, device=x.device) for _ in range(3)] if debug else [None] * 3
    ss, ef, ej = _transmil_side(x.device) if side_stream else (None, None, None)
    rc = lib.acmil_transmil_forward_ex(x.data_ptr(), N, D, Di, n_class, small[0].data_ptr(), small[1].data_ptr(), small[2].data_ptr(),
                                       l1, l2, pp, small[3].data_ptr(), small[4].data_ptr(), small[5].data_ptr(), small[6].data_ptr(),
                                       logits.data_ptr(), _ptr(dbg[0]), _ptr(dbg[1]), _ptr(dbg[2]), ws.data_ptr(), _stream(), ss, ef, ej)
    _lib.check(rc, "acmil_transmil_forward_ex")
    out = {"logits": logits}
    if debug:
        out.update(h1=dbg[0], hp=dbg[1], h2=dbg[2])
    return out


def ga_loss(sub_preds: torch.Tensor, slide_pred: Optional[torch.Tensor], A_out: torch.Tensor, label: torch.Tensor):
    """acmil_ga_loss: (losses [4] = loss0, loss1, diff, total; d_sub [K,C]; d_slide [C] or None; d_A [K,N])."""
    lib = _lib.load()
    _need_cuda(sub_preds, A_out, label)
    K, N = A_out.shape[-2], A_out.shape[-1]
    Cc = sub_preds.shape[1]
    dev = A_out.device
    losses = torch.empty(4, dtype=torch.float32, device=dev)
    d_sub = torch.empty(K, Cc, dtype=torch.float32, device=dev)
    d_slide = torch.empty(Cc, dtype=torch.float32, device=dev) if slide_pred is not None else None
    d_A = torch.empty(K, N, dtype=torch.float32, device=dev)
    ws = torch.empty(lib.acmil_ga_loss_workspace_bytes(N, K), dtype=torch.uint8, device=dev)
    label = label.to(torch.int64)
    rc = lib.acmil_ga_loss(sub_preds.data_ptr(), _ptr(slide_pred), A_out.data_ptr(), label.data_ptr(), N, K, Cc,
                           losses.data_ptr(), d_sub.data_ptr(), _ptr(d_slide), d_A.data_ptr(), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_ga_loss")
    return losses, d_sub, d_slide, d_A


def mha_forward(x: torch.Tensor, sd: Dict[str, torch.Tensor], n_token: int, n_class: int, precision="f16x3") -> Dict[str, torch.Tensor]:
    """acmil_mha_forward.  x [N,D] fp32 CUDA; sd: ACMIL_MHA parameters under the reference's state_dict names (fp32, CUDA,
    contiguous).  Returns {'sub_preds' [K,C], 'slide_pred' [C], 'attns' [8,K,N]}."""
    lib = _lib.load()
    _need_cuda(x)
    if x.dtype != torch.float32 or not x.is_contiguous():
        raise RuntimeError("acmil_amd.mha_forward: x must be contiguous fp32 [N, D]")
    mode = mode_id(precision)
    N, D = x.shape
    W1 = sd["dimreduction.fc1.weight"]
    Di, K, C = W1.shape[0], n_token, n_class
    keep = []

    def ptr(name):
        t = sd[name]
        if not t.is_cuda or t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError("acmil_amd.mha_forward: parameter %s must be contiguous fp32 on the GPU" % name)
        keep.append(t)
        return t.data_ptr()
    names = ("q_proj.weight", "q_proj.bias", "k_proj.weight", "k_proj.bias", "v_proj.weight", "v_proj.bias", "out_proj.weight",
             "out_proj.bias", "layer_norm.weight", "layer_norm.bias")
    branch = (ctypes.c_void_p * (10 * K))(*[ptr("sub_attention.%d.%s" % (i, nm)) for i in range(K) for nm in names])
    bag = (ctypes.c_void_p * 6)(*[ptr("bag_attention." + nm) for nm in names[4:]])
    Wc = (ctypes.c_void_p * K)(*[ptr("classifier.%d.fc.weight" % i) for i in range(K)])
    bc = (ctypes.c_void_p * K)(*[ptr("classifier.%d.fc.bias" % i) for i in range(K)])
    q = sd["q"].reshape(K, Di)
    nbytes = lib.acmil_mha_workspace_bytes(N, D, Di, K, C)
    if nbytes == 0:
        raise RuntimeError("acmil_amd.mha_forward: unsupported shape (Di %% 64 == 0, Di <= 512, n_token <= 5)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    sub = torch.empty(K, C, dtype=torch.float32, device=x.device)
    slide = torch.empty(C, dtype=torch.float32, device=x.device)
    attns = torch.empty(8, K, N, dtype=torch.float32, device=x.device)
    rc = lib.acmil_mha_forward(x.data_ptr(), N, D, Di, K, C, ptr("dimreduction.fc1.weight"), q.data_ptr(), branch, bag, Wc, bc,
                               ptr("Slide_classifier.fc.weight"), ptr("Slide_classifier.fc.bias"), mode, sub.data_ptr(),
                               slide.data_ptr(), attns.data_ptr(), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_mha_forward")
    return {"sub_preds": sub, "slide_pred": slide, "attns": attns}


def gated_scores(h: torch.Tensor, Wv, bv, Wu, bu, Ww, bw, precision="f16x3") -> torch.Tensor:
    """acmil_gated_scores: raw gated-attention scores A [K,N] of an already projected bag h [N,L] (any attention width Da)."""
    lib = _lib.load()
    ts = [h, Wv, bv, Wu, bu, Ww, bw]
    _need_cuda(*ts)
    ts = [t.detach() for t in ts]
    for t in ts:
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError("acmil_amd.gated_scores: operands must be contiguous fp32")
    h, Wv, bv, Wu, bu, Ww, bw = ts
    N, L = h.shape
    Da, K = Wv.shape[0], Ww.shape[0]
    A = torch.empty(K, N, dtype=torch.float32, device=h.device)
    ws = torch.empty(lib.acmil_gated_scores_workspace_bytes(N, L, Da, K), dtype=torch.uint8, device=h.device)
    rc = lib.acmil_gated_scores(h.data_ptr(), N, L, Da, K, Wv.data_ptr(), bv.data_ptr(), Wu.data_ptr(), bu.data_ptr(), Ww.data_ptr(),
                                bw.data_ptr(), mode_id(precision), A.data_ptr(), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_gated_scores")
    return A


def pack_gate(Wv: torch.Tensor, bv: torch.Tensor, Wu: torch.Tensor, bu: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Operands of gated_scores_packed: the fragment stream of the [256, L] matrix whose rows alternate 32 Wv / 32 Wu units (a
    storage rearrangement of the two weight matrices, then acmil_linear_pack) and the bias vector in the same order."""
    _need_cuda(Wv, bv, Wu, bu)
    if Wv.shape[0] != GA_DA or Wu.shape != Wv.shape:
        raise RuntimeError("acmil_amd.pack_gate: attention width must be 128")
    L = Wv.shape[1]
    wcat = torch.stack([Wv.detach().view(4, 32, L), Wu.detach().view(4, 32, L)], dim=1).reshape(2 * GA_DA, L).contiguous()
    bcat = torch.stack([bv.detach().view(4, 32), bu.detach().view(4, 32)], dim=1).reshape(2 * GA_DA).contiguous()
    return linear_pack(wcat), bcat


def gated_scores_packed(h: torch.Tensor, packed_vu: torch.Tensor, bias_vu: torch.Tensor, Ww: torch.Tensor, bw: torch.Tensor) -> torch.Tensor:
    """acmil_gated_scores_packed: raw gated-attention scores A [K, N] of a projected bag h [N, L] in ONE pass over h (split-f16 MFMA
    product with the gate formed in the accumulators; the [N, 256] pre-activations never exist).  Attention width 128."""
    lib = _lib.load()
    _need_cuda(h, packed_vu, bias_vu, Ww, bw)
    Ww, bw = Ww.detach(), bw.detach()
    if h.dim() != 2 or h.stride(1) != 1 or h.dtype not in _DT or not Ww.is_contiguous() or Ww.dtype != torch.float32 or Ww.shape[1] != GA_DA:
        raise RuntimeError("acmil_amd.gated_scores_packed: h [N, L] with unit inner stride, Ww contiguous fp32 [K, 128]")
    N, L = h.shape
    K = Ww.shape[0]
    A = torch.empty(K, N, dtype=torch.float32, device=h.device)
    ws = torch.empty(256, dtype=torch.uint8, device=h.device)
    rc = lib.acmil_gated_scores_packed(h.data_ptr(), _DT[h.dtype], N, L, h.stride(0), packed_vu.data_ptr(), bias_vu.data_ptr(), Ww.data_ptr(),
                                       bw.data_ptr(), K, A.data_ptr(), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_gated_scores_packed")
    return A


def attn_pool(h: torch.Tensor, A: torch.Tensor) -> torch.Tensor:
    """acmil_attn_pool: softmax over N of the raw scores A [K,N], then the weighted sum afeat [K,Di] = P h."""
    lib = _lib.load()
    _need_cuda(h, A)
    h, A = h.detach(), A.detach()
    if h.dtype != torch.float32 or A.dtype != torch.float32 or not h.is_contiguous() or not A.is_contiguous():
        raise RuntimeError("acmil_amd.attn_pool: h and A must be contiguous fp32")
    N, Di = h.shape
    K = A.shape[0]
    nbytes = lib.acmil_attn_pool_workspace_bytes(N, Di, K)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    af = torch.empty(K, Di, dtype=torch.float32, device=h.device)
    _lib.check(lib.acmil_attn_pool(h.data_ptr(), A.data_ptr(), N, Di, K, af.data_ptr(), ws.data_ptr(), _stream()), "acmil_attn_pool")
    return af


def softmax_rows(S: torch.Tensor) -> torch.Tensor:
    """acmil_softmax_rows: softmax over the last axis of a 2-D fp32 tensor (long rows: the attention maps [K,N])."""
    lib = _lib.load()
    _need_cuda(S)
    S = S.detach()
    if S.dim() != 2 or S.dtype != torch.float32 or not S.is_contiguous():
        raise RuntimeError("acmil_amd.softmax_rows: S must be contiguous fp32 [rows, cols]")
    P = torch.empty_like(S)
    _lib.check(lib.acmil_softmax_rows(S.data_ptr(), P.data_ptr(), S.shape[0], S.shape[1], _stream()), "acmil_softmax_rows")
    return P


def attn_row_stats(A: torch.Tensor) -> torch.Tensor:
    """acmil_attn_row_stats: [rows, 4] = (max, sum e^{s-m}, sum e^{s-m}(s-m), sum_n p log p) per row of the raw scores A [rows, N]."""
    lib = _lib.load()
    _need_cuda(A)
    A2 = A.detach().reshape(-1, A.shape[-1]).to(torch.float32).contiguous()
    stats = torch.empty(A2.shape[0], 4, dtype=torch.float32, device=A.device)
    _lib.check(lib.acmil_attn_row_stats(A2.data_ptr(), A2.shape[0], A2.shape[1], stats.data_ptr(), _stream()), "acmil_attn_row_stats")
    return stats


def attn_entropy_loss(attn: torch.Tensor) -> torch.Tensor:
    """evaluate()'s div_loss = sum(softmax(attn) * log_softmax(attn)) / attn.shape[1] (Step3_WSI_classification_ACMIL.py:259)
    for attn [B, K, N] (GA: B = 1; MHA: B = 8 heads), as a device scalar; one HIP launch, no [K,N] temporaries."""
    return attn_row_stats(attn)[:, 3].sum() / attn.shape[1]


def attn_heatmap(attn: torch.Tensor, zoom_factor: float = 1.0) -> torch.Tensor:
    """acmil_attn_heatmap: probs [N] = softmax(attn, -1)[0].mean(0) * N * zoom_factor (Step4_visualize_heatmap_camelyon.py:117-118)."""
    lib = _lib.load()
    _need_cuda(attn)
    A = attn.detach()
    A = (A[0] if A.dim() == 3 else A).to(torch.float32).contiguous()
    K, N = A.shape
    probs = torch.empty(N, dtype=torch.float32, device=A.device)
    stats = torch.empty(K, 4, dtype=torch.float32, device=A.device)
    _lib.check(lib.acmil_attn_heatmap(A.data_ptr(), K, N, float(N * zoom_factor), probs.data_ptr(), stats.data_ptr(), _stream()),
               "acmil_attn_heatmap")
    return probs


def linear_pack(W: torch.Tensor) -> torch.Tensor:
    """acmil_linear_pack: W [n_out, K] fp32 (CUDA, contiguous) -> packed fragment stream (uint8) for linear_f16x3."""
    lib = _lib.load()
    _need_cuda(W)
    W = W.detach()
    if W.dtype != torch.float32 or not W.is_contiguous() or W.dim() != 2:
        raise RuntimeError("acmil_amd.linear_pack: W must be contiguous fp32 [n_out, K]")
    n_out, K = W.shape
    nbytes = lib.acmil_linear_packed_bytes(n_out, K)
    if nbytes == 0:
        raise RuntimeError("acmil_amd.linear_pack: needs n_out % 128 == 0, K % 16 == 0 and K >= 32, got %s" % (tuple(W.shape),))
    packed = torch.empty(nbytes, dtype=torch.uint8, device=W.device)
    _lib.check(lib.acmil_linear_pack(W.data_ptr(), K, n_out, K, packed.data_ptr(), _stream()), "acmil_linear_pack")
    return packed


def linear_f16x3(x: torch.Tensor, packed: torch.Tensor, n_out: int, bias: Optional[torch.Tensor] = None, relu: bool = False,
                 out: Optional[torch.Tensor] = None, beta: float = 0.0, want_status: bool = False):
    """acmil_linear_f16x3: y = act(x W^T + bias) + beta * y for x [M, K] (fp32 / fp16 / bf16, unit inner stride).
    want_status: also the device int32 range word of this call (non-zero: an output left the f16 range / was not finite)."""
    lib = _lib.load()
    _need_cuda(x, packed)
    if x.dim() != 2 or x.stride(1) != 1 or x.dtype not in _DT:
        raise RuntimeError("acmil_amd.linear_f16x3: x must be [M, K] with unit inner stride")
    M, K = x.shape
    if out is None:
        out = torch.empty(M, n_out, dtype=torch.float32, device=x.device)
    ws = torch.empty(256, dtype=torch.uint8, device=x.device)
    rc = lib.acmil_linear_f16x3(x.data_ptr(), _DT[x.dtype], M, K, x.stride(0), packed.data_ptr(), n_out, _ptr(bias), int(relu),
                                float(beta), out.data_ptr(), out.stride(0), ws.data_ptr(), _stream())
    _lib.check(rc, "acmil_linear_f16x3")
    return (out, ws[8:12].view(torch.int32)) if want_status else out



# ---------------------------------------------------------------------------------------------------------------------
# 16-bit linear layer with a fused epilogue, gated feed-forward block (csrc/mm16*.hip)
# ---------------------------------------------------------------------------------------------------------------------
_HALF = (torch.float16, torch.bfloat16)
_MAX_ROWS, _MAX_DIM, _MAX_LD = 1 << 30, 1 << 22, 1 << 22
_NO_WORKSPACE_ROWS = 4     # acmil_linear_act of at most so many rows takes no workspace


def _half_inputs(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """One CUDA device and one 16-bit type for every tensor of the call."""
    dt, dev = first.dtype, first.device
    for t in others:
        if t is not None and (t.dtype != dt or t.device != dev):
            _need_cuda(first, t)
            raise RuntimeError("acmil_amd.%s: all tensors must have one type and one device (%s on %s and %s on %s)" % (name, dt, dev, t.dtype, t.device))
    if dev.type != "cuda" or dt not in _HALF:
        _need_cuda(first)
        raise RuntimeError("acmil_amd.%s: fp16 or bf16 tensors (got %s); fp32 layers are acmil_amd.autograd.linear / ops.linear_f16x3" % (name, dt))
    return dev


def _act_id(name: str, act: str) -> int:
    if act not in _lib.ACTS:
        raise ValueError("acmil_amd.%s: act must be one of %s, got %r" % (name, ", ".join(_lib.ACTS), act))
    return _lib.ACTS[act]


def _rows16(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """t [..., C] as a matrix the library can address: (2-D tensor with unit inner stride, leading dimension).  Row strides are kept
    (0 = every row the same); anything else -- a strided inner dimension, overlapping rows -- is copied once."""
    if t.dim() != 2:
        t = t.detach().reshape(-1, t.shape[-1])
    rows, c = t.shape
    ld, inner = t.stride()
    if rows <= 1:
        ld = c
    if (inner == 1 or c == 1) and (ld >= c or ld == 0) and ld <= _MAX_LD:
        return t, ld
    return t.detach().contiguous(), c


def _vec16(name: str, what: str, t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError("acmil_amd.%s: %s must be [%d], got %s" % (name, what, n, tuple(t.shape)))
    return t if t.stride(0) == 1 else t.detach().contiguous()


def _half_call(lib, name: str, args, device: torch.device, may_need: bool = True) -> None:
    """Workspace query + call of a C entry that takes one argument block, on the tensors' device and its current stream."""
    if device.index != torch._C._cuda_getDevice():
        with torch.cuda.device(device):
            return _half_call(lib, name, args, device, may_need)
    ref, ws, need = ctypes.byref(args), None, 0
    if may_need:
        need = getattr(lib, name + "_workspace_bytes")(ref)
        if need == 0:
            raise RuntimeError("%s: the arguments are refused (a dimension or leading dimension is out of range)" % name)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.check(getattr(lib, name)(ref, None if ws is None else ws.data_ptr(), need, torch._C._cuda_getCurrentRawStream(device.index)), name)


def _linear_args(name: str, x: torch.Tensor, weight: torch.Tensor, act: str):
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise RuntimeError("acmil_amd.%s: x [..., in] and weight [out, in] expected, got %s and %s" % (name, tuple(x.shape), tuple(weight.shape)))
    N, K = weight.shape
    x2, ldx = _rows16(x)
    w2, ldw = _rows16(weight)
    M = x2.shape[0]
    if N > _MAX_DIM or K > _MAX_DIM or M > _MAX_ROWS:
        raise RuntimeError("acmil_amd.%s: at most %d features and %d rows" % (name, _MAX_DIM, _MAX_ROWS))
    return _lib.LinearArgs(_DT[x.dtype], _act_id(name, act), M, K, N, x2.data_ptr(), ldx, w2.data_ptr(), ldw), x2, w2


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act: str = "none",
               residual: Optional[torch.Tensor] = None, keep_pre: bool = False):
    """acmil_linear_act: y = act(x @ weight^T + bias) + residual, fp16 or bf16 (fp32 accumulation and epilogue, one rounding at the end).  Bias,
    activation and residual take no pass over the output of their own; sizes and alignment decide whether there are launches beside the
    product's (a copy of operands that do not lie on 16 bytes, a split K with its join, the last rows as a product of their own).
    x [..., in], weight [out, in], bias [out], residual [..., out]; act one of none, relu, silu, gelu, gelu_tanh, sigmoid.  Any row strides and sizes; no rows give an empty result.  keep_pre: also x @ weight^T + bias in fp32
    ([rows, round8(out)]), what linear_act_bwd wants.  No gradient is recorded (acmil_amd.autograd.linear_act is the differentiable form)."""
    dev = _half_inputs("linear_act", x, weight, bias, residual)
    a, x2, w2 = _linear_args("linear_act", x, weight, act)
    M, N = a.M, a.N
    shape = x.shape[:-1] + (N,)
    b = _vec16("linear_act", "bias", bias, N)
    if residual is not None and residual.shape != shape:
        raise RuntimeError("acmil_amd.linear_act: residual must be %s, got %s" % (tuple(shape), tuple(residual.shape)))
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    pre = torch.empty(M, (N + 7) // 8 * 8, dtype=torch.float32, device=dev) if keep_pre else None
    if M > 0:
        a.y, a.ldy = y.data_ptr(), N
        if b is not None:
            a.bias = b.data_ptr()
        if keep_pre:
            a.pre = pre.data_ptr()
        if residual is not None:
            r2, a.ldr = _rows16(residual)
            a.res = r2.data_ptr()
        _half_call(_lib.load(), "acmil_linear_act", a, dev, may_need=M > _NO_WORKSPACE_ROWS)
    return (y, pre) if keep_pre else y


def linear_act_bwd(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, pre: Optional[torch.Tensor] = None, act: str = "none",
                   need: Sequence[bool] = (True, True, True)):
    """acmil_linear_act_bwd: (dx, dweight, dbias) of linear_act for the incoming dy [..., out] and the kept `pre` (act "none" needs none);
    need = which of the three to form (None in the others' places).  dz = dy act'(pre) is held in the tensors' type between the passes (in fp16, beyond
    65504 it is infinite and below 2^-25 zero: scale the loss accordingly).  The residual's gradient is dy."""
    dev = _half_inputs("linear_act_bwd", x, weight, dy)
    a, x2, w2 = _linear_args("linear_act_bwd", x, weight, act)
    if tuple(dy.shape) != tuple(x.shape[:-1]) + (a.N,):
        raise RuntimeError("acmil_amd.linear_act_bwd: dy must be %s, got %s" % (tuple(x.shape[:-1]) + (a.N,), tuple(dy.shape)))
    if act != "none" and (pre is None or pre.dtype != torch.float32 or pre.device != dev or not pre.is_contiguous()
                          or tuple(pre.shape) != (a.M, (a.N + 7) // 8 * 8)):
        raise RuntimeError("acmil_amd.linear_act_bwd: act %r needs the pre-activations linear_act(keep_pre=True) returned" % act)
    make = torch.empty if a.M > 0 else torch.zeros
    dx = make(x.shape, dtype=x.dtype, device=dev) if need[0] else None
    dw = make(weight.shape, dtype=x.dtype, device=dev) if need[1] else None
    db = make(a.N, dtype=x.dtype, device=dev) if need[2] else None
    if a.M > 0 and any(need):
        dy2, a.lddy = _rows16(dy)
        a.dy, a.pre, a.dx, a.dW, a.db = dy2.data_ptr(), _ptr(pre), _ptr(dx), _ptr(dw), _ptr(db)
        _half_call(_lib.load(), "acmil_linear_act_bwd", a, dev)
    return dx, dw, db


def _ffn_args(name: str, x, w_gate, w_up, w_down, act: str):
    if (w_gate.dim() != 2 or x.dim() < 1 or x.shape[-1] != w_gate.shape[1] or w_up.shape != w_gate.shape
            or tuple(w_down.shape) != (w_gate.shape[1], w_gate.shape[0]) or 0 in w_gate.shape):
        raise RuntimeError("acmil_amd.%s: x [..., D], w_gate and w_up [F, D], w_down [D, F] expected, got %s, %s, %s, %s"
                           % (name, tuple(x.shape), tuple(w_gate.shape), tuple(w_up.shape), tuple(w_down.shape)))
    F, D = w_gate.shape
    x2, ldx = _rows16(x)
    g2, ldg = _rows16(w_gate)
    u2, ldu = _rows16(w_up)
    d2, ldd = _rows16(w_down)
    M = x2.shape[0]
    if D > _MAX_DIM or F > _MAX_DIM // 2 or M > _MAX_ROWS:
        raise RuntimeError("acmil_amd.%s: at most %d features, %d hidden features and %d rows" % (name, _MAX_DIM, _MAX_DIM // 2, _MAX_ROWS))
    return _lib.FfnArgs(_DT[x.dtype], _act_id(name, act), M, D, F, x2.data_ptr(), ldx, g2.data_ptr(), ldg, u2.data_ptr(), ldu, d2.data_ptr(),
                        ldd), (x2, g2, u2, d2)


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, b_gate: Optional[torch.Tensor] = None,
              b_up: Optional[torch.Tensor] = None, b_down: Optional[torch.Tensor] = None, act: str = "silu",
              residual: Optional[torch.Tensor] = None, keep: bool = False):
    """acmil_gated_ffn: y = (act(x @ w_gate^T + b_gate) * (x @ w_up^T + b_up)) @ w_down^T + b_down + residual, fp16 or bf16, in two products:
    both projections with the activation and the gate, then the projection back with bias and residual (launches beside them as in linear_act).
    x [..., D], w_gate and w_up [F, D], w_down [D, F], residual [..., D]; act as linear_act ("silu" is the SwiGLU block, "gelu" GeGLU, "sigmoid" GLU, ...).
    The gated features between the launches are held in x's type (in fp16, beyond 65504 they are infinite).  keep: also (g, u, h) for
    gated_ffn_bwd (g, u fp32 and h, each [rows, round8(F)]).  No gradient is recorded (acmil_amd.autograd.gated_ffn is the differentiable form)."""
    dev = _half_inputs("gated_ffn", x, w_gate, w_up, w_down, b_gate, b_up, b_down, residual)
    a, hold = _ffn_args("gated_ffn", x, w_gate, w_up, w_down, act)
    bg, bu, bd = _vec16("gated_ffn", "b_gate", b_gate, a.F), _vec16("gated_ffn", "b_up", b_up, a.F), _vec16("gated_ffn", "b_down", b_down, a.D)
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError("acmil_amd.gated_ffn: residual must be %s, got %s" % (tuple(x.shape), tuple(residual.shape)))
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    saved = None
    if keep:
        f8 = (a.F + 7) // 8 * 8
        saved = (torch.empty(a.M, f8, dtype=torch.float32, device=dev), torch.empty(a.M, f8, dtype=torch.float32, device=dev),
                 torch.empty(a.M, f8, dtype=x.dtype, device=dev))
        a.g, a.u, a.h = (t.data_ptr() for t in saved)
    if a.M > 0:
        a.y, a.ldy = y.data_ptr(), a.D
        if bg is not None or bu is not None or bd is not None:
            a.bg, a.bu, a.bd = _ptr(bg), _ptr(bu), _ptr(bd)
        if residual is not None:
            r2, a.ldr = _rows16(residual)
            a.res = r2.data_ptr()
        _half_call(_lib.load(), "acmil_gated_ffn", a, dev)
    return (y, saved) if keep else y


def gated_ffn_bwd(dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, saved,
                  act: str = "silu", need_x: bool = True, need_gate_up: bool = True, need_down: bool = True, need_gate_up_bias: bool = False,
                  need_down_bias: bool = False):
    """acmil_gated_ffn_bwd: (dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down) of gated_ffn for the incoming dy [..., D] and what
    gated_ffn(keep=True) kept; None where not asked for.  dw_gate / dw_up and db_gate / db_up are views of one buffer each.  The gradients of both
    projections are held in the tensors' type between the products (in fp16, beyond 65504 infinite and below 2^-25 zero).  The residual's gradient
    is dy."""
    dev = _half_inputs("gated_ffn_bwd", x, w_gate, w_up, w_down, dy)
    a, hold = _ffn_args("gated_ffn_bwd", x, w_gate, w_up, w_down, act)
    if dy.shape != x.shape:
        raise RuntimeError("acmil_amd.gated_ffn_bwd: dy must be %s, got %s" % (tuple(x.shape), tuple(dy.shape)))
    f8 = (a.F + 7) // 8 * 8
    g, u, h = saved
    for t, dt in ((g, torch.float32), (u, torch.float32), (h, x.dtype)):
        if t.dtype != dt or t.device != dev or not t.is_contiguous() or tuple(t.shape) != (a.M, f8):
            raise RuntimeError("acmil_amd.gated_ffn_bwd: saved must be what gated_ffn(keep=True) returned for this x")
    make = torch.empty if a.M > 0 else torch.zeros
    dx = make(x.shape, dtype=x.dtype, device=dev) if need_x else None
    dgu = make(2 * f8, a.D, dtype=x.dtype, device=dev) if need_gate_up else None
    dd = make(a.D, a.F, dtype=x.dtype, device=dev) if need_down else None
    bgu = make(2 * f8, dtype=x.dtype, device=dev) if need_gate_up_bias else None
    bd = make(a.D, dtype=x.dtype, device=dev) if need_down_bias else None
    if a.M > 0:
        dy2, a.lddy = _rows16(dy)
        a.dy, a.g, a.u, a.h = dy2.data_ptr(), g.data_ptr(), u.data_ptr(), h.data_ptr()
        a.dx, a.dWgu, a.dWd, a.dbgu, a.dbd = _ptr(dx), _ptr(dgu), _ptr(dd), _ptr(bgu), _ptr(bd)
        _half_call(_lib.load(), "acmil_gated_ffn_bwd", a, dev)
    F = a.F
    return (dx, None if dgu is None else dgu[:F], None if dgu is None else dgu[f8:f8 + F], dd,
            None if bgu is None else bgu[:F], None if bgu is None else bgu[f8:f8 + F], bd)


def _no_overlap(gs, outs) -> None:
    """Nothing is written that another matrix of an orthogonalize call reads or writes; g[i] and out[i] may be the same memory."""
    spans = []
    for i, (g, o) in enumerate(zip(gs, outs)):
        if g.numel():
            end = 1 + sum((n - 1) * s for n, s in zip(g.shape, g.stride()))
            own = (g.data_ptr(), g.data_ptr() + end * g.element_size())
            to = (o.data_ptr(), o.data_ptr() + o.numel() * o.element_size())
            if own != to or not g.is_contiguous():
                spans.append(own + (False,))
            spans.append(to + (True,))
    reach = written = 0                                            # ends of what lies in front: of everything, of the outputs
    for start, end, write in sorted(spans):
        if start < (reach if write else written):
            raise RuntimeError("acmil_amd.orthogonalize: out overlaps another matrix of the call")
        reach = max(reach, end)
        written = max(written, end if write else 0)


NS_COEFFS = (3.4445, -4.7750, 2.0315)      # drives singular values from [0.002, 1] into [0.68, 1.14] in 5 steps
MAX_ORTHO_DIM, MAX_ORTHO_STEPS = 1 << 16, 64


def orthogonalize(g, steps: int = 5, coeffs: Sequence = NS_COEFFS, eps: float = 1e-7, out=None):
    """acmil_orthogonalize: the Newton-Schulz approximation of the orthogonal factor of each matrix (U V^T of G = U S V^T): X = G / (|G|_F + eps),
    then `steps` times X <- a X + (b A + c A A) X with A = X X^T, on the transpose where a matrix is tall.
    g: [m, n], a stack [..., m, n], or a list of [m, n] of any shapes (one type and device): all matrices share the launches.  fp32, fp16 or bf16,
    returned in the same type and structure; inside, whatever the type, values are held to 2^-22 of themselves and 2^-37 of |G|_F.  coeffs: one
    (a, b, c) or one per step.  The same list gives the same bits; beside other matrices one may differ in its last.  No gradient is recorded.
    out: contiguous tensor(s) of g's structure, type and shapes to write to; a matrix may be its own output, other overlaps are refused."""
    lib = _lib.load()
    many = isinstance(g, (list, tuple))
    ts = list(g) if many else [g]
    if not ts:
        return []
    _need_cuda(*ts)
    dev, dt = ts[0].device, ts[0].dtype
    if dt not in _DT or any(t.dtype != dt or t.device != dev for t in ts):
        raise RuntimeError("acmil_amd.orthogonalize: fp32, fp16 or bf16 matrices of one type and one device")
    if any(t.dim() != 2 for t in ts) if many else g.dim() < 2:
        raise RuntimeError("acmil_amd.orthogonalize: [m, n], a stack [..., m, n] or a list of [m, n] expected")
    table = [float(c) for c in coeffs] * steps if not isinstance(coeffs[0], (list, tuple)) else [float(c) for s in coeffs for c in s]
    if steps < 1 or len(table) != 3 * steps:
        raise ValueError("acmil_amd.orthogonalize: coeffs must be (a, b, c) or one (a, b, c) for each of the steps")
    outs = [torch.empty(t.shape, dtype=dt, device=dev) for t in ts] if out is None else list(out) if many else [out]
    if out is not None and (len(outs) != len(ts) or any(o.shape != t.shape or o.dtype != dt or o.device != dev or not o.is_contiguous()
                                                       for o, t in zip(outs, ts))):
        raise RuntimeError("acmil_amd.orthogonalize: out must be contiguous tensors of g's structure, type and shapes")
    if out is not None:
        _no_overlap(ts, outs)
    mats, hold = [], []
    for t, o in zip(ts, outs):
        if t.numel() == 0:
            continue
        m, n = t.shape[-2:]
        t = t.detach()
        t = t.reshape(-1, m, n) if t.dim() != 3 else t
        if (n > 1 and t.stride(2) != 1) or (m > 1 and t.stride(1) < n):
            t = t.contiguous()
        hold.append(t)
        size = t.element_size()
        ld = t.stride(1) if m > 1 else n
        for k in range(t.shape[0]):
            mats.append(_lib.OrthoMat(t.data_ptr() + k * t.stride(0) * size, ld, o.data_ptr() + k * m * n * size, n, m, n))
    if mats:
        with torch.cuda.device(dev):
            arr, co = (_lib.OrthoMat * len(mats))(*mats), (ctypes.c_float * len(table))(*table)
            need = lib.acmil_orthogonalize_workspace_bytes(len(mats), arr, _DT[dt])
            if need == 0:
                raise RuntimeError("acmil_amd.orthogonalize: matrices of at most %d rows and columns" % MAX_ORTHO_DIM)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            _lib.check(lib.acmil_orthogonalize(len(mats), arr, _DT[dt], steps, co, float(eps), ws.data_ptr(), need, _stream()), "acmil_orthogonalize")
    return outs if many else outs[0]
