"""The bolt ops on torch CUDA tensors -- a host-side mirror of the reference's ORT ops.

Each function is one node of the reference's custom-op domain ``bolt`` (src/bolt_ops.cu:1469-1589):
same name, inputs in the same order, same attributes, and outputs allocated in the shapes the
reference's ``ComputeV2`` allocates.  The work runs on the current torch CUDA stream through
libbolt_b200.so; there is no CPU path.  A failing shape check raises ``RuntimeError`` with the
reference's message (the reference returns ORT_FAIL with the same text).
"""
from __future__ import annotations

import ctypes
import threading

import torch

from ._lib import last_error, lib, shape_arg

__all__ = ["Nvfp4Gemv", "Q8Gemv", "Q4Gemv", "MoeRoute", "MoeDecode", "MoeVerify", "moe_verify_shard",
           "KvAppend", "KvRead", "KvAttention", "KvScore", "KvEvict", "KV_INT8", "KV_E4M3",
           "f32_to_bf16", "copy_async", "dequant", "set_launch_options", "device_status", "FMT_Q8", "FMT_Q4", "FMT_NVFP4",
           "FMT_IQ2_LUT", "FMT_IQ2_NATIVE"]

FMT_Q8, FMT_Q4, FMT_NVFP4, FMT_IQ2_LUT, FMT_IQ2_NATIVE = 0, 1, 2, 3, 4
KV_INT8, KV_E4M3 = 0, 1


def _ptr(t):
    # plain ints: ctypes converts them for c_void_p parameters without a wrapper object per call
    return t.data_ptr() if t is not None else None


def _stream(t):
    # the raw cudaStream_t of torch's current stream on t's device (as current_stream().cuda_stream)
    return torch._C._cuda_getCurrentRawStream(t.device.index)


def _need(*tensors):
    for t in tensors:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise RuntimeError("bolt ops take CUDA tensors (there is no CPU implementation)")
        if not t.is_contiguous():
            raise RuntimeError("bolt ops take contiguous tensors")


def _check(rc):
    if rc != 0:
        raise RuntimeError(last_error())


def set_launch_options(pdl: bool = True, early_weights: bool = False, smem_budget: int = 0) -> None:
    """Process-wide launch options (see bolt_set_launch_options in include/bolt_b200.h); the
    defaults are the library's own (programmatic dependent launch on, early weights off)."""
    _check(lib().bolt_set_launch_options(int(pdl), int(early_weights), int(smem_budget)))


def device_status() -> int:
    """Read and clear the device status word of the current device (0 = no kernel gave up)."""
    v = ctypes.c_uint(0)
    _check(lib().bolt_get_device_status(ctypes.byref(v)))
    return v.value


def Nvfp4Gemv(x, w, w_scale, g):
    """y[..., N] = bf16(g * x @ (e2m1 * e4m3)^T); w u8 [N, K/2], w_scale u8 [N, K/16], g f32 [1]."""
    _need(x, w, w_scale, g)
    y = torch.empty(*x.shape[:-1], w.shape[0], dtype=torch.bfloat16, device=x.device)
    xs, _k1 = shape_arg(x.shape)
    ws, _k2 = shape_arg(w.shape)
    _check(lib().bolt_nvfp4_gemv(_ptr(x), xs, x.dim(), _ptr(w), ws, w.dim(), _ptr(w_scale), _ptr(g), _ptr(y),
                                 _stream(x)))
    return y


def Q8Gemv(x, B, scales):
    """y[..., N] = x @ W^T, W = (B - 128) * s; B u8 [N, K/32, 32], scales bf16 [N, K/32]."""
    _need(x, B, scales)
    y = torch.empty(*x.shape[:-1], B.shape[0], dtype=torch.bfloat16, device=x.device)
    xs, _k1 = shape_arg(x.shape)
    bs, _k2 = shape_arg(B.shape)
    _check(lib().bolt_q8_gemv(_ptr(x), xs, x.dim(), _ptr(B), bs, B.dim(), _ptr(scales), _ptr(y), _stream(x)))
    return y


def Q4Gemv(x, B, scales, iq2: int = 0):
    """int4 (iq2=0), IQ2_XXS LUT codes (iq2=1) or native IQ2_XXS records (iq2=2)."""
    _need(x, B, scales)
    y = torch.empty(*x.shape[:-1], B.shape[0], dtype=torch.bfloat16, device=x.device)
    xs, _k1 = shape_arg(x.shape)
    bs, _k2 = shape_arg(B.shape)
    _check(lib().bolt_q4_gemv(_ptr(x), xs, x.dim(), _ptr(B), bs, B.dim(), _ptr(scales), int(iq2), _ptr(y),
                              _stream(x)))
    return y


def MoeRoute(x, gate_w, bias, topk: int, scale: float):
    """Returns (idx i32 [R, topk], w f32 [R, topk], scores f32 [R, E])."""
    _need(x, gate_w, bias)
    R, E = x.shape[0], gate_w.shape[0]
    idx = torch.empty(R, topk, dtype=torch.int32, device=x.device)
    w = torch.empty(R, topk, dtype=torch.float32, device=x.device)
    scores = torch.empty(R, E, dtype=torch.float32, device=x.device)
    xs, _k1 = shape_arg(x.shape)
    gs, _k2 = shape_arg(gate_w.shape)
    _check(lib().bolt_moe_route(_ptr(x), xs, x.dim(), _ptr(gate_w), gs, gate_w.dim(), _ptr(bias), int(topk),
                                float(scale), _ptr(idx), _ptr(w), _ptr(scores), _stream(x)))
    return idx, w, scores


def _moe_outputs(z, fc1_w, topk):
    R = z.shape[0]
    I = fc1_w.shape[1]
    P = R * topk
    out = torch.empty(R, 1024, dtype=torch.bfloat16, device=z.device)
    h = torch.empty(P, I, dtype=torch.bfloat16, device=z.device)
    part = torch.empty(P, 1024, dtype=torch.float32, device=z.device)
    return out, h, part


def MoeDecode(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk: int):
    """Returns (out bf16 [R, 1024], h bf16 [R*topk, I], part f32 [R*topk, 1024])."""
    _need(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s)
    out, h, part = _moe_outputs(z, fc1_w, topk)
    zs, _k1 = shape_arg(z.shape)
    w1s, _k2 = shape_arg(fc1_w.shape)
    _check(lib().bolt_moe_decode(_ptr(z), zs, z.dim(), _ptr(idx), _ptr(w), _ptr(fc1_w), w1s, fc1_w.dim(),
                                 _ptr(fc1_s), _ptr(fc2_w), _ptr(fc2_s), int(topk), _ptr(out), _ptr(h), _ptr(part),
                                 _stream(z)))
    return out, h, part


def MoeVerify(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk: int, iq2: int = 0):
    """Returns (out, h, part, meta i32 [1 + P + 8P])."""
    _need(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s)
    out, h, part = _moe_outputs(z, fc1_w, topk)
    P = z.shape[0] * topk
    meta = torch.empty(1 + P + 8 * P, dtype=torch.int32, device=z.device)
    zs, _k1 = shape_arg(z.shape)
    w1s, _k2 = shape_arg(fc1_w.shape)
    _check(lib().bolt_moe_verify(_ptr(z), zs, z.dim(), _ptr(idx), _ptr(w), _ptr(fc1_w), w1s, fc1_w.dim(),
                                 _ptr(fc1_s), _ptr(fc2_w), _ptr(fc2_s), int(topk), int(iq2), _ptr(out), _ptr(h),
                                 _ptr(part), _ptr(meta), _stream(z)))
    return out, h, part, meta


def _expert_ptr(t, e_begin: int):
    """Device address of expert 0 for a tensor holding experts [e_begin, ...) only (the kernels
    read experts >= e_begin exclusively, so the shifted base is never dereferenced below them)."""
    return ctypes.c_void_p(t.data_ptr() - int(e_begin) * t[0].numel() * t.element_size())


def moe_verify_shard(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk: int, iq2: int, e_begin: int, e_end: int,
                     num_experts: int = None, out_partial=None, outputs=None):
    """MoeVerify over experts [e_begin, e_end) only; returns (out_partial f32 [R, 1024], h, part, meta).

    The weight tensors hold either all ``num_experts`` experts, or only the local experts
    [e_begin, e_end) (then ``num_experts`` gives the global count).  Rows of h / part of
    non-local pairs are left untouched.
    """
    _need(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s)
    R = z.shape[0]
    P = R * topk
    E = int(num_experts) if num_experts is not None else fc1_w.shape[0]
    local = fc1_w.shape[0] != E
    if local and fc1_w.shape[0] != e_end - e_begin:
        raise RuntimeError("moe_verify_shard: local weights must hold exactly experts [e_begin, e_end)")
    if outputs is None:
        _, h, part = _moe_outputs(z, fc1_w, topk)
        meta = torch.empty(1 + P + 8 * P, dtype=torch.int32, device=z.device)
    else:
        h, part, meta = outputs
    if out_partial is None:
        out_partial = torch.empty(R, 1024, dtype=torch.float32, device=z.device)
    zs, _k1 = shape_arg(z.shape)
    w1s, _k2 = shape_arg((E,) + tuple(fc1_w.shape[1:]))
    wp = [_expert_ptr(t, e_begin) if local else _ptr(t) for t in (fc1_w, fc1_s, fc2_w, fc2_s)]
    _check(lib().bolt_moe_verify_shard(_ptr(z), zs, z.dim(), _ptr(idx), _ptr(w), wp[0], w1s, fc1_w.dim(),
                                       wp[1], wp[2], wp[3], int(topk), int(iq2), int(e_begin), int(e_end),
                                       ctypes.c_void_p(0), _ptr(h), _ptr(part), _ptr(meta), _ptr(out_partial),
                                       _stream(z)))
    return out_partial, h, part, meta


def moe_verify_shard_allreduce(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk: int, iq2: int, e_begin: int,
                               e_end: int, reducer, num_experts: int = None, out=None, outputs=None):
    """Expert-sharded MoeVerify whose last kernel also sums every rank's partial through peer
    memory (``reducer``: a :class:`nemotron_ops_b200.sharded.PeerReducer`); returns out bf16
    [R, 1024], identical on every rank.  Weights and ``outputs`` as for :func:`moe_verify_shard`."""
    _need(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s)
    R = z.shape[0]
    P = R * topk
    E = int(num_experts) if num_experts is not None else fc1_w.shape[0]
    local = fc1_w.shape[0] != E
    if local and fc1_w.shape[0] != e_end - e_begin:
        raise RuntimeError("moe_verify_shard_allreduce: local weights must hold exactly experts [e_begin, e_end)")
    if outputs is None:
        _, h, part = _moe_outputs(z, fc1_w, topk)
        meta = torch.empty(1 + P + 8 * P, dtype=torch.int32, device=z.device)
    else:
        h, part, meta = outputs
    if out is None:
        out = torch.empty(R, 1024, dtype=torch.bfloat16, device=z.device)
    zs, _k1 = shape_arg(z.shape)
    w1s, _k2 = shape_arg((E,) + tuple(fc1_w.shape[1:]))
    wp = [_expert_ptr(t, e_begin) if local else _ptr(t) for t in (fc1_w, fc1_s, fc2_w, fc2_s)]
    _check(lib().bolt_moe_verify_shard_allreduce(
        _ptr(z), zs, z.dim(), _ptr(idx), _ptr(w), wp[0], w1s, fc1_w.dim(), wp[1], wp[2], wp[3], int(topk), int(iq2),
        int(e_begin), int(e_end), _ptr(h), _ptr(part), _ptr(meta), ctypes.c_void_p(reducer.bufs_dev),
        _ptr(reducer.counters), int(reducer.half), int(reducer.rank), int(reducer.world), _ptr(out), _stream(z)))
    return out


def moe_decode_shard(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s, topk: int, e_begin: int, e_end: int,
                     num_experts: int = None, out_partial=None, outputs=None):
    """MoeDecode over experts [e_begin, e_end) only; returns (out_partial f32 [R, 1024], h, part).

    Weight tensors as for :func:`moe_verify_shard` (all experts, or only the local ones with
    ``num_experts`` giving the global count).  Requires I % 256 == 0.
    """
    _need(z, idx, w, fc1_w, fc1_s, fc2_w, fc2_s)
    R = z.shape[0]
    E = int(num_experts) if num_experts is not None else fc1_w.shape[0]
    local = fc1_w.shape[0] != E
    if local and fc1_w.shape[0] != e_end - e_begin:
        raise RuntimeError("moe_decode_shard: local weights must hold exactly experts [e_begin, e_end)")
    if outputs is None:
        _, h, part = _moe_outputs(z, fc1_w, topk)
    else:
        h, part = outputs
    if out_partial is None:
        out_partial = torch.empty(R, 1024, dtype=torch.float32, device=z.device)
    zs, _k1 = shape_arg(z.shape)
    w1s, _k2 = shape_arg((E,) + tuple(fc1_w.shape[1:]))
    wp = [_expert_ptr(t, e_begin) if local else _ptr(t) for t in (fc1_w, fc1_s, fc2_w, fc2_s)]
    _check(lib().bolt_moe_decode_shard(_ptr(z), zs, z.dim(), _ptr(idx), _ptr(w), wp[0], w1s, fc1_w.dim(),
                                       wp[1], wp[2], wp[3], int(topk), int(e_begin), int(e_end), ctypes.c_void_p(0),
                                       _ptr(h), _ptr(part), _ptr(out_partial), _stream(z)))
    return out_partial, h, part


def _mamba(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, sel, heads, head_dim,
           d_state, n_groups, epsilon, time_step_min):
    tensors = [proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w]
    _need(*tensors + ([sel] if sel is not None else []))
    R = proj.shape[0]
    di = heads * head_dim
    cd = di + 2 * n_groups * d_state
    dev = proj.device
    y = torch.empty(R, di, dtype=torch.bfloat16, device=dev)
    conv_out = torch.empty_like(conv_state)
    ssm_out = torch.empty_like(ssm_state)
    xbc = torch.empty(R, cd, dtype=torch.bfloat16, device=dev)
    ypre = torch.empty(R, di, dtype=torch.float32, device=dev)
    ps, _k1 = shape_arg(proj.shape)
    cs, _k2 = shape_arg(conv_state.shape)
    ss, _k3 = shape_arg(ssm_state.shape)
    head = [_ptr(proj), ps, proj.dim(), _ptr(conv_state), cs, conv_state.dim(), _ptr(ssm_state), ss,
            ssm_state.dim()] + [_ptr(t) for t in tensors[3:]]
    tail = [int(heads), int(head_dim), int(d_state), int(n_groups), float(epsilon), float(time_step_min), _ptr(y),
            _ptr(conv_out), _ptr(ssm_out), _ptr(xbc), _ptr(ypre), _stream(proj)]
    if sel is None:
        _check(lib().bolt_mamba_step(*head, *tail))
    else:
        _check(lib().bolt_mamba_verify(*head, _ptr(sel), *tail))
    return y, conv_out, ssm_out, xbc, ypre


def MambaStep(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, heads: int,
              head_dim: int, d_state: int, n_groups: int, epsilon: float, time_step_min: float):
    """Returns (y bf16 [R, di], conv_state_out, ssm_state_out, xbc_act bf16 [R, cd], ypre f32 [R, di])
    (src/bolt_ops.cu:299-357); the state outputs are shaped like the inputs, row 0 written."""
    return _mamba(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, None, heads, head_dim,
                  d_state, n_groups, epsilon, time_step_min)


def MambaVerify(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, sel, heads: int,
                head_dim: int, d_state: int, n_groups: int, epsilon: float, time_step_min: float):
    """As MambaStep from state row sel (i32 [1] on the device); the state after token r goes to
    row r of the state outputs (rows >= R only are left unwritten)."""
    return _mamba(proj, conv_state, ssm_state, conv_w, conv_b, dt_bias, a_neg, d_skip, norm_w, sel, heads, head_dim,
                  d_state, n_groups, epsilon, time_step_min)


def Relu2(x):
    """Returns y bf16 of x's shape, bf16(max(x, 0)^2) (src/bolt_ops.cu:624-646)."""
    _need(x)
    if x.dtype != torch.bfloat16:
        raise RuntimeError("Relu2 takes bf16")
    y = torch.empty_like(x)
    xs, _keep = shape_arg(x.shape)
    _check(lib().bolt_relu2(_ptr(x), xs, x.dim(), _ptr(y), _stream(x)))
    return y


# ---------------------------------------------------------------------------------------------
# paged 8-bit key/value cache (include/bolt_b200.h has the formulas)
#   k_cache, v_cache u8 [pages, heads, T, D], k_scale, v_scale f32 [pages, heads]
#   table i32 [S, width]: position j of sequence s is slot j % T of page table[s, j // T]
#   start, lens i32 [S]: row r of a call is position start[s] + r, if that is below lens[s]
# ---------------------------------------------------------------------------------------------
def _kv_args(op, k_cache, v_cache, k_scale, v_scale, table, lens, start=None):
    """Checks what the cache ops share; returns the shape arguments of the cache and the page table."""
    start = lens if start is None else start
    try:
        if not (k_cache.is_cuda and v_cache.is_cuda and k_scale.is_cuda and v_scale.is_cuda and table.is_cuda
                and lens.is_cuda and start.is_cuda):
            raise RuntimeError("bolt ops take CUDA tensors (there is no CPU implementation)")
        if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous()
                and v_scale.is_contiguous() and table.is_contiguous() and lens.is_contiguous()
                and start.is_contiguous()):
            raise RuntimeError("bolt ops take contiguous tensors")
    except AttributeError:
        raise RuntimeError("bolt ops take CUDA tensors (there is no CPU implementation)") from None
    if not (k_cache.dtype is v_cache.dtype is torch.uint8 and k_scale.dtype is v_scale.dtype is torch.float32):
        raise RuntimeError(f"{op}: caches are u8, scales f32")
    shape, pages = k_cache.shape, k_scale.shape
    if len(shape) != 4 or v_cache.shape != shape or pages != shape[:2] or v_scale.shape != pages:
        raise RuntimeError(f"{op}: cache must be [pages, heads, tokens, head size], scales [pages, heads]")
    if not (table.dtype is lens.dtype is start.dtype is torch.int32):
        raise RuntimeError(f"{op}: page tables, starts and lengths are i32")
    tables = table.shape
    if len(tables) != 2:
        raise RuntimeError(f"{op}: page table must be [sequences, pages of a sequence]")
    if lens.shape != tables[:1] or start.shape != tables[:1]:
        raise RuntimeError(f"{op}: starts and lengths must be [sequences]")
    # the library launches on the current device, which has to have every tensor
    if not (torch._C._cuda_getDevice() == k_cache.get_device() == v_cache.get_device() == k_scale.get_device()
            == v_scale.get_device() == table.get_device() == lens.get_device() == start.get_device()):
        raise RuntimeError(f"{op}: tensors must be on the current device")
    return shape_arg(shape)[0], shape_arg(tables)[0]


def _kv_rows(op, t, what, cache):
    """Shape argument of rows [S, R, heads, D] whose last two axes are dense, and that of the strides of the
    sequence and row axes.  They are on the cache's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError("bolt ops take CUDA tensors (there is no CPU implementation)")
    if t.dtype != torch.bfloat16 or t.dim() != 4:
        raise RuntimeError(f"{op}: {what} must be bf16 [sequences, rows, heads, head size]")
    if t.get_device() != cache.get_device():
        raise RuntimeError(f"{op}: tensors must be on the current device")
    seq, row, head, one = t.stride()
    S, R, H, D = shape = t.shape
    if (one != 1 and D != 1) or (head != D and H != 1):
        raise RuntimeError(f"{op}: {what} must be dense over its heads and values")
    # an axis of one entry has no step
    return shape_arg(shape)[0], shape_arg((seq if S > 1 else 0, row if R > 1 else 0))[0]


_WORKSPACES = threading.local()


def _kv_workspace(like, nbytes):
    """Scratch memory of a call, whose two kernels meet in it.  The calls that one host thread makes on one
    stream follow one another, kernel by kernel, so they share a tensor (an allocation costs two microseconds).
    Two threads may enqueue their kernels on one stream in turn, so each has its own; and so has a captured
    call, which may be replayed on any stream."""
    if torch.cuda.is_current_stream_capturing():
        return like.new_empty((nbytes,))
    held = _WORKSPACES.__dict__  # this thread's
    key = like.device.index, _stream(like)
    ws = held.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = held[key] = like.new_empty((nbytes,))
    return ws


def KvAppend(k, v, k_cache, v_cache, k_scale, v_scale, table, start, lens, fmt: int = KV_INT8):
    """Quantise the rows k, v bf16 [S, R, heads, D] into their pages, in place: a page's scale grows to
    max|x| / 127 (KV_INT8) or / 448 (KV_E4M3) where a row needs it, and its older codes with it."""
    cs, ts = _kv_args("KvAppend", k_cache, v_cache, k_scale, v_scale, table, lens, start)
    shape, ks = _kv_rows("KvAppend", k, "k", k_cache)
    _, vs = _kv_rows("KvAppend", v, "v", k_cache)
    if v.shape != k.shape:
        raise RuntimeError("KvAppend: k and v must have the same shape")
    _check(lib().bolt_kv_append(_ptr(k), shape, ks, _ptr(v), vs, _ptr(k_cache), cs, _ptr(v_cache), _ptr(k_scale),
                                _ptr(v_scale), _ptr(table), ts, _ptr(start), _ptr(lens), int(fmt), _stream(k_cache)))


def KvRead(k_cache, v_cache, k_scale, v_scale, table, start, lens, rows: int, fmt: int = KV_INT8):
    """Returns (k, v) bf16 [S, rows, heads, D]: what the cache holds of the positions from start on, 0 from
    lens on."""
    cs, ts = _kv_args("KvRead", k_cache, v_cache, k_scale, v_scale, table, lens, start)
    k = k_cache.new_empty((table.shape[0], rows, k_cache.shape[1], k_cache.shape[3]), dtype=torch.bfloat16)
    v = torch.empty_like(k)
    _check(lib().bolt_kv_read(_ptr(k_cache), cs, _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(table), ts,
                              _ptr(start), _ptr(lens), int(rows), int(fmt), _ptr(k), _ptr(v), _stream(k_cache)))
    return k, v


def KvAttention(q, k_cache, v_cache, k_scale, v_scale, table, start, lens, scale: float, window: int = 0,
                sinks: int = 0, fmt: int = KV_INT8):
    """Returns (o bf16 [S, R, Hq, D], lse f32 [S, R, Hq]) of the rows q bf16 [S, R, Hq, D]: the row at
    position p sees the positions j <= p and, with a window, only j > p - window or j < sinks."""
    cs, ts = _kv_args("KvAttention", k_cache, v_cache, k_scale, v_scale, table, lens, start)
    shape, st = _kv_rows("KvAttention", q, "q", k_cache)
    # new_empty of a tensor of the type: half the host time of torch.empty with a type and a device
    o = q.new_empty(q.shape)
    lse = k_scale.new_empty(q.shape[:3])
    ws = _kv_workspace(k_cache, max(0, lib().bolt_kv_attention_workspace(shape, cs)))
    _check(lib().bolt_kv_attention(_ptr(q), shape, st, _ptr(k_cache), cs, _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
                                   _ptr(table), ts, _ptr(start), _ptr(lens), float(scale), int(window), int(sinks),
                                   int(fmt), _ptr(o), _ptr(lse), _ptr(ws), ws.numel(), _stream(k_cache)))
    return o, lse


def KvScore(q, k_cache, k_scale, table, start, lens, lse, score, scale: float, window: int = 0, sinks: int = 0,
            fmt: int = KV_INT8):
    """Adds every cached position's attention weight to score f32 [S, heads, >= width * T], in place (and
    returns it); q, the mask and lse as in the KvAttention call whose weights are taken."""
    cs, ts = _kv_args("KvScore", k_cache, k_cache, k_scale, k_scale, table, lens, start)
    _need(lse, score)
    if not lse.get_device() == score.get_device() == k_cache.get_device():
        raise RuntimeError("KvScore: tensors must be on the current device")
    shape, st = _kv_rows("KvScore", q, "q", k_cache)
    if lse.dtype != torch.float32 or lse.shape != q.shape[:3]:
        raise RuntimeError("KvScore: lse must be f32 [sequences, rows, query heads]")
    if score.dtype != torch.float32 or score.dim() != 3 or score.shape[:2] != (table.shape[0], k_cache.shape[1]):
        raise RuntimeError("KvScore: score must be f32 [sequences, heads, positions]")
    _check(lib().bolt_kv_score(_ptr(q), shape, st, _ptr(k_cache), cs, _ptr(k_scale), _ptr(table), ts, _ptr(start),
                               _ptr(lens), _ptr(lse), float(scale), int(window), int(sinks), int(fmt), _ptr(score),
                               score.shape[2], _stream(k_cache)))
    return score


def KvEvict(k_cache, v_cache, k_scale, v_scale, table, lens, score, new_table, keep: int, sinks: int = 0,
            recent: int = 0, fmt: int = KV_INT8):
    """Cuts every (sequence, head) to its first `sinks` positions, its last `recent` and those of the largest
    score, `keep` in all, laid out in order in the pages of new_table i32 [S, >= keep / T].  Returns
    (kept i32 [S, heads, keep], new_lens i32 [S], new_score f32 [S, heads, keep])."""
    cs, ts = _kv_args("KvEvict", k_cache, v_cache, k_scale, v_scale, table, lens)
    _need(score, new_table)
    if not score.get_device() == new_table.get_device() == k_cache.get_device():
        raise RuntimeError("KvEvict: tensors must be on the current device")
    S, heads = table.shape[0], k_cache.shape[1]
    if new_table.dtype != torch.int32 or new_table.dim() != 2 or new_table.shape[0] != S:
        raise RuntimeError("KvEvict: the new page table must be i32 [sequences, pages of a sequence]")
    if score.dtype != torch.float32 or score.dim() != 3 or score.shape[:2] != (S, heads):
        raise RuntimeError("KvEvict: score must be f32 [sequences, heads, positions]")
    kept = table.new_empty((S, heads, keep))
    new_lens = torch.empty_like(lens)
    new_score = score.new_empty((S, heads, keep))
    _check(lib().bolt_kv_evict(_ptr(k_cache), cs, _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(table), ts,
                               _ptr(lens), _ptr(score), score.shape[2], _ptr(new_table), new_table.shape[1],
                               int(keep), int(sinks), int(recent), int(fmt), _ptr(kept), _ptr(new_lens),
                               _ptr(new_score), _stream(k_cache)))
    return kept, new_lens, new_score


def f32_to_bf16(t, out=None):
    _need(t)
    if out is None:
        out = torch.empty(t.shape, dtype=torch.bfloat16, device=t.device)
    _check(lib().bolt_f32_to_bf16(_ptr(t), _ptr(out), t.numel(), _stream(t)))
    return out


def copy_async(dst, src):
    """dst <- src between host (pinned for an asynchronous copy) and device memory, ordered on
    the current stream of whichever tensor is on the GPU (one cudaMemcpyAsync)."""
    if dst.nbytes != src.nbytes or not dst.is_contiguous() or not src.is_contiguous():
        raise RuntimeError("copy_async: contiguous tensors of the same byte size")
    _check(lib().bolt_memcpy_async(_ptr(dst), _ptr(src), dst.nbytes, _stream(dst if dst.is_cuda else src)))
    return dst


def dequant(fmt: int, w, scales, N: int, K: int, exact: bool = False):
    """Weights [N, K] f32 decoded by the kernels' own decoders (contract checks)."""
    _need(w, scales)
    out = torch.empty(N, K, dtype=torch.float32, device=w.device)
    _check(lib().bolt_dequant(int(fmt), int(exact), _ptr(w), _ptr(scales), int(N), int(K), _ptr(out), _stream(w)))
    return out
