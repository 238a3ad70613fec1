"""ctypes bindings of libmatvec_hip.so, the MI355X replacement for the reference's FPGA backend.

The library is C (include/matvec_fpga.h: the reference's six-function driver API; include/llm_hip.h: the
device-resident token loop).  These bindings are what the Python tests and bench.py call; the C hosts in
host/ and the reference's own hosts link the library directly.  Nothing here computes: every call goes
through the C ABI, and loading fails loudly when the built library is missing.  The operators on device memory
(kv_write, kv_read, tree_attention, logprobs) take torch tensors; torch is imported by their first call.

The directory name is not a Python identifier, so callers load this file by path, e.g.
    spec = importlib.util.spec_from_file_location("llm_hip", ".../local-llama-pynq-z2_amd/__init__.py")
"""
import ctypes as C
import os
import struct

import numpy as np

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
LIB_PATH = os.path.join(PKG_DIR, "libmatvec_hip.so")
HOST_DIR = os.path.join(PKG_DIR, "host")
MAX_N = 32768

_lib = None


class LlmInfo(C.Structure):
    _fields_ = [("kind", C.c_int), ("dim", C.c_int), ("hidden_dim", C.c_int), ("n_layers", C.c_int),
                ("n_heads", C.c_int), ("n_kv_heads", C.c_int), ("vocab_size", C.c_int), ("n_logits", C.c_int),
                ("ctx", C.c_int), ("group_size", C.c_int), ("rope_theta", C.c_float), ("rms_eps", C.c_float),
                ("gemv_bytes_per_token", C.c_double), ("weight_bytes", C.c_double)]


class LlmKv(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("type", C.c_int), ("n_seq", C.c_int), ("n_kv", C.c_int), ("hs", C.c_int), ("ctx", C.c_int),
                ("seq", C.c_int64), ("head", C.c_int64), ("pos", C.c_int64),
                ("s_seq", C.c_int64), ("s_head", C.c_int64), ("s_pos", C.c_int64)]


class LlmRows(C.Structure):
    _fields_ = [("p", C.c_void_p), ("type", C.c_int), ("seq", C.c_int64), ("tok", C.c_int64), ("head", C.c_int64)]


class LlmTiming(C.Structure):
    _fields_ = [("n_prompt", C.c_int), ("n_generated", C.c_int), ("n_forward", C.c_int),
                ("prompt_ms", C.c_double), ("decode_ms", C.c_double)]


class LlmKernelStat(C.Structure):
    _fields_ = [("name", C.c_char * 40), ("launches", C.c_int), ("total_ms", C.c_double),
                ("bytes_per_launch", C.c_double)]


def build_hint():
    return "build it first: python -c 'import __graft_entry__ as g; g.build()' (or make -C local-llama-pynq-z2_amd)"


def lib():
    """The loaded libmatvec_hip.so, with argument types set.  Raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is missing; {build_hint()}")
    L = C.CDLL(LIB_PATH)
    u64, i32, vp, sz = C.c_uint64, C.c_int, C.c_void_p, C.c_size_t
    L.fpga_open.restype = i32
    L.fpga_alloc.restype = vp
    L.fpga_alloc.argtypes = [sz, C.POINTER(u64)]
    L.fpga_alloc_try.restype = vp
    L.fpga_alloc_try.argtypes = [sz, C.POINTER(u64)]
    L.fpga_matvec.argtypes = [u64, u64, u64, u64, u64, i32, i32, i32]
    L.fpga_matvec.restype = i32
    L.fpga_matvec4.argtypes = [u64, u64, u64, u64, u64, i32, i32, i32]
    L.fpga_matvec4.restype = i32
    L.fpga_close.restype = None
    L.llm_open.restype = vp
    L.llm_open.argtypes = [C.c_char_p, i32]
    L.llm_get_info.argtypes = [vp, C.POINTER(LlmInfo)]
    L.llm_head_ids.restype = C.POINTER(C.c_int32)
    L.llm_head_ids.argtypes = [vp]
    L.llm_forward.argtypes = [vp, i32, i32, vp]
    L.llm_generate.argtypes = [vp, vp, i32, i32, vp, vp, C.POINTER(LlmTiming)]
    L.llm_continue.argtypes = [vp, i32, vp, i32, i32, i32, vp, C.POINTER(LlmTiming)]
    L.llm_decode_replay.argtypes = [vp, i32, C.POINTER(C.c_double)]
    L.llm_profile.argtypes = [vp, i32, C.POINTER(LlmKernelStat), i32]
    L.llm_profile_graph.argtypes = [vp, i32, i32, C.POINTER(LlmKernelStat), i32, C.POINTER(C.c_double)]
    L.llm_prefill.argtypes = [vp, vp, i32, vp]
    L.llm_close.argtypes = [vp]
    L.llm_close.restype = None
    L.llm_read_state.argtypes = [vp, i32, i32, vp, sz]
    L.mvh_quantize.argtypes = [vp, i32, i32, i32, vp, vp]
    L.mvh_group_dots.argtypes = [vp, vp, i32, i32, i32, i32, vp]
    L.mvh_prefill_gemm.argtypes = [vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, i32, vp]
    L.llm_set_prefill.argtypes = [vp, i32]
    L.llm_set_sampler.argtypes = [vp, C.c_float, C.c_float, C.c_ulonglong]
    L.llm_sampler_state.argtypes = [vp, C.POINTER(C.c_ulonglong)]
    L.mvh_sample.argtypes = [vp, i32, i32, C.c_float, C.c_float, C.POINTER(C.c_ulonglong), vp]
    L.mvh_sample_noalloc.argtypes = [vp, i32, i32, C.c_float, C.c_float, C.POINTER(C.c_ulonglong), vp]
    L.mvh_sample_strict.argtypes = [vp, i32, i32, C.c_float, C.c_float, C.POINTER(C.c_ulonglong), vp]
    L.mvh_sample_strict_skew.argtypes = [vp, i32, i32, C.c_float, C.c_float, C.POINTER(C.c_ulonglong), vp, i32]
    L.mvh_ref_expf.argtypes = [vp, i32, vp]
    L.mvh_read_floor.argtypes = [C.c_size_t, i32, i32, i32, i32, C.POINTER(C.c_float)]
    L.mvh_ref_expf_host.argtypes = [vp, i32, vp]
    L.mvh_seq_sum.argtypes = [vp, i32, i32, i32, vp]
    L.llm_set_kv.argtypes = [vp, i32]
    L.llm_get_kv.argtypes = [vp]
    L.llm_verify.argtypes = [vp, i32, vp, vp, i32, vp, vp, vp]
    L.llm_keep.argtypes = [vp, i32, vp, i32]
    L.llm_score.argtypes = [vp, vp, i32, C.c_float, vp, vp, i32, vp, vp]
    L.llm_set_strict.argtypes = [vp, i32]
    L.llm_get_strict.argtypes = [vp]
    L.llm_kv_write.argtypes = [vp, vp, vp, vp, vp, i32, vp]
    L.llm_kv_read.argtypes = [vp, vp, vp, vp, vp, i32, i32, vp]
    L.llm_tree_attention_work.argtypes = [vp, i32, i32, i32]
    L.llm_tree_attention_work.restype = sz
    L.llm_tree_attention.argtypes = [vp, vp, vp, i32, vp, vp, vp, i32, i32, C.c_float, i32, vp, sz, vp]
    L.llm_logprobs_work.argtypes = [i32, i32, i32]
    L.llm_logprobs_work.restype = sz
    L.llm_logprobs.argtypes = [vp, i32, i32, i32, C.c_int64, C.c_float, vp, i32, vp, vp, vp, i32, vp, vp, vp, sz, vp]
    _lib = L
    return L


def _ptr(a):
    return a.ctypes.data_as(C.c_void_p)


# ---- test hooks -----------------------------------------------------------------------------------------

def quantize(x, flavor, gs=32):
    """Device activation quantization: flavor 0 = qwen.c:354-364, 1 = runq.c:244-270."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    q = np.empty(x.size, np.int8)
    s = np.empty(x.size // gs, np.float32)
    if lib().mvh_quantize(_ptr(x), x.size, flavor, gs, _ptr(q), _ptr(s)) != 0:
        raise RuntimeError("mvh_quantize failed")
    return q, s


def group_dots(w, xq, n, d, bits, gs=32):
    """Exact int32 group sums through the GEMV's dot-product code: [d, n/gs]."""
    w = np.ascontiguousarray(w, dtype=np.uint8)
    xq = np.ascontiguousarray(xq, dtype=np.int8)
    out = np.empty((d, n // gs), np.int32)
    if lib().mvh_group_dots(_ptr(w), _ptr(xq), n, d, bits, gs, _ptr(out)) != 0:
        raise RuntimeError("mvh_group_dots failed")
    return out


def prefill_gemm(w, ws, xq, xs, M, n, d, bits, gs=32, rb=16, shape=0):
    """The prefill GEMM (int8 MFMA) on caller data: [M, d] float32.  bits 4/8: qwen planes with fp16 scales;
    bits 0: runq int8 with fp32 scales, group gs.  shape: 0 the library's choice, 10 TA + TB one wave per
    16 TA rows x 16 TB tokens (TA 1, 2; TB 1, 2, 4), 32 and 33 the 32 x 32 tiles (int4) in the strict and the fast form,
    13 the 16 x 16 tiles (int4) in the fast form."""
    w = np.ascontiguousarray(w).view(np.uint8)
    ws = np.ascontiguousarray(ws)
    xq = np.ascontiguousarray(xq, dtype=np.int8)
    xs = np.ascontiguousarray(xs, dtype=np.float32)
    y = np.empty((M, d), np.float32)
    if lib().mvh_prefill_gemm(_ptr(w), _ptr(ws), _ptr(xq), _ptr(xs), M, n, d, bits, gs, rb, shape, _ptr(y)) != 0:
        raise RuntimeError("mvh_prefill_gemm failed")
    return y


def sample(logits, temperature, topp, seed, noalloc=False, strict=False, skew=None):
    """The on-device sampler on caller logits [count, n] (or [n]), drawn in order with one RNG state seeded by
    `seed`: (rows, the advanced RNG state).  noalloc: the entry point that allocates no device memory; strict:
    the strict mode's draw (the reference's sample() operation for operation); skew: the strict draw with its
    segment predictions moved by that many ulps (its term-by-term path)."""
    lg = np.ascontiguousarray(np.atleast_2d(logits), dtype=np.float32)
    rows = np.empty(lg.shape[0], np.int32)
    st = C.c_ulonglong(seed)
    args = [_ptr(lg), lg.shape[1], lg.shape[0], temperature, topp, C.byref(st), _ptr(rows)]
    if skew is not None:
        name, args = "mvh_sample_strict_skew", args + [skew]
    else:
        name = "mvh_sample_strict" if strict else "mvh_sample_noalloc" if noalloc else "mvh_sample"
    if getattr(lib(), name)(*args) != 0:
        raise RuntimeError(name + " failed")
    return rows, st.value


def read_floor(nbytes, copies, blocks, nt=True, reps=20):
    """µs per launch of a plain streaming read of nbytes (one launch per distinct buffer, in a graph)"""
    us = C.c_float(0)
    if lib().mvh_read_floor(nbytes, copies, blocks, int(nt), reps, C.byref(us)) != 0:
        raise RuntimeError("mvh_read_floor failed")
    return us.value


def seq_sum(x, which="block", threads=512):
    """the strict mode's sequential fp32 sum ((0 + x[0]) + x[1]) + ... on the device: which "block" (the block's
    speculative segments, `threads` threads), "wave" (one wave's chain) or "thread" (one thread's chain)"""
    x = np.ascontiguousarray(x, dtype=np.float32)
    out = np.zeros(1, np.float32)
    w = {"block": 0, "wave": 1, "thread": 2}[which]
    if lib().mvh_seq_sum(_ptr(x), x.size, w, threads, _ptr(out)) != 0:
        raise RuntimeError("mvh_seq_sum failed")
    return out[0]


def ref_expf(x, host=False):
    """expf as the reference's C library evaluates it (the strict mode's softmax and SiLU): on the device, or
    the same restatement compiled for the host CPU with host=True"""
    x = np.ascontiguousarray(x, dtype=np.float32)
    y = np.empty_like(x)
    fn = lib().mvh_ref_expf_host if host else lib().mvh_ref_expf
    if fn(_ptr(x), x.size, _ptr(y)) != 0:
        raise RuntimeError("mvh_ref_expf failed")
    return y


# ---- operators on device memory (torch tensors) -----------------------------------------------------------
# (a call's host time is most of a small call's: the C structs are packed in one step, and what the library checks by
# itself, that every address is memory of one device, is not checked here again.  There is no backward pass: tensors that
# require a gradient are refused where gradients are on)

_torch = None
_PACK_KV = struct.Struct("4P5i4x6q").pack
_PACK_ROWS = struct.Struct("Pi4x3q").pack


def _types():
    """torch and its types' LLM_* numbers (torch is imported by the first call that is given its tensors)"""
    global _torch
    if _torch is None:
        import torch
        _torch = torch, {torch.float32: 0, torch.bfloat16: 1, torch.int8: 2, torch.float8_e4m3fn: 3}
    return _torch


def _stream(t):
    """the current stream of a tensor's device"""
    dev = t.get_device()
    if dev < 0:
        raise ValueError("device tensors are needed")
    return _torch[0]._C._cuda_getCurrentRawStream(dev)  # (torch.cuda.current_stream(dev).cuda_stream, without its object)


def _ints(name, t, count, dtype):
    """the address of `count` contiguous integers (None: NULL)"""
    if t is None:
        return None
    if t.dtype is not dtype or t.numel() != count or not t.is_contiguous():
        raise ValueError(f"{name}: {count} contiguous {dtype} are needed")
    return t.data_ptr()


def _no_grad(*tensors):
    """refuses tensors that a gradient is asked of: the operators have none"""
    for t in tensors:
        if t is not None and t.requires_grad and _types()[0].is_grad_enabled():
            raise ValueError("the operators have no gradient: call them under torch.no_grad(), or with detached tensors")


def _written(*tensors):
    """tensors changed in place, as autograd counts it: a graph that saved one of them refuses its backward pass"""
    _torch[0].autograd.graph.increment_version([t for t in tensors if t is not None])


def _kv(k, v, k_scale, v_scale):
    """llm_kv of tensors [seqs, kv heads, positions, head size] (any strides, a row's values together) and, for int8 and
    e4m3, scales [seqs, kv heads, positions]; and its dimensions"""
    torch, types = _torch or _types()
    shape, dtype, st = k.shape, k.dtype, k.stride()
    ty = types.get(dtype)
    if ty is None or v.dtype is not dtype or v.shape != shape or len(shape) != 4:
        raise ValueError("k and v: tensors [seqs, kv heads, positions, head size] of one type (float32, bfloat16, int8, "
                         "float8_e4m3fn) are needed")
    b, h, ctx, hs = shape
    # (a dimension of one has no stride that counts)
    seq, head, pos, s_seq, s_head, s_pos = st[0] if b > 1 else 0, st[1] if h > 1 else 0, st[2] if ctx > 1 else hs, 0, 0, 1
    sv = v.stride()
    if st[3] != 1 or (st != sv and (sv[3] != 1 or (b > 1 and sv[0] != seq) or (h > 1 and sv[1] != head) or
                                    (ctx > 1 and sv[2] != pos))):
        raise ValueError("k and v: equal strides with a row's values together are needed")
    if ty < 2:
        if k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to int8 and e4m3 caches")
        return _PACK_KV(k.data_ptr(), v.data_ptr(), 0, 0, ty, b, h, hs, ctx, seq, head, pos, s_seq, s_head, s_pos), shape
    f32, rows = torch.float32, shape[:3]
    if k_scale is None or v_scale is None or k_scale.shape != rows or v_scale.shape != rows or \
            k_scale.dtype is not f32 or v_scale.dtype is not f32:
        raise ValueError("an int8 or e4m3 cache needs float32 scales [seqs, kv heads, positions]")
    ss, sv = k_scale.stride(), v_scale.stride()
    if ss != sv and ((b > 1 and ss[0] != sv[0]) or (h > 1 and ss[1] != sv[1]) or (ctx > 1 and ss[2] != sv[2])):
        raise ValueError("k_scale and v_scale: equal strides are needed")
    if b > 1:
        s_seq = ss[0]
    if h > 1:
        s_head = ss[1]
    if ctx > 1:
        s_pos = ss[2]
    return _PACK_KV(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), ty, b, h, hs, ctx, seq, head, pos,
                    s_seq, s_head, s_pos), shape


def _rows(name, x, b, t, h, hs):
    """llm_rows of a tensor [b, t, h, hs], float32 or bfloat16, a row's values together"""
    ty, st = _torch[1].get(x.dtype, 4), x.stride()
    if ty > 1 or x.shape != (b, t, h, hs) or st[3] != 1:
        raise ValueError(f"{name}: float32 or bfloat16 rows {(b, t, h, hs)} are needed")
    return _PACK_ROWS(x.data_ptr(), ty, st[0] if b > 1 else 0, st[1] if t > 1 else 0, st[2] if h > 1 else 0)


def kv_write(k_rows, v_rows, k, v, pos, n=None, k_scale=None, v_scale=None):
    """Rows [seqs, tokens, kv heads, head size] into the cache (llm_kv_write): token t < n[b] of sequence b at position
    pos[b] + t.  The cache: k and v [seqs, kv heads, positions, head size] of float32, bfloat16, int8 or float8_e4m3fn, the
    last two with float32 scales [seqs, kv heads, positions]."""
    _no_grad(k_rows, v_rows, k, v, k_scale, v_scale)
    c, (b, h, _, hs) = _kv(k, v, k_scale, v_scale)
    t, i32 = k_rows.shape[1], _torch[0].int32
    if lib().llm_kv_write(c, _rows("k_rows", k_rows, b, t, h, hs), _rows("v_rows", v_rows, b, t, h, hs),
                          _ints("pos", pos, b, i32), _ints("n", n, b, i32), t, _stream(k)) != 0:
        raise RuntimeError("llm_kv_write failed")
    _written(k, v, k_scale, v_scale)


def kv_read(k, v, pos, tokens, n=None, k_scale=None, v_scale=None, out=None, dtype=None):
    """The values of positions pos[b] .. pos[b] + n[b] - 1 (n None: `tokens` each) as rows [seqs, tokens, kv heads, head
    size] of K and V (llm_kv_read), float32 or `dtype`; new tensors (rows that are not read: zero) or `out`, a pair (such
    rows left as they were)."""
    _no_grad(k, v, k_scale, v_scale, *(() if out is None else (out[0], out[1])))
    c, (b, h, _, hs) = _kv(k, v, k_scale, v_scale)
    torch, fresh = _torch[0], out is None
    if fresh:
        out = torch.empty(2, b, tokens, h, hs, dtype=dtype or torch.float32, device=k.device).unbind()
    if lib().llm_kv_read(c, _rows("out", out[0], b, tokens, h, hs), _rows("out", out[1], b, tokens, h, hs),
                         _ints("pos", pos, b, torch.int32), _ints("n", n, b, torch.int32), tokens, fresh, _stream(k)) != 0:
        raise RuntimeError("llm_kv_read failed")
    if not fresh:
        _written(out[0], out[1])
    return out[0], out[1]


def tree_attention(q, k, v, lens, n=None, mask=None, k_scale=None, v_scale=None, scale=None, max_len=None, out=None):
    """Attention of the newest tokens of every sequence over its cache (llm_tree_attention; no gradient).  q [seqs, tokens <= 64,
    heads, head size] float32 or bfloat16; the cache as in kv_write; token i of sequence b has its rows at position lens[b] + i
    and sees the positions before lens[b] and the new tokens of mask[b, i]'s bits (int64; None: a chain).  n[b] tokens count
    (None: all); scale None: head size ** -0.5; max_len: the host's bound of lens (None: the cache's positions).  Returns
    a new tensor (rows behind n[b]: zero), or `out` (such rows left as they were)."""
    _no_grad(q, k, v, k_scale, v_scale, out)
    c, (b, _, ctx, hs) = _kv(k, v, k_scale, v_scale)
    torch, fresh = _torch[0], out is None
    t, heads = q.shape[1:3]
    if mask is not None and mask.dim() > 1 and mask.shape != (b, t):
        raise ValueError(f"mask: int64 {(b, t)} are needed")
    if fresh:
        out = torch.empty(b, t, heads, hs, dtype=q.dtype, device=k.device)
    L, bound = lib(), ctx if max_len is None else max_len
    need = L.llm_tree_attention_work(c, heads, t, bound)
    work = torch.empty(need, dtype=torch.uint8, device=k.device) if need else None
    if L.llm_tree_attention(c, _rows("q", q, b, t, heads, hs), _rows("out", out, b, t, heads, hs), heads,
                            _ints("lens", lens, b, torch.int32), _ints("n", n, b, torch.int32),
                            _ints("mask", mask, b * t, torch.int64), t, bound, hs ** -0.5 if scale is None else scale, fresh,
                            work.data_ptr() if need else None, need, _stream(k)) != 0:
        raise RuntimeError("llm_tree_attention failed")
    if not fresh:
        _written(out)
    return out


def logprobs(logits, tokens=None, top=0, temperature=1.0):
    """Log probabilities of logits / temperature (llm_logprobs): logits [rows, vocab] float32 or bfloat16 (any row stride),
    tokens [rows, count] int32.  Returns (logp [rows, count] of the tokens, entropy [rows], top_ids [rows, top] and top_logp
    [rows, top] of the largest logits in descending order, lse [rows])."""
    torch, types = _types()
    _no_grad(logits)
    rows, vocab = logits.shape
    ty, st = types.get(logits.dtype, 4), logits.stride()
    if ty > 1 or (vocab > 1 and st[1] != 1) or (tokens is not None and (tokens.dim() != 2 or tokens.shape[0] != rows)):
        raise ValueError("logits: float32 or bfloat16 rows [rows, vocab], tokens: [rows, count] are needed")
    count = tokens.shape[1] if tokens is not None else 0
    L = lib()
    need = L.llm_logprobs_work(rows, vocab, top)
    # one allocation: the results, and the scratch memory behind them
    at = rows * (2 + 2 * top + count)
    at += -at % 4
    mem = torch.empty(at + need // 4, dtype=torch.float32, device=logits.device)
    entropy, lse, ids, top_logp, logp, _ = mem.split_with_sizes(
        (rows, rows, rows * top, rows * top, rows * count, mem.numel() - rows * (2 + 2 * top + count)))
    ids = ids.view(torch.int32)
    p = mem.data_ptr()
    if rows and L.llm_logprobs(logits.data_ptr(), ty, rows, vocab, st[0] if rows > 1 else vocab, temperature,
                               _ints("tokens", tokens, rows * count, torch.int32) if count else None, count,
                               p + 4 * rows * (2 + 2 * top), p, p + 4 * rows, top, p + 8 * rows, p + 4 * rows * (2 + top),
                               p + 4 * at if need else None, need, _stream(logits)) != 0:
        raise RuntimeError("llm_logprobs failed")
    return logp.view(rows, count), entropy, ids.view(rows, top), top_logp.view(rows, top), lse


# ---- drop-in driver API -----------------------------------------------------------------------------------

class DropIn:
    """The reference's driver API (fpga_open / fpga_alloc / fpga_matvec[4] / fpga_close) through ctypes."""

    def __init__(self):
        self.L = lib()
        if self.L.fpga_open() != 0:
            raise RuntimeError("fpga_open failed")
        self.bufs = []

    def alloc(self, nbytes):
        """(numpy uint8 view of the host buffer, device address)"""
        phys = C.c_uint64(0)
        p = self.L.fpga_alloc(nbytes, C.byref(phys))
        if not p:
            raise MemoryError("fpga_alloc failed")
        view = np.ctypeslib.as_array((C.c_uint8 * nbytes).from_address(p))
        self.bufs.append(view)
        return view, phys.value

    def put(self, arr, align=64):
        """copy an array into a new buffer; returns (view, device address)"""
        b = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
        view, phys = self.alloc(max(b.size, 1))
        view[:b.size] = b
        return view, phys

    def matvec4(self, w, ws, xq, xs, out, n, d, wbits):
        return self.L.fpga_matvec4(w, ws, xq, xs, out, n, d, wbits)

    def matvec(self, wq, ws, xq, xs, out, n, d, gs):
        return self.L.fpga_matvec(wq, ws, xq, xs, out, n, d, gs)

    def close(self):
        self.bufs = []
        self.L.fpga_close()


# ---- device-resident model -----------------------------------------------------------------------------------

class Model:
    """A .qwb or llama2.c .bin model resident in HBM (llm_open)."""

    def __init__(self, path, ctx=1024):
        self.L = lib()
        self.h = self.L.llm_open(os.fsencode(path), ctx)
        if not self.h:
            raise RuntimeError(f"llm_open({path}) failed")
        self.info = LlmInfo()
        self.L.llm_get_info(self.h, C.byref(self.info))
        hid = self.L.llm_head_ids(self.h)
        n = self.info.n_logits
        self.head_ids = np.ctypeslib.as_array(hid, shape=(n,)).copy() if hid else np.arange(n, dtype=np.int32)

    def forward(self, token, pos):
        lg = np.empty(self.info.n_logits, np.float32)
        if self.L.llm_forward(self.h, int(token), int(pos), _ptr(lg)) != 0:
            raise RuntimeError("llm_forward failed")
        return lg

    def generate(self, prompt, max_new, logits=False):
        """greedy ids (and the logits of every position run, when asked)"""
        p = np.ascontiguousarray(prompt, dtype=np.int32)
        out = np.empty(max_new, np.int32)
        lg = np.empty((len(p) + max_new) * self.info.n_logits, np.float32) if logits else None
        t = LlmTiming()
        n = self.L.llm_generate(self.h, _ptr(p), len(p), max_new, _ptr(out), _ptr(lg) if logits else None,
                                C.byref(t))
        if n < 0:
            raise RuntimeError("llm_generate failed")
        res = {"ids": out[:n].copy(), "timing": t}
        if logits:
            res["logits"] = lg[:t.n_forward * self.info.n_logits].reshape(t.n_forward, self.info.n_logits)
        return res

    def continue_at(self, pos0, tokens, max_new, stop_id=-1):
        """the tokens forced from position pos0 over the cache earlier calls left, then up to max_new generated
        ids until stop_id (-1: the format's stop ids)"""
        p = np.ascontiguousarray(tokens, dtype=np.int32)
        out = np.empty(max_new, np.int32)
        t = LlmTiming()
        n = self.L.llm_continue(self.h, pos0, _ptr(p), len(p), max_new, stop_id, _ptr(out), C.byref(t))
        if n < 0:
            raise RuntimeError("llm_continue failed")
        return {"ids": out[:n].copy(), "timing": t}

    def decode_replay(self, steps):
        ms = C.c_double(0)
        if self.L.llm_decode_replay(self.h, steps, C.byref(ms)) != 0:
            raise RuntimeError("llm_decode_replay failed")
        return ms.value

    def profile(self, steps):
        st = (LlmKernelStat * 16)()
        n = self.L.llm_profile(self.h, steps, st, 16)
        if n < 0:
            raise RuntimeError("llm_profile failed")
        return [{"name": st[i].name.decode(), "launches": st[i].launches, "total_ms": st[i].total_ms,
                 "bytes_per_launch": st[i].bytes_per_launch} for i in range(n)]

    def profile_graph(self, steps, rounds=3):
        """per-kernel-kind device time inside the replayed step graph (see llm_profile_graph); returns
        (records, median step ms)"""
        st = (LlmKernelStat * 16)()
        step = C.c_double(0.0)
        n = self.L.llm_profile_graph(self.h, steps, rounds, st, 16, C.byref(step))
        if n < 0:
            raise RuntimeError("llm_profile_graph failed")
        return [{"name": st[i].name.decode(), "launches": st[i].launches, "total_ms": st[i].total_ms,
                 "bytes_per_launch": st[i].bytes_per_launch} for i in range(n)], step.value

    def read_state(self, which, layer=0, count=None):
        n = self.info.dim if which == 0 else self.info.ctx * (self.info.dim // self.info.n_heads * self.info.n_kv_heads)
        if count is not None:
            n = min(n, count)
        out = np.empty(n, np.float32)
        if self.L.llm_read_state(self.h, which, layer, _ptr(out), n) != 0:
            raise RuntimeError("llm_read_state failed")
        return out

    def set_sampler(self, temperature, topp=0.9, seed=1):
        """temperature > 0: generate() draws tokens on the device (temperature, top-p, xorshift coin from
        seed); 0: greedy"""
        if self.L.llm_set_sampler(self.h, temperature, topp, seed) != 0:
            raise RuntimeError("llm_set_sampler failed")

    def sampler_state(self):
        st = C.c_ulonglong(0)
        if self.L.llm_sampler_state(self.h, C.byref(st)) != 0:
            raise RuntimeError("llm_sampler_state failed")
        return st.value

    def set_strict(self, on):
        """reference-order mode: logits bitwise those of the reference's strict-IEEE build (llm_set_strict)"""
        if self.L.llm_set_strict(self.h, 1 if on else 0) != 0:
            raise RuntimeError("llm_set_strict failed")

    @property
    def strict(self):
        return self.L.llm_get_strict(self.h) == 1

    def set_prefill(self, on):
        """whether generate() runs the prompt as one batched prefill (default) or one step per position"""
        self.L.llm_set_prefill(self.h, 1 if on else 0)

    def prefill(self, ids):
        """batched prefill of positions 0..len(ids)-1; the logits of the last position"""
        p = np.ascontiguousarray(ids, dtype=np.int32)
        lg = np.empty(self.info.n_logits, np.float32)
        if self.L.llm_prefill(self.h, _ptr(p), len(p), _ptr(lg)) != 0:
            raise RuntimeError("llm_prefill failed")
        return lg

    KV_TYPES = ["fp32", "bf16", "int8", "e4m3"]

    def set_kv(self, kind):
        """the cache's type ("fp32", "bf16", "int8", "e4m3"); the cache is empty afterwards (llm_set_kv)"""
        if self.L.llm_set_kv(self.h, self.KV_TYPES.index(kind)) != 0:
            raise RuntimeError("llm_set_kv failed")

    @property
    def kv(self):
        return self.KV_TYPES[self.L.llm_get_kv(self.h)]

    def verify(self, pos0, tokens, parents=None, logits=False):
        """one pass over a drafted tree from position pos0 (llm_verify): (the most likely next token after each, the log
        probability of each after its parent), and the logits of each where asked"""
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        p = None if parents is None else np.ascontiguousarray(parents, dtype=np.int32)
        if p is not None and p.size != t.size:
            raise ValueError("a parent for every token is needed")
        nxt, lp = np.empty(t.size, np.int32), np.empty(t.size, np.float32)
        lg = np.empty((t.size, self.info.n_logits), np.float32) if logits else None
        if self.L.llm_verify(self.h, pos0, _ptr(t), None if p is None else _ptr(p), t.size, _ptr(nxt), _ptr(lp),
                             _ptr(lg) if logits else None) != 0:
            raise RuntimeError("llm_verify failed")
        return (nxt, lp, lg) if logits else (nxt, lp)

    def keep(self, pos0, path):
        """the cache rows of the accepted tokens of a verified tree moved to positions pos0, pos0 + 1, ... (llm_keep)"""
        p = np.ascontiguousarray(path, dtype=np.int32)
        if self.L.llm_keep(self.h, pos0, _ptr(p), p.size) != 0:
            raise RuntimeError("llm_keep failed")

    def score(self, ids, top=0, temperature=1.0):
        """log probabilities of a text (llm_score): (of every token after the first, the entropy after every token, the top
        alternatives' ids and their log probabilities)"""
        p = np.ascontiguousarray(ids, dtype=np.int32)
        lp, ent = np.empty(max(p.size - 1, 0), np.float32), np.empty(p.size, np.float32)
        ti, tl = np.empty((p.size, top), np.int32), np.empty((p.size, top), np.float32)
        if self.L.llm_score(self.h, _ptr(p), p.size, temperature, _ptr(lp), _ptr(ent), top, _ptr(ti), _ptr(tl)) != 0:
            raise RuntimeError("llm_score failed")
        return lp, ent, ti, tl

    def close(self):
        if self.h:
            self.L.llm_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
