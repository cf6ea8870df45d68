"""ctypes binding of libm27b.so, the C ABI declared in include/m27b_qmv.h.

This is the Python mirror of the reference's matvec seam (WeightView +
quantize/matvec calls, src/mono27b_executor.cu:1989-2261) used by the tests and
the benchmark.  PyTorch only provides device memory and streams; every
computation goes through the CUDA library.  There is no fallback: if
libm27b.so is missing or fails to load, every call raises.
"""
import ctypes
import os
import struct
import threading

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libm27b.so")

# ggml type codes (reference include/mono27b_gguf.h:28-44; IQ4_XS = 23)
F32, F16, Q8_0, Q4_K, Q5_K, Q6_K, Q8_K, IQ4_XS = 0, 1, 8, 12, 13, 14, 15, 23
LAYOUT_PLANAR = 0x100
MAX_TOKENS = 16
BLOCK = {F32: (1, 4), F16: (1, 2), Q8_0: (32, 34), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210),
         Q8_K: (256, 292), IQ4_XS: (256, 136)}

ERR_CAP = 512


class WeightView(ctypes.Structure):
    """Same layout as the reference's WeightView (include/mono27b_config.h:63-68)."""
    _fields_ = [("ptr", ctypes.c_void_p), ("ggml_type", ctypes.c_uint32), ("row_blocks", ctypes.c_uint32),
                ("row_count", ctypes.c_uint32)]


class M27BError(RuntimeError):
    pass


_lib = None


def lib():
    """Load libm27b.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise M27BError(f"libm27b.so is not built ({LIB_PATH}); run __graft_entry__.build()")
    L = ctypes.CDLL(LIB_PATH)
    vp, u32, i32, sz, cp = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int, ctypes.c_size_t, ctypes.c_char_p
    fp, b = ctypes.c_float, ctypes.c_bool
    wvp = ctypes.POINTER(WeightView)
    sig = {
        "m27b_version": (cp, []),
        "m27b_device_status": (b, [ctypes.POINTER(ctypes.c_int), i32, cp, sz]),
        "m27b_act_bytes": (sz, [u32, i32]),
        "m27b_act_type_for": (u32, [u32]),
        "m27b_act_quant": (b, [vp, i32, i32, i32, u32, vp, vp, cp, sz]),
        "m27b_act_quant_gated": (b, [vp, vp, i32, i32, i32, u32, vp, vp, cp, sz]),
        "m27b_act_quant_swiglu": (b, [vp, vp, i32, i32, i32, u32, vp, vp, cp, sz]),
        "m27b_act_quant_rmsnorm": (b, [vp, vp, fp, i32, i32, i32, u32, vp, vp, cp, sz]),
        "m27b_repacked_bytes": (sz, [u32, u32, u32]),
        "m27b_repack": (b, [vp, u32, u32, u32, vp, vp, cp, sz]),
        "m27b_qmv": (b, [wvp, vp, i32, vp, i32, vp, vp, cp, sz]),
        "m27b_qmv_swiglu": (b, [wvp, wvp, vp, i32, vp, i32, vp, cp, sz]),
        "m27b_qmv_argmax": (b, [wvp, vp, i32, vp, i32, vp, u32, vp, cp, sz]),
        "m27b_qmv_f32": (b, [wvp, vp, i32, i32, vp, vp, i32, vp, vp, cp, sz]),
        "m27b_qmv_f32_rmsnorm": (b, [wvp, wvp, vp, i32, vp, fp, i32, vp, vp, i32, vp, vp, cp, sz]),
        "m27b_dequant_rows": (b, [wvp, vp, i32, vp, i32, vp, cp, sz]),
        "m27b_hbm_read_probe": (b, [vp, sz, vp, cp, sz]),
        "m27b_hbm_read_probe_shape": (b, [vp, sz, i32, i32, i32, i32, vp, cp, sz]),
        "m27b_qmv_mma_split_part_bytes": (sz, [wvp, i32]),
        "m27b_qmv_mma_split_count_bytes": (sz, [wvp]),
        "m27b_qmv_mma_split": (b, [wvp, vp, i32, vp, i32, vp, vp, vp, vp, cp, sz]),
        "m27b_qmv_q6k_mma_part_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_mma_count_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_mma": (b, [wvp, vp, i32, vp, i32, vp, vp, vp, vp, cp, sz]),
        "m27b_qmv_q6k_mma_argmax": (b, [wvp, vp, i32, vp, i32, vp, u32, vp, cp, sz]),
        "m27b_qmv_q6k_stream_part_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_stream_count_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_stream": (b, [wvp, vp, vp, vp, vp, vp, vp, cp, sz]),
        "m27b_qmv_q6k_ksplit_part_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_ksplit_count_bytes": (sz, [wvp]),
        "m27b_qmv_q6k_ksplit": (b, [wvp, vp, i32, vp, i32, vp, vp, vp, vp, cp, sz]),
        "m27b_allreduce_norm_quant": (b, [vp, i32, i32, vp, vp, vp, fp, i32, vp, vp, ctypes.c_ulonglong, vp, cp, sz]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _lib = L
    return L


def version():
    return lib().m27b_version().decode()


def device_status(clear=True):
    """The device status word (0 = every bounded kernel wait completed)."""
    v = ctypes.c_int(0)
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(lib().m27b_device_status(ctypes.byref(v), 1 if clear else 0, err, ERR_CAP), err, "m27b_device_status")
    return v.value


def row_bytes(qtype, k):
    be, bb = BLOCK[qtype & 0xff]
    assert k % be == 0
    return k // be * bb


def act_type_for(qtype):
    """q8_0 for q8_0 weights, q8_K for the 256-value types, 0 (fp32 rows) for f16 / f32."""
    b = qtype & 0xff
    return Q8_0 if b == Q8_0 else (0 if b in (F16, F32) else Q8_K)


def act_bytes(act_type, k):
    return lib().m27b_act_bytes(act_type, k)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream(stream):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _check(ok, err, what):
    if not ok:
        raise M27BError(f"{what}: {err.value.decode(errors='replace')}")


class QWeight:
    """A quantized (or f16 / f32) weight matrix resident on the device.

    Holds the device bytes (a torch uint8 tensor) and the WeightView the C ABI
    consumes.  q6_K and q8_0 are repacked to the planar layout on upload; for
    f16 / f32 row_blocks counts values, as in the reference loader.
    """

    def __init__(self, raw_u8, qtype, k, rows, device="cuda", stream=None, keep_raw=False):
        import torch
        self.qtype, self.k, self.rows = qtype, k, rows
        be = BLOCK[qtype][0]
        self.row_blocks = k // be
        raw = torch.as_tensor(raw_u8).reshape(-1)
        if raw.dtype != torch.uint8:
            raw = raw.view(torch.uint8)
        assert raw.numel() == rows * row_bytes(qtype, k), (raw.numel(), rows, row_bytes(qtype, k))
        raw_dev = raw.to(device) if raw.device.type != "cuda" else raw
        if qtype in (Q6_K, Q8_0):
            n = lib().m27b_repacked_bytes(qtype, self.row_blocks, rows)
            self.data = torch.empty(n, dtype=torch.uint8, device=raw_dev.device)
            err = ctypes.create_string_buffer(ERR_CAP)
            _check(lib().m27b_repack(_ptr(raw_dev), qtype, self.row_blocks, rows, _ptr(self.data), _stream(stream), err,
                                     ERR_CAP), err, "m27b_repack")
            self.view = WeightView(self.data.data_ptr(), qtype | LAYOUT_PLANAR, self.row_blocks, rows)
            self.raw = raw_dev if keep_raw else None
        else:
            self.data = raw_dev.contiguous()
            self.view = WeightView(self.data.data_ptr(), qtype, self.row_blocks, rows)
            self.raw = self.data
        self.nbytes = rows * row_bytes(qtype, k)  # stored GGUF bytes (algorithmic)

    @property
    def act_type(self):
        return act_type_for(self.qtype)


def act_quant(x, act_type, out=None, stream=None, gate=None, norm_w=None, eps=None):
    """Quantize fp32 rows x [n, k] (device) to q8_K / q8_0 blocks (device uint8)."""
    import torch
    x = x if x.dim() == 2 else x.reshape(1, -1)
    n, k = x.shape
    nb = act_bytes(act_type, k)
    if nb == 0:
        raise M27BError(f"act_quant: bad k={k} for type {act_type}")
    if out is None:
        out = torch.empty(n * nb, dtype=torch.uint8, device=x.device)
    err = ctypes.create_string_buffer(ERR_CAP)
    L = lib()
    if gate is not None:
        ok = L.m27b_act_quant_gated(_ptr(x), _ptr(gate), k, n, x.stride(0), act_type, _ptr(out), _stream(stream), err,
                                    ERR_CAP)
    elif eps is not None:
        ok = L.m27b_act_quant_rmsnorm(_ptr(x), _ptr(norm_w), ctypes.c_float(eps), k, n, x.stride(0), act_type, _ptr(out),
                                      _stream(stream), err, ERR_CAP)
    else:
        ok = L.m27b_act_quant(_ptr(x), k, n, x.stride(0), act_type, _ptr(out), _stream(stream), err, ERR_CAP)
    _check(ok, err, "m27b_act_quant")
    return out


def allreduce_norm_quant(words, nsrc, src_stride, ss_words, epoch, k, x_out, xq, norm_w=None, eps=1e-6, wait_ns=0,
                         stream=None):
    """The fused all-reduce's consumer (include/m27b_allreduce.h): sum the nsrc
    ranks' epoch-tagged words (device int64 tensors, value bits low, epoch
    high) once they carry *epoch (device uint32), then RMSNorm + q8_K into xq."""
    err = ctypes.create_string_buffer(ERR_CAP)
    ok = lib().m27b_allreduce_norm_quant(_ptr(words), nsrc, src_stride, _ptr(ss_words), _ptr(epoch), _ptr(norm_w),
                                         ctypes.c_float(eps), k, _ptr(x_out), _ptr(xq), ctypes.c_ulonglong(wait_ns),
                                         _stream(stream), err, ERR_CAP)
    _check(ok, err, "m27b_allreduce_norm_quant")
    return xq


def qmv_q6k_ksplit(w, xq, n_tok, y, residual=None, part=None, count=None, stream=None, ldy=None):
    """q6_K x n_tok (5..16) tokens with K split across CTAs (m27b_qmv_q6k_ksplit);
    part / count scratch are allocated here (counters zeroed) unless given."""
    import torch
    L = lib()
    if part is None:
        part = torch.empty(max(16, L.m27b_qmv_q6k_ksplit_part_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                           device="cuda")
    if count is None:
        count = torch.zeros(max(16, L.m27b_qmv_q6k_ksplit_count_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                            device="cuda")
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(L.m27b_qmv_q6k_ksplit(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(y),
                                 ldy if ldy is not None else w.view.row_count, _ptr(residual), _ptr(part), _ptr(count),
                                 _stream(stream), err, ERR_CAP), err, "m27b_qmv_q6k_ksplit")
    return y


def qmv_mma_split(w, xq, n_tok, y, residual=None, part=None, count=None, stream=None, ldy=None):
    """q4_K x n_tok (5..16) tokens on the tensor cores with K split across CTAs
    (m27b_qmv_mma_split); part / count scratch are allocated here (counters
    zeroed) unless given."""
    import torch
    L = lib()
    if part is None:
        part = torch.empty(max(16, L.m27b_qmv_mma_split_part_bytes(ctypes.byref(w.view), n_tok)), dtype=torch.uint8,
                           device="cuda")
    if count is None:
        count = torch.zeros(max(16, L.m27b_qmv_mma_split_count_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                            device="cuda")
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(L.m27b_qmv_mma_split(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(y),
                                ldy if ldy is not None else w.view.row_count, _ptr(residual), _ptr(part), _ptr(count),
                                _stream(stream), err, ERR_CAP), err, "m27b_qmv_mma_split")
    return y


def qmv_q6k_mma(w, xq, n_tok, y, residual=None, part=None, count=None, stream=None, ldy=None, split=True):
    """q6_K x n_tok (1..8) tokens on the tensor cores (m27b_qmv_q6k_mma); with
    split, K-split scratch is allocated here (counters zeroed) unless given."""
    import torch
    L = lib()
    if split and part is None:
        part = torch.empty(max(16, L.m27b_qmv_q6k_mma_part_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                           device="cuda")
    if split and count is None:
        count = torch.zeros(max(16, L.m27b_qmv_q6k_mma_count_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                            device="cuda")
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(L.m27b_qmv_q6k_mma(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(y),
                              ldy if ldy is not None else w.view.row_count, _ptr(residual), _ptr(part), _ptr(count),
                              _stream(stream), err, ERR_CAP), err, "m27b_qmv_q6k_mma")
    return y


def qmv_q6k_mma_argmax(w, xq, n_tok, best, logits=None, row_offset=0, stream=None, ldl=None):
    """q6_K x n_tok (1..8) tokens on the tensor cores with the argmax epilogue
    (m27b_qmv_q6k_mma_argmax)."""
    err = ctypes.create_string_buffer(ERR_CAP)
    ldl = ldl if ldl is not None else w.rows
    _check(lib().m27b_qmv_q6k_mma_argmax(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(logits), ldl, _ptr(best),
                                         row_offset, _stream(stream), err, ERR_CAP), err, "m27b_qmv_q6k_mma_argmax")
    return best


def qmv_q6k_stream(w, xq, y, residual=None, part=None, count=None, stream=None):
    """q6_K x one token with the items cut evenly over warps
    (m27b_qmv_q6k_stream); part / count scratch are allocated here (counters
    zeroed) unless given."""
    import torch
    L = lib()
    if part is None:
        part = torch.empty(max(16, L.m27b_qmv_q6k_stream_part_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                           device="cuda")
    if count is None:
        count = torch.zeros(max(16, L.m27b_qmv_q6k_stream_count_bytes(ctypes.byref(w.view))), dtype=torch.uint8,
                            device="cuda")
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(L.m27b_qmv_q6k_stream(ctypes.byref(w.view), _ptr(xq), _ptr(y), _ptr(residual), _ptr(part), _ptr(count),
                                 _stream(stream), err, ERR_CAP), err, "m27b_qmv_q6k_stream")
    return y


def hbm_read_probe(buf, shape=None, stream=None):
    """One streaming read of the device tensor `buf` (see
    m27b_hbm_read_probe_shape); shape = (warps, stages, chunk, ctas_per_sm)
    or None for the default one."""
    err = ctypes.create_string_buffer(ERR_CAP)
    n = buf.numel() * buf.element_size()
    if shape is None:
        ok = lib().m27b_hbm_read_probe(_ptr(buf), n, _stream(stream), err, ERR_CAP)
    else:
        ok = lib().m27b_hbm_read_probe_shape(_ptr(buf), n, *[int(v) for v in shape], _stream(stream), err, ERR_CAP)
    _check(ok, err, "m27b_hbm_read_probe")


def act_quant_swiglu(gate, up, act_type, out=None, stream=None):
    """Quantize silu(gate) * up (device rows [n, k]) to q8_K / q8_0 blocks."""
    import torch
    n, k = up.shape
    nb = act_bytes(act_type, k)
    if out is None:
        out = torch.empty(n * nb, dtype=torch.uint8, device=up.device)
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(lib().m27b_act_quant_swiglu(_ptr(gate), _ptr(up), k, n, up.stride(0), act_type, _ptr(out), _stream(stream),
                                       err, ERR_CAP), err, "m27b_act_quant_swiglu")
    return out


def qmv(w, xq, n_tok, y, residual=None, stream=None, ldy=None):
    err = ctypes.create_string_buffer(ERR_CAP)
    ldy = ldy if ldy is not None else w.rows
    _check(lib().m27b_qmv(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(y), ldy, _ptr(residual), _stream(stream), err,
                          ERR_CAP), err, "m27b_qmv")
    return y


def qmv_swiglu(gate, up, xq, n_tok, y, stream=None, ldy=None):
    err = ctypes.create_string_buffer(ERR_CAP)
    ldy = ldy if ldy is not None else gate.rows
    _check(lib().m27b_qmv_swiglu(ctypes.byref(gate.view), ctypes.byref(up.view), _ptr(xq), n_tok, _ptr(y), ldy,
                                 _stream(stream), err, ERR_CAP), err, "m27b_qmv_swiglu")
    return y


def qmv_argmax(w, xq, n_tok, best, logits=None, row_offset=0, stream=None, ldl=None):
    err = ctypes.create_string_buffer(ERR_CAP)
    ldl = ldl if ldl is not None else w.rows
    _check(lib().m27b_qmv_argmax(ctypes.byref(w.view), _ptr(xq), n_tok, _ptr(logits), ldl, _ptr(best), row_offset,
                                 _stream(stream), err, ERR_CAP), err, "m27b_qmv_argmax")
    return best


def qmv_f32(w, x, n_tok, y, residual=None, xq_scratch=None, norm_w=None, eps=None, up=None, stream=None, ldy=None):
    """y = W . q8(x) (+ residual) from fp32 rows x [n_tok, k] (device); with eps
    given, x is RMSNormed (weights norm_w) first; with `up`, SwiGLU epilogue."""
    err = ctypes.create_string_buffer(ERR_CAP)
    L = lib()
    ldx = x.stride(0) if x.dim() == 2 else x.shape[-1]
    ldy = ldy if ldy is not None else w.view.row_count
    if eps is None and up is None:
        ok = L.m27b_qmv_f32(ctypes.byref(w.view), _ptr(x), ldx, n_tok, _ptr(xq_scratch), _ptr(y), ldy, _ptr(residual),
                            _stream(stream), err, ERR_CAP)
        _check(ok, err, "m27b_qmv_f32")
    else:
        ok = L.m27b_qmv_f32_rmsnorm(ctypes.byref(w.view), ctypes.byref(up.view) if up is not None else None, _ptr(x),
                                    ldx, _ptr(norm_w), ctypes.c_float(1e-6 if eps is None else eps), n_tok,
                                    _ptr(xq_scratch), _ptr(y), ldy, _ptr(residual), _stream(stream), err, ERR_CAP)
        _check(ok, err, "m27b_qmv_f32_rmsnorm")
    return y


def argmax_key_index(key):
    return 0xffffffff - (int(key) & 0xffffffff)


def dequant_rows(w, rows_dev, out, stream=None, view=None):
    err = ctypes.create_string_buffer(ERR_CAP)
    v = view if view is not None else w.view
    k = v.row_blocks * BLOCK[v.ggml_type & 0xff][0]
    _check(lib().m27b_dequant_rows(ctypes.byref(v), _ptr(rows_dev), rows_dev.numel(), _ptr(out), k, _stream(stream), err,
                                   ERR_CAP), err, "m27b_dequant_rows")
    return out


def call_raw(name, *args):
    """Call a C-ABI function with an error buffer appended; returns (ok, message)."""
    err = ctypes.create_string_buffer(ERR_CAP)
    ok = getattr(lib(), name)(*args, err, ERR_CAP)
    return bool(ok), err.value.decode(errors="replace")


# --------------------------------------------------------------------------
# decode attention (include/m27b_attn.h)


def _attn_lib():
    L = lib()
    if getattr(L, "_attn_sigs", False):
        return L
    vp, i32, sz, cp, fp, b = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_char_p, ctypes.c_float, ctypes.c_bool
    L.m27b_attn_part_bytes.restype = sz
    L.m27b_attn_part_bytes.argtypes = [i32, i32, i32]
    L.m27b_attn_decode.restype = b
    L.m27b_attn_decode.argtypes = [vp, vp, vp, vp, i32, i32, i32, i32, fp, vp, vp, vp, cp, sz]
    L.m27b_attn_decode_noalloc.restype = b
    L.m27b_attn_decode_noalloc.argtypes = [vp, vp, vp, vp, i32, i32, i32, i32, fp, vp, vp, cp, sz]
    L.m27b_attn_noalloc_scratch_bytes.restype = sz
    L.m27b_attn_noalloc_scratch_bytes.argtypes = []
    L._attn_sigs = True
    return L


def attn_part_bytes(n_q, head_dim, splits):
    return _attn_lib().m27b_attn_part_bytes(n_q, head_dim, splits)


def attn_decode(q, k_cache, v_cache, pos, n_q, n_kv, head_dim, splits, scale, part, out, stream=None):
    """Decode attention of n_q heads over cache positions [0, pos[0]] (all device tensors)."""
    err = ctypes.create_string_buffer(ERR_CAP)
    ok = _attn_lib().m27b_attn_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(pos), n_q, n_kv, head_dim, splits,
                                      ctypes.c_float(scale), _ptr(part), _ptr(out), _stream(stream), err, ERR_CAP)
    _check(ok, err, "m27b_attn_decode")
    return out


def attn_noalloc_scratch_bytes():
    """Capacity of m27b_attn_decode_noalloc's static scratch, as compiled into the library."""
    return _attn_lib().m27b_attn_noalloc_scratch_bytes()


def attn_decode_noalloc(q, k_cache, v_cache, pos, n_q, n_kv, head_dim, splits, scale, out, stream=None):
    """m27b_attn_decode with the library's static scratch (no scratch argument, no allocation)."""
    err = ctypes.create_string_buffer(ERR_CAP)
    ok = _attn_lib().m27b_attn_decode_noalloc(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(pos), n_q, n_kv, head_dim,
                                              splits, ctypes.c_float(scale), _ptr(out), _stream(stream), err, ERR_CAP)
    _check(ok, err, "m27b_attn_decode_noalloc")
    return out


# --------------------------------------------------------------------------
# decode engine (include/m27b_engine.h)


class ModelConfig(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int), ("hidden", ctypes.c_int), ("ffn", ctypes.c_int), ("n_head", ctypes.c_int),
                ("n_kv_head", ctypes.c_int), ("head_dim", ctypes.c_int), ("vocab", ctypes.c_int), ("n_rot", ctypes.c_int),
                ("rope_theta", ctypes.c_float), ("rms_eps", ctypes.c_float), ("max_ctx", ctypes.c_int),
                ("tp_rank", ctypes.c_int), ("tp_size", ctypes.c_int), ("weight_type", ctypes.c_uint32),
                ("attn_interval", ctypes.c_int), ("ssm_d_inner", ctypes.c_int), ("ssm_d_state", ctypes.c_int),
                ("ssm_dt_rank", ctypes.c_int), ("ssm_n_group", ctypes.c_int), ("ssm_conv_kern", ctypes.c_int)]


class Partition(ctypes.Structure):
    _fields_ = [("q_lo", ctypes.c_int), ("n_q", ctypes.c_int), ("kv_lo", ctypes.c_int), ("n_kv", ctypes.c_int),
                ("f_lo", ctypes.c_int), ("n_f", ctypes.c_int), ("v_lo", ctypes.c_int), ("n_v", ctypes.c_int)]


QWEN27 = dict(n_layers=64, hidden=5120, ffn=17408, n_head=24, n_kv_head=4, head_dim=256, vocab=248320, n_rot=64,
              rope_theta=1e7, rms_eps=1e-6)
# the BASELINE cfg4 draft: a 0.6B-shaped q8_0 model (hidden 1024, FFN 3072,
# 28 layers; 16 query / 8 kv heads of 128, the target's vocabulary)
DRAFT = dict(n_layers=28, hidden=1024, ffn=3072, n_head=16, n_kv_head=8, head_dim=128, vocab=248320, n_rot=64,
             rope_theta=1e6, rms_eps=1e-6, weight_type=8)
# the reference's hybrid layout (include/mono27b_config.h:43-50; every 4th layer attention)
HYBRID = dict(attn_interval=4, ssm_d_inner=6144, ssm_d_state=128, ssm_dt_rank=48, ssm_n_group=16, ssm_conv_kern=4)


def model_config(max_ctx=1024, tp_rank=0, tp_size=1, **kw):
    d = dict(QWEN27)
    d.update(kw)
    return ModelConfig(max_ctx=max_ctx, tp_rank=tp_rank, tp_size=tp_size, **d)


def _engine_lib():
    L = lib()
    if getattr(L, "_engine_sigs", False):
        return L
    vp, cp, sz, i32, u32, b = ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint32, ctypes.c_bool
    sig = {
        "m27b_engine_partition": (b, [ctypes.POINTER(ModelConfig), ctypes.POINTER(Partition), cp, sz]),
        "m27b_nccl_unique_id": (b, [vp, cp, sz]),
        "m27b_engine_create": (b, [ctypes.POINTER(ModelConfig), ctypes.POINTER(vp), cp, sz]),
        "m27b_engine_set_nccl": (b, [vp, vp, cp, sz]),
        "m27b_engine_enable_p2p": (b, [vp, cp, sz]),
        "m27b_engine_load_tensor": (b, [vp, cp, u32, u32, u32, vp, cp, sz]),
        "m27b_engine_random_weights": (b, [vp, ctypes.c_uint64, ctypes.c_float, cp, sz]),
        "m27b_engine_weight_bytes_per_token": (sz, [vp]),
        "m27b_engine_reset": (b, [vp, cp, sz]),
        "m27b_engine_decode_step": (b, [vp, i32, i32, ctypes.POINTER(ctypes.c_int), vp, cp, sz]),
        "m27b_engine_generate": (b, [vp, i32, i32, i32, vp, cp, sz]),
        "m27b_engine_verify": (b, [vp, vp, i32, i32, vp, vp, cp, sz]),
        "m27b_engine_hidden": (b, [vp, vp, cp, sz]),
        "m27b_engine_stream": (vp, [vp]),
        "m27b_engine_destroy": (None, [vp]),
        "m27b_engine_create_sharing": (b, [vp, i32, ctypes.POINTER(vp), cp, sz]),
        "m27b_engine_speculative_generate": (b, [vp, vp, vp, i32, i32, i32, vp, ctypes.POINTER(SpecStats), cp, sz]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    L._engine_sigs = True
    return L


def partition(cfg):
    p = Partition()
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_engine_lib().m27b_engine_partition(ctypes.byref(cfg), ctypes.byref(p), err, ERR_CAP), err,
           "m27b_engine_partition")
    return p


def nccl_unique_id():
    buf = ctypes.create_string_buffer(128)
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_engine_lib().m27b_nccl_unique_id(buf, err, ERR_CAP), err, "m27b_nccl_unique_id")
    return buf.raw


class Engine:
    """One tensor-parallel rank of the decode engine on the current device."""

    def __init__(self, cfg):
        self.cfg = cfg
        self.L = _engine_lib()
        self.h = ctypes.c_void_p()
        self._call("m27b_engine_create", ctypes.byref(cfg), ctypes.byref(self.h))

    def _call(self, name, *args):
        err = ctypes.create_string_buffer(ERR_CAP)
        _check(getattr(self.L, name)(*args, err, ERR_CAP), err, name)

    def set_nccl(self, uid):
        buf = ctypes.create_string_buffer(bytes(uid), 128)
        self._call("m27b_engine_set_nccl", self.h, buf)

    def enable_p2p(self):
        """Fused NVLink all-reduce instead of NCCL (tp_size > 1; after set_nccl)."""
        self._call("m27b_engine_enable_p2p", self.h)

    def load_tensor(self, name, ggml_type, row_elems, row_count, data):
        import numpy as np
        a = np.ascontiguousarray(data)
        self._call("m27b_engine_load_tensor", self.h, name.encode(), ggml_type, row_elems, row_count,
                   ctypes.c_void_p(a.ctypes.data))

    def load_blob(self, blob, source=1):
        """Load a .m27b blob's entries of `source` (a Blob, or a path)."""
        b = blob if isinstance(blob, Blob) else Blob(blob)
        engine_load_blob(self, b, source)

    def random_weights(self, seed=0, sigma=0.02):
        self._call("m27b_engine_random_weights", self.h, seed, ctypes.c_float(sigma))

    def weight_bytes_per_token(self):
        return self.L.m27b_engine_weight_bytes_per_token(self.h)

    def decode_step(self, token, pos, logits=False):
        import numpy as np
        nxt = ctypes.c_int(-1)
        lg = np.empty(self.cfg.vocab, dtype=np.float32) if logits else None
        self._call("m27b_engine_decode_step", self.h, int(token), int(pos), ctypes.byref(nxt),
                   ctypes.c_void_p(lg.ctypes.data) if logits else None)
        return (nxt.value, lg) if logits else nxt.value

    def reset(self):
        """Start a new sequence: the DeltaNet states return to zero (attention needs nothing)."""
        self._call("m27b_engine_reset", self.h)

    def generate(self, token, pos, n):
        """Greedy tokens of steps pos..pos+n-1 (step i consumes step i-1's token), all on the device."""
        import numpy as np
        out = np.empty(n, dtype=np.int32)
        self._call("m27b_engine_generate", self.h, int(token), int(pos), int(n), ctypes.c_void_p(out.ctypes.data))
        return out

    def verify(self, tokens, pos, logits=False):
        """Greedy next token after each of `tokens` (at positions pos, pos+1, ...), one pass."""
        import numpy as np
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        nxt = np.empty(len(t), dtype=np.int32)
        lg = np.empty((len(t), self.cfg.vocab), dtype=np.float32) if logits else None
        self._call("m27b_engine_verify", self.h, ctypes.c_void_p(t.ctypes.data), len(t), int(pos),
                   ctypes.c_void_p(nxt.ctypes.data), ctypes.c_void_p(lg.ctypes.data) if logits else None)
        return (nxt, lg) if logits else nxt

    def stream(self):
        """The engine's cudaStream_t as an integer handle."""
        return self.L.m27b_engine_stream(self.h)

    def hidden(self):
        import numpy as np
        out = np.empty(self.cfg.hidden, dtype=np.float32)
        self._call("m27b_engine_hidden", self.h, ctypes.c_void_p(out.ctypes.data))
        return out

    def close(self):
        if self.h:
            self.L.m27b_engine_destroy(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# --------------------------------------------------------------------------
# .m27b blobs (include/m27b_blob.h)

SOURCE_TARGET, SOURCE_DRAFT = 1, 2
ROLE_NONE, ROLE_TARGET_MATVEC, ROLE_DRAFT_MATVEC, ROLE_OUTPUT_HEAD = 0, 1, 2, 3


class BlobHeader(ctypes.Structure):
    _fields_ = [("magic", ctypes.c_uint32), ("schema_version", ctypes.c_uint32), ("section_count", ctypes.c_uint32),
                ("reserved0", ctypes.c_uint32), ("file_bytes", ctypes.c_uint64), ("tensor_table_offset", ctypes.c_uint64),
                ("section_table_offset", ctypes.c_uint64), ("tokenizer_offset", ctypes.c_uint64),
                ("tokenizer_bytes", ctypes.c_uint64), ("max_ctx_hint", ctypes.c_uint32),
                ("target_layers", ctypes.c_uint32), ("draft_layers", ctypes.c_uint32), ("target_arch", ctypes.c_char * 16),
                ("draft_arch", ctypes.c_char * 16), ("target_quant", ctypes.c_char * 16),
                ("draft_quant", ctypes.c_char * 16)]


class WeightEntry(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 64), ("ggml_type", ctypes.c_uint32), ("source_model", ctypes.c_uint32),
                ("role", ctypes.c_uint32), ("row_elems", ctypes.c_uint32), ("row_count", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("data_offset", ctypes.c_uint64), ("data_bytes", ctypes.c_uint64)]


class PackTensor(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("ggml_type", ctypes.c_uint32), ("source", ctypes.c_uint32),
                ("role", ctypes.c_uint32), ("row_elems", ctypes.c_uint32), ("row_count", ctypes.c_uint32),
                ("data", ctypes.c_void_p), ("bytes", ctypes.c_uint64)]


class PackInfo(ctypes.Structure):
    _fields_ = [("max_ctx_hint", ctypes.c_uint32), ("target_layers", ctypes.c_uint32), ("draft_layers", ctypes.c_uint32),
                ("target_arch", ctypes.c_char_p), ("draft_arch", ctypes.c_char_p), ("target_quant", ctypes.c_char_p),
                ("draft_quant", ctypes.c_char_p), ("vocab_size", ctypes.c_uint32), ("bos_id", ctypes.c_uint32),
                ("eos_id", ctypes.c_uint32), ("im_start_id", ctypes.c_uint32), ("im_end_id", ctypes.c_uint32)]


def _blob_lib():
    L = lib()
    if getattr(L, "_blob_sigs", False):
        return L
    vp, cp, sz, b = ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t, ctypes.c_bool
    L.m27b_blob_pack.restype = b
    L.m27b_blob_pack.argtypes = [cp, ctypes.POINTER(PackInfo), ctypes.POINTER(PackTensor), sz, cp, sz]
    L.m27b_blob_open.restype = b
    L.m27b_blob_open.argtypes = [cp, ctypes.POINTER(vp), cp, sz]
    L.m27b_blob_header.restype = ctypes.POINTER(BlobHeader)
    L.m27b_blob_header.argtypes = [vp]
    L.m27b_blob_count.restype = sz
    L.m27b_blob_count.argtypes = [vp]
    L.m27b_blob_entry.restype = b
    L.m27b_blob_entry.argtypes = [vp, sz, ctypes.POINTER(WeightEntry), ctypes.POINTER(vp), cp, sz]
    L.m27b_blob_close.restype = None
    L.m27b_blob_close.argtypes = [vp]
    L.m27b_engine_load_blob.restype = b
    L.m27b_engine_load_blob.argtypes = [vp, vp, ctypes.c_uint32, cp, sz]
    L._blob_sigs = True
    return L


def blob_pack(path, tensors, max_ctx_hint=8192, target_layers=0, draft_layers=0, target_arch="qwen35",
              draft_arch="dflash-draft", target_quant="q4_k_m", draft_quant="q8_0", vocab_size=1, bos_id=0, eos_id=0,
              im_start_id=0, im_end_id=0):
    """Write a .m27b blob.  tensors: iterable of dicts with name, ggml_type,
    data (numpy bytes in GGUF layout or fp32), row_elems, row_count and
    optionally source (default target) and role (default: output head for
    output.weight, target/draft matvec for quantized 2-D tensors, 0 otherwise)."""
    import numpy as np
    keep, arr = [], []
    for t in tensors:
        d = np.ascontiguousarray(t["data"])
        keep.append(d)
        src = t.get("source", SOURCE_TARGET)
        role = t.get("role")
        if role is None:
            if t["name"] == "output.weight":
                role = ROLE_OUTPUT_HEAD
            elif t["ggml_type"] != F32 and t["row_count"] > 1:
                role = ROLE_TARGET_MATVEC if src == SOURCE_TARGET else ROLE_DRAFT_MATVEC
            else:
                role = ROLE_NONE
        arr.append(PackTensor(t["name"].encode(), t["ggml_type"], src, role, t["row_elems"], t["row_count"],
                              ctypes.c_void_p(d.ctypes.data), d.nbytes))
    tarr = (PackTensor * len(arr))(*arr)
    info = PackInfo(max_ctx_hint, target_layers, draft_layers, target_arch.encode(), draft_arch.encode(),
                    target_quant.encode(), draft_quant.encode(), vocab_size, bos_id, eos_id, im_start_id, im_end_id)
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_blob_lib().m27b_blob_pack(str(path).encode(), ctypes.byref(info), tarr, len(arr), err, ERR_CAP), err,
           "m27b_blob_pack")


class Blob:
    """A mapped, validated .m27b blob."""

    def __init__(self, path):
        self.L = _blob_lib()
        self.h = ctypes.c_void_p()
        err = ctypes.create_string_buffer(ERR_CAP)
        _check(self.L.m27b_blob_open(str(path).encode(), ctypes.byref(self.h), err, ERR_CAP), err, "m27b_blob_open")

    @property
    def header(self):
        return self.L.m27b_blob_header(self.h).contents

    def __len__(self):
        return self.L.m27b_blob_count(self.h)

    def entry(self, i):
        """(WeightEntry, payload as a read-only numpy uint8 view of the mapping)."""
        import numpy as np
        e = WeightEntry()
        p = ctypes.c_void_p()
        err = ctypes.create_string_buffer(ERR_CAP)
        _check(self.L.m27b_blob_entry(self.h, i, ctypes.byref(e), ctypes.byref(p), err, ERR_CAP), err,
               "m27b_blob_entry")
        buf = (ctypes.c_uint8 * e.data_bytes).from_address(p.value)
        return e, np.frombuffer(buf, dtype=np.uint8)

    def entries(self):
        return [self.entry(i) for i in range(len(self))]

    def close(self):
        if self.h:
            self.L.m27b_blob_close(self.h)
            self.h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def engine_load_blob(engine, blob, source=SOURCE_TARGET):
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_blob_lib().m27b_engine_load_blob(engine.h, blob.h, source, err, ERR_CAP), err, "m27b_engine_load_blob")


# --------------------------------------------------------------------------
# speculative decoding (draft engine + target engine, greedy)


class SpecStats(ctypes.Structure):
    """M27BSpecStats (include/m27b_engine.h)."""
    _fields_ = [("iterations", ctypes.c_int), ("proposed", ctypes.c_int), ("accepted", ctypes.c_int),
                ("prefill_ms", ctypes.c_double), ("draft_ms", ctypes.c_double), ("verify_ms", ctypes.c_double)]


def speculative_generate(target, draft, prompt, n_new, k=7):
    """Greedy speculative decoding through m27b_engine_speculative_generate
    (the loop runs in the library): the draft proposes k tokens, the target
    verifies k + 1 in one pass and keeps the longest agreeing prefix plus its
    own next token.  Lossless: equals the target's greedy decoding of
    `prompt`.  Both engines must start empty; returns (tokens, stats)."""
    import numpy as np
    p = np.ascontiguousarray(prompt, dtype=np.int32)
    out = np.empty(n_new, dtype=np.int32)
    st = SpecStats()
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_engine_lib().m27b_engine_speculative_generate(target.h, draft.h, ctypes.c_void_p(p.ctypes.data), len(p),
                                                          int(n_new), int(k), ctypes.c_void_p(out.ctypes.data),
                                                          ctypes.byref(st), err, ERR_CAP),
           err, "m27b_engine_speculative_generate")
    stats = {f: getattr(st, f) for f, _ in SpecStats._fields_}
    return [int(t) for t in out], stats


M27B_VERIFY_MAX = 16

# --------------------------------------------------------------------------
# paged key/value cache (include/m27b_paged.h)

BF16, I32 = 30, 26
ROPE_NONE, ROPE_LINEAR, ROPE_YARN = 0, 1, 2
PAGES_FULL, PAGES_BAD = 1, 2


class _PagedKV(ctypes.Structure):
    """M27BPagedKV"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p), ("type", ctypes.c_uint32),
                ("n_pages", ctypes.c_int), ("page_size", ctypes.c_int), ("n_kv", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("n_rows", ctypes.c_int), ("n_cols", ctypes.c_int),
                ("page_stride", ctypes.c_longlong)]


# Small by-reference arguments of the calls a decode step makes, packed as C
# lays them out (a bytes object is passed as the pointer to it; packing one
# takes a third of the time of filling a ctypes.Structure).
_PagedBatch = struct.Struct("@PPPii")               # M27BPagedBatch: cu_q, lens, rows, n_seq, n_tok
_Rope = struct.Struct("@PiiiP")                     # M27BRope: table, n_pos, n_rot, interleaved, positions
_Heads = struct.Struct("@PPPqqqIiPPf4x")            # M27BHeads: q, k, v, strides, src_type, n_q, q_norm, k_norm, eps


class _RopeScaling(ctypes.Structure):
    """M27BRopeScaling"""
    _fields_ = [("kind", ctypes.c_int), ("factor", ctypes.c_float), ("original_ctx", ctypes.c_int),
                ("beta_fast", ctypes.c_float), ("beta_slow", ctypes.c_float), ("attn_factor", ctypes.c_float)]


class _Pages(ctypes.Structure):
    """M27BPages"""
    _fields_ = [("ref", ctypes.c_void_p), ("table", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("n_pages", ctypes.c_int), ("page_size", ctypes.c_int), ("n_rows", ctypes.c_int),
                ("n_cols", ctypes.c_int)]


class _PagePool(ctypes.Structure):
    """M27BPagePool"""
    _fields_ = [("base", ctypes.c_void_p), ("n_planes", ctypes.c_int), ("plane_stride", ctypes.c_size_t),
                ("page_stride", ctypes.c_size_t), ("page_bytes", ctypes.c_size_t)]


_paged = None


def _paged_lib():
    global _paged
    if _paged is not None and _paged is _lib:
        return _paged
    L = lib()
    vp, cp, sz, i32, ll, b = (ctypes.c_void_p, ctypes.c_char_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_longlong,
                              ctypes.c_bool)
    kv, pg, pool = (ctypes.POINTER(t) for t in (_PagedKV, _Pages, _PagePool))
    sig = {
        "m27b_rope_table": (b, [vp, i32, i32, ctypes.c_double, ctypes.POINTER(_RopeScaling), vp, cp, sz]),
        "m27b_rope_append": (b, [kv, cp, cp, cp, vp, ll, vp, cp, sz]),
        "m27b_paged_attn_scratch_bytes": (sz, [i32, i32, i32]),
        "m27b_paged_attn": (b, [kv, cp, vp, ll, i32, ctypes.c_float, i32, vp, ll, vp, vp, vp, cp, sz]),
        "m27b_pages_scratch_bytes": (sz, [i32, i32, i32]),
        "m27b_pages_resize": (b, [pg, pool, i32, vp, vp, i32, vp, vp, vp, cp, sz]),
        "m27b_pages_fork": (b, [pg, pool, i32, vp, vp, i32, vp, vp, vp, cp, sz]),
        "m27b_pages_free": (b, [pg, vp, i32, vp, cp, sz]),
        "m27b_pages_compact": (b, [pg, pool, i32, vp, vp, vp, cp, sz]),
        "m27b_pages_copy": (b, [pool, i32, i32, vp, vp, i32, vp, cp, sz]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _paged = L
    return L


_types = {}  # torch type -> ggml code, filled at the first use (torch is imported late)


def _paged_type(dtype):
    if not _types:
        import torch
        _types.update({torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32, torch.int32: I32})
    t = _types.get(dtype)
    if t is None:
        raise M27BError(f"paged cache: unsupported type {dtype} (f16, bf16; f32 and int32 where named)")
    return t


def _f32(t, dev):
    """A contiguous fp32 tensor on device `dev`?"""
    return t.get_device() == dev and _paged_type(t.dtype) == F32 and t.is_contiguous()


# A decode step makes these calls once per layer on a few rows, so what they
# cost on the host counts: plain attribute reads, one error buffer per thread,
# the current stream's handle without a Stream object.
_tls = threading.local()


def _err():
    try:
        return _tls.err
    except AttributeError:
        _tls.err = ctypes.create_string_buffer(ERR_CAP)
        return _tls.err


def _raw_stream(stream, dev):
    """The handle of `stream` or the current one.  The C entries work on the
    current device, so that has to be the tensors' (`dev`), and the stream's."""
    import torch
    cur = torch._C._cuda_getDevice()
    if cur != dev or (stream is not None and stream.device_index != dev):
        raise M27BError(f"paged cache: the tensors are on device {dev}, the current device is {cur}"
                        + ("" if stream is None else f", the stream's {stream.device_index}"))
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


def _int32(t, what, n=0, dev=None):
    """The data pointer of a contiguous int32 tensor on device `dev` (None: any; 0 for no tensor)."""
    if t is None:
        return 0
    d = t.get_device()
    if d < 0 or _paged_type(t.dtype) != I32 or t.numel() < n or not t.is_contiguous():
        raise M27BError(f"{what} must be a contiguous int32 device tensor" + (f" of at least {n} values" if n else ""))
    if dev is not None and d != dev:
        raise M27BError(f"{what} is on device {d}, the cache on device {dev}")
    return t.data_ptr()


def _token_heads(t, what, n_tok, n_head, head_dim, dtype, dev):
    """(pointer, token stride) of [n_tok, n_head, head_dim] rows on device `dev` whose heads are contiguous."""
    if t.shape != (n_tok, n_head, head_dim) or t.dtype != dtype or t.get_device() != dev:
        raise M27BError(f"{what} must be a tensor [{n_tok}, {n_head}, {head_dim}] of {dtype} on device {dev} "
                        f"(got {list(t.shape)} of {t.dtype} on {t.get_device()})")
    s = t.stride()
    if s[2] != 1 or (s[1] != head_dim and n_head > 1):
        raise M27BError(f"{what}: a token's heads must be contiguous (strides {s})")
    return t.data_ptr(), s[0] if n_tok > 1 else n_head * head_dim


def _no_grad(what, *tensors):
    """As torch's functions with out=: results in given buffers carry no gradient."""
    for t in tensors:
        if t is not None and t.requires_grad:
            import torch
            if torch.is_grad_enabled():
                raise M27BError(f"{what} has no backward pass, and a tensor given to it requires grad (use torch.no_grad())")
            return


class PagedKV:
    """One layer's pools of a paged cache, with the page table.

    k, v: device tensors [n_pages, page_size, n_kv, head_dim] in f16 or bf16,
    contiguous but for the first stride (the pools of several layers may
    interleave); table: int32 [n_rows, n_cols] page ids."""

    def __init__(self, k, v, table):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise M27BError("PagedKV: k and v must be [n_pages, page_size, n_kv, head_dim] of one type and layout")
        n_pages, page_size, n_kv, head_dim = k.shape
        s = k.stride()
        want = (n_kv * head_dim, head_dim, 1)
        if any(n > 1 and a != b for n, a, b in zip(k.shape[1:], s[1:], want)) or not k.is_cuda or not v.is_cuda:
            raise M27BError(f"PagedKV: a page must be contiguous on the device (strides {s})")
        if table.dim() != 2:
            raise M27BError("PagedKV: table must be [n_rows, n_cols]")
        self.k, self.v, self.table = k, v, table
        self.n_kv, self.head_dim, self.dtype, self.dev = n_kv, head_dim, k.dtype, k.get_device()
        if v.get_device() != self.dev:
            raise M27BError(f"PagedKV: k is on device {self.dev}, v on device {v.get_device()}")
        self.c = _PagedKV(k.data_ptr(), v.data_ptr(), _int32(table, "table", 0, self.dev), _paged_type(k.dtype), n_pages, page_size,
                          n_kv, head_dim, table.shape[0], table.shape[1],
                          s[0] if n_pages > 1 else page_size * n_kv * head_dim)
        self._ref = ctypes.byref(self.c)
        _paged_lib()


def _batch(kv, cu_q, lens, rows, n_tok):
    n_seq = cu_q.numel() - 1
    if n_seq < 0:
        raise M27BError("cu_q needs n_seq + 1 values")
    return _PagedBatch.pack(_int32(cu_q, "cu_q", 0, kv.dev),
                            _int32(lens, "lens", kv.c.n_rows if rows is not None else n_seq, kv.dev),
                            _int32(rows, "rows", n_seq, kv.dev), n_seq, n_tok)


def rope_table(n_pos, n_rot, theta, kind=ROPE_NONE, factor=1.0, original_ctx=0, beta_fast=32.0, beta_slow=1.0,
               attn_factor=0.0, device="cuda", stream=None):
    """cos / sin of every position's rotary angles, fp32 [n_pos, n_rot / 2, 2] (m27b_rope_table)."""
    import torch
    if n_pos < 1 or n_rot < 2 or n_rot % 2:
        raise M27BError(f"rope_table: bad n_pos ({n_pos}) or n_rot ({n_rot})")
    # allocated on the stream that writes it: memory that work on another one is
    # still to use is not handed out there
    with torch.cuda.stream(stream):
        out = torch.empty(n_pos, n_rot // 2, 2, dtype=torch.float32, device=device)
    s = _RopeScaling(kind, factor, original_ctx, beta_fast, beta_slow, attn_factor)
    err = ctypes.create_string_buffer(ERR_CAP)
    _check(_paged_lib().m27b_rope_table(_ptr(out), n_pos, n_rot, theta, ctypes.byref(s),
                                        _raw_stream(stream, out.get_device()), err, ERR_CAP), err, "m27b_rope_table")
    return out


def rope_append(kv, q, k, v, cu_q, lens, rope, q_out, interleaved=False, q_norm=None, k_norm=None, eps=1e-6, rows=None,
                positions=None, stream=None):
    """Head RMSNorm and rotary positions of the new tokens' q [n_tok, n_q, hd]
    and k [n_tok, n_kv, hd]; q goes to q_out, k and v to the tokens' slots of
    the cache (m27b_rope_append).  cu_q [n_seq + 1]: each sequence's token
    rows; lens: positions of each table row, the new ones included; rope: a
    table of rope_table.  q may be None (append only).  No backward pass."""
    dt, n_kv, hd, dev = k.dtype, kv.n_kv, kv.head_dim, kv.dev
    n_tok = k.shape[0]
    _no_grad("rope_append", q, k, v, q_norm, k_norm)
    kp, ks = _token_heads(k, "k", n_tok, n_kv, hd, dt, dev)
    vp, vs = _token_heads(v, "v", n_tok, n_kv, hd, dt, dev)
    n_q = qp = op = qs = os_ = 0
    if q is not None:
        n_q = q.shape[1]
        qp, qs = _token_heads(q, "q", n_tok, n_q, hd, dt, dev)
        op, os_ = _token_heads(q_out, "q_out", n_tok, n_q, hd, kv.dtype, dev)
    n_pos, half, two = rope.shape
    if two != 2 or not _f32(rope, dev):
        raise M27BError(f"rope must be an fp32 table [n_pos, n_rot / 2, 2] on device {dev}")
    if (q_norm is not None and (q_norm.numel() != hd or not _f32(q_norm, dev))) or \
            (k_norm is not None and (k_norm.numel() != hd or not _f32(k_norm, dev))):
        raise M27BError(f"q_norm and k_norm must be {hd} fp32 values on device {dev}")
    bt = _batch(kv, cu_q, lens, rows, n_tok)
    rp = _Rope.pack(rope.data_ptr(), n_pos, 2 * half, 1 if interleaved else 0, _int32(positions, "positions", n_tok, dev))
    h = _Heads.pack(qp, kp, vp, qs, ks, vs, _paged_type(dt), n_q, 0 if q_norm is None else q_norm.data_ptr(),
                    0 if k_norm is None else k_norm.data_ptr(), eps)
    err = _err()
    if not _paged_lib().m27b_rope_append(kv._ref, bt, rp, h, op, os_, _raw_stream(stream, dev), err,
                                         ERR_CAP):
        _check(False, err, "m27b_rope_append")
    return q_out


def paged_attn_scratch(n_q, n_kv, head_dim, device="cuda"):
    """Scratch of paged_attn (one for each stream that calls it)."""
    import torch
    n = _paged_lib().m27b_paged_attn_scratch_bytes(n_q, n_kv, head_dim)
    if n == 0:
        raise M27BError(f"paged_attn: unsupported heads ({n_q} on {n_kv}, head_dim {head_dim})")
    return torch.empty(n, dtype=torch.uint8, device=device)


def paged_attn(kv, q, cu_q, lens, out, scratch, scale=None, window=0, lse=None, rows=None, stream=None):
    """Causal attention of the new tokens q [n_tok, n_q, hd] over the cache
    (m27b_paged_attn): one token or many per sequence, the newest at position
    lens - 1; window > 0 limits a token to the last `window` positions; lse
    [n_tok, n_q] fp32 receives the log sum of exponentials.  scale defaults to
    1 / sqrt(hd).  No backward pass."""
    hd, dt, dev = kv.head_dim, kv.dtype, kv.dev
    n_tok, n_q, _ = q.shape
    _no_grad("paged_attn", q, kv.k, kv.v)
    qp, qs = _token_heads(q, "q", n_tok, n_q, hd, dt, dev)
    op, os_ = _token_heads(out, "out", n_tok, n_q, hd, dt, dev)
    L = _paged_lib()
    need = L.m27b_paged_attn_scratch_bytes(n_q, kv.n_kv, hd)
    # contiguous: an expanded tensor has more values than memory
    if scratch.get_device() != dev or not scratch.is_contiguous() or scratch.numel() * scratch.element_size() < need:
        raise M27BError(f"paged_attn: scratch must be {need} contiguous bytes on device {dev} (use paged_attn_scratch)")
    lp = None
    if lse is not None:
        if lse.numel() != n_tok * n_q or not _f32(lse, dev):
            raise M27BError(f"lse must be {n_tok} x {n_q} fp32 values on device {dev}")
        lp = lse.data_ptr()
    bt = _batch(kv, cu_q, lens, rows, n_tok)
    err = _err()
    if not L.m27b_paged_attn(kv._ref, bt, qp, qs, n_q, hd ** -0.5 if scale is None else scale, window, op, os_, lp,
                             scratch.data_ptr(), _raw_stream(stream, dev), err, ERR_CAP):
        _check(False, err, "m27b_paged_attn")
    return out


class PageSet:
    """The pages of a paged cache: which rows of `table` hold which pages, how
    many hold each (`ref`, int32 [n_pages]; free where it is 0) and the rows'
    lengths (`lens`, int32 [n_rows]).

    pool: the data, a device tensor (or up to two, one for keys and one for
    values) [n_planes, n_pages, ...] whose pages are contiguous; a plane is a
    layer's keys or values.  Requests are device int32 tensors.  A refused
    request (too few free pages, or a bad one) changes nothing and shows in
    check(); rope_append must not follow a refused resize, since the lengths are
    still the old ones.  The set has one scratch and one status word: its calls
    belong on one stream at a time."""

    def __init__(self, table, ref, lens, page_size, pool, max_requests=None):
        import torch
        if table.dim() != 2 or lens.numel() != table.shape[0]:
            raise M27BError("PageSet: table must be [n_rows, n_cols], lens [n_rows]")
        self.table, self.ref, self.lens, self.page_size = table, ref, lens, page_size
        self.pools = list(pool) if isinstance(pool, (list, tuple)) else [pool]
        n_pages, self.dev = ref.numel(), ref.get_device()
        arr = []
        for p in self.pools:
            if p.dim() < 3 or p.shape[1] != n_pages or p.get_device() != self.dev or not p[0, 0].is_contiguous():
                raise M27BError(f"PageSet: a pool is [n_planes, {n_pages}, ...] on ref's device ({self.dev}), its pages contiguous")
            es = p.element_size()
            page_bytes = p[0, 0].numel() * es
            arr.append(_PagePool(p.data_ptr(), p.shape[0], p.stride(0) * es if p.shape[0] > 1 else 0,
                                 p.stride(1) * es if n_pages > 1 else page_bytes, page_bytes))
        self._pools = (_PagePool * len(arr))(*arr)
        self.c = _Pages(_int32(ref, "ref"), _int32(table, "table", 0, self.dev), _int32(lens, "lens", 0, self.dev), n_pages, page_size,
                        table.shape[0], table.shape[1])
        self._ref = ctypes.byref(self.c)
        self.max_requests = table.shape[0] if max_requests is None else max_requests
        L = _paged_lib()
        self._scratch = torch.empty(L.m27b_pages_scratch_bytes(n_pages, table.shape[0], self.max_requests),
                                    dtype=torch.uint8, device=ref.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=ref.device)

    @classmethod
    def empty(cls, n_rows, n_cols, n_pages, page_size, pool, device="cuda"):
        """A cache that holds nothing."""
        import torch
        return cls(torch.full((n_rows, n_cols), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device),
                   torch.zeros(n_rows, dtype=torch.int32, device=device), page_size, pool)

    def _call(self, name, *args, stream=None):
        err = _err()
        if not getattr(_paged_lib(), name)(*args, _raw_stream(stream, self.dev), err, ERR_CAP):
            _check(False, err, name)

    def _requests(self, a, b, names):
        n = a.numel()
        if n > self.max_requests or (b is not None and b.numel() != n):
            raise M27BError(f"PageSet: {names}: at most {self.max_requests} requests, as many of each")
        return _int32(a, names, 0, self.dev), _int32(b, names, 0, self.dev), n

    def resize(self, rows, new_lens, stream=None):
        """Set the rows' lengths (m27b_pages_resize)."""
        a, b, n = self._requests(rows, new_lens, "rows and new_lens")
        self._call("m27b_pages_resize", self._ref, self._pools, len(self._pools), a, b, n, self._scratch.data_ptr(),
                   self.status.data_ptr(), stream=stream)

    def fork(self, src, dst, stream=None):
        """Make the empty rows dst copies of the rows src (m27b_pages_fork)."""
        a, b, n = self._requests(src, dst, "src and dst")
        self._call("m27b_pages_fork", self._ref, self._pools, len(self._pools), a, b, n, self._scratch.data_ptr(),
                   self.status.data_ptr(), stream=stream)

    def free(self, rows, stream=None):
        """Empty the rows (m27b_pages_free)."""
        self._call("m27b_pages_free", self._ref, _int32(rows, "rows", 0, self.dev), rows.numel(), stream=stream)

    def compact(self, n_live=None, stream=None):
        """Move the pages in use to the lowest ids (m27b_pages_compact); n_live, an int32 device tensor, receives their number."""
        self._call("m27b_pages_compact", self._ref, self._pools, len(self._pools), _int32(n_live, "n_live", 1, self.dev),
                   self._scratch.data_ptr(), stream=stream)

    def copy(self, src, dst, stream=None):
        """Copy page src[i] to page dst[i] in every plane (m27b_pages_copy)."""
        if src.numel() != dst.numel():
            raise M27BError("PageSet: src and dst need as many pages")
        self._call("m27b_pages_copy", self._pools, len(self._pools), self.c.n_pages, _int32(src, "src", 0, self.dev),
                   _int32(dst, "dst", 0, self.dev), src.numel(), stream=stream)

    def check(self):
        """Raise if a request was refused since the last check (reads the device)."""
        s = int(self.status.item())
        if s:
            self.status.zero_()
            raise M27BError("PageSet: " + {PAGES_FULL: "too few free pages"}.get(s, "bad request (row, length, or a row named twice)"))
