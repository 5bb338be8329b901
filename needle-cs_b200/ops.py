"""Tensor-level wrappers over the C ABI.

torch is plumbing here: device memory, the current CUDA stream and shape
bookkeeping.  All arithmetic happens in libneedle_b200.so.  Every wrapper
checks device, dtype and contiguity before handing raw pointers to the ABI.
"""
import numpy as np
import torch

from ._native import call, lib


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dev(t, dtype, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


# ---------------------------------------------------------------- synth --

def synth_normal_f32(seed, stream, count, scale=1.0, first=0):
    out = np.empty(count, np.float32)
    lib().ndl_synth_normal_f32(seed, stream, first, count, scale, out.ctypes.data)
    return out


def synth_normal_f16(seed, stream, count, scale=1.0, first=0):
    out = np.empty(count, np.uint16)
    lib().ndl_synth_normal_f16(seed, stream, first, count, scale, out.ctypes.data)
    return out


def synth_uniform_f16(seed, stream, count, lo, hi, first=0):
    out = np.empty(count, np.uint16)
    lib().ndl_synth_uniform_f16(seed, stream, first, count, lo, hi, out.ctypes.data)
    return out


def synth_int8(seed, stream, count, first=0):
    out = np.empty(count, np.int8)
    lib().ndl_synth_int8(seed, stream, first, count, out.ctypes.data)
    return out


def synth_normal_f32_device(seed, stream, out, scale=1.0, first=0):
    call("ndl_synth_normal_f32_device", seed, stream, first, out.numel(), scale, _dev(out, torch.float32, "out"),
         _stream())


def synth_normal_f16_device(seed, stream, out, scale=1.0, first=0):
    call("ndl_synth_normal_f16_device", seed, stream, first, out.numel(), scale, _dev(out, torch.int16, "out"),
         _stream())


def synth_uniform_f16_device(seed, stream, out, lo, hi, first=0):
    call("ndl_synth_uniform_f16_device", seed, stream, first, out.numel(), lo, hi, _dev(out, torch.int16, "out"),
         _stream())


def synth_int8_device(seed, stream, out, first=0):
    call("ndl_synth_int8_device", seed, stream, first, out.numel(), _dev(out, torch.int8, "out"), _stream())


# -------------------------------------------------------------- kernels --

def quantize_rows(x, q=None, scales=None):
    """Per-row int8 quantizer (Quant.QuantizeInt8 per row)."""
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device) if q is None else q
    scales = torch.empty(rows, dtype=torch.float32, device=x.device) if scales is None else scales
    call("ndl_quantize_rows", _dev(x, torch.float32, "x"), rows, cols, _dev(q, torch.int8, "q"),
         _dev(scales, torch.float32, "scales"), _stream())
    return q, scales


def rmsnorm_quantize(x, weight, q=None, scales=None):
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.int8, device=x.device) if q is None else q
    scales = torch.empty(rows, dtype=torch.float32, device=x.device) if scales is None else scales
    call("ndl_rmsnorm_quantize", _dev(x, torch.float32, "x"), _dev(weight, torch.float32, "weight"), rows, cols,
         _dev(q, torch.int8, "q"), _dev(scales, torch.float32, "scales"), _stream())
    return q, scales


def matmul_i8g32(q, sa, w, sw, y=None, residual=None, acc=None):
    """I8G32 linear: y[t][n] = sa[t] * (fma chain over groups of half(sw[n][g]) * D[t][n][g]).

    q int8 [m,k], sa fp32 [m], w int8 [n,k], sw fp16 bits as int16 [n,k/32].
    """
    m, k = q.shape
    n = w.shape[0]
    y = torch.empty((m, n), dtype=torch.float32, device=q.device) if y is None else y
    res_ptr = _dev(residual, torch.float32, "residual") if residual is not None else None
    acc_ptr = _dev(acc, torch.int32, "acc") if acc is not None else None
    call("ndl_matmul_i8g32", _dev(q, torch.int8, "q"), _dev(sa, torch.float32, "sa"), m,
         _dev(w, torch.int8, "w"), _dev(sw, torch.int16, "sw"), n, k, _dev(y, torch.float32, "y"), y.stride(0),
         res_ptr, acc_ptr, _stream())
    return y


def matmul_i8g32_batched(q, sa, w, sw, y):
    """Batched I8G32 linear over weight sets w [B,n,k], sw [B,n,k/32] -> y [B,m,n]."""
    m, k = q.shape
    batch, n, _ = w.shape
    call("ndl_matmul_i8g32_batched", _dev(q, torch.int8, "q"), _dev(sa, torch.float32, "sa"), m,
         _dev(w, torch.int8, "w"), _dev(sw, torch.int16, "sw"), n, k, batch, n * k, n * (k // 32),
         _dev(y, torch.float32, "y"), n, m * n, _stream())
    return y


def cq_prepare(x, bits, values=None, scales=None, offsets=None):
    """Quant.Prepare for CQ weights: per (token, 128 columns) FWHT, int8
    quantize and plane reorder.  x fp32 [tokens, cols] -> (values int8
    [tokens, cols], scales and offsets fp32 [tokens, stride])."""
    tokens, cols = x.shape
    stride = ((cols // 128) + 7) & ~7
    values = torch.empty((tokens, cols), dtype=torch.int8, device=x.device) if values is None else values
    scales = torch.empty((tokens, stride), dtype=torch.float32, device=x.device) if scales is None else scales
    offsets = torch.empty((tokens, stride), dtype=torch.float32, device=x.device) if offsets is None else offsets
    call("ndl_cq_prepare", _dev(x, torch.float32, "x"), tokens, cols, bits, _dev(values, torch.int8, "values"),
         _dev(scales, torch.float32, "scales"), _dev(offsets, torch.float32, "offsets"), scales.stride(0),
         _stream())
    return values, scales, offsets


def cq_matmul(indices, norms, book_bytes, byte_scale, bits, values, scales, offsets, y=None):
    """MatMulRows on a CQ matrix: indices uint8 [rows, cols*bits/8], norms fp16
    bits as int16 [rows, cols/128], book_bytes the codebook's 16 level bytes
    (host); activations from cq_prepare -> y fp32 [tokens, rows]."""
    import ctypes

    rows = indices.shape[0]
    tokens, cols = values.shape
    y = torch.empty((tokens, rows), dtype=torch.float32, device=values.device) if y is None else y
    table = (ctypes.c_uint8 * 16).from_buffer_copy(bytes(book_bytes[:16]))
    call("ndl_cq_matmul", _dev(indices, torch.uint8, "indices"), _dev(norms, torch.int16, "norms"),
         ctypes.addressof(table), float(byte_scale), rows, cols, bits, _dev(values, torch.int8, "values"),
         _dev(scales, torch.float32, "scales"), _dev(offsets, torch.float32, "offsets"), scales.stride(0), tokens,
         _dev(y, torch.float32, "y"), y.stride(0), 0, rows, _stream())
    return y


def attention_paged_workspace(rows, heads, max_pages):
    return lib().ndl_attention_paged_workspace(rows, heads, max_pages)


def attention_paged(q8, qs, row_slot, row_pos, page_table, pool, page_bytes, layer, out=None, workspace=None,
                    status=None):
    """Paged int8 decode attention (ndl_attention_paged).

    q8 int8 [rows,heads,64] in the page K dim order, qs fp32 [rows,heads],
    row_slot/row_pos int32 [rows], page_table int32 [slots,max_pages],
    pool uint8 [num_pages*page_bytes]; out fp32 [rows,heads,64]."""
    rows, heads, _ = q8.shape
    slots, max_pages = page_table.shape
    out = torch.empty((rows, heads, 64), dtype=torch.float32, device=q8.device) if out is None else out
    ws_ptr, ws_bytes = (None, 0) if workspace is None else (_dev(workspace, torch.uint8, "workspace"),
                                                             workspace.numel())
    call("ndl_attention_paged", _dev(q8, torch.int8, "q8"), _dev(qs, torch.float32, "qs"),
         _dev(row_slot, torch.int32, "row_slot"), _dev(row_pos, torch.int32, "row_pos"), rows, heads,
         _dev(page_table, torch.int32, "page_table"), slots, max_pages, _dev(pool, torch.uint8, "pool"), page_bytes,
         pool.numel() // page_bytes, layer, _dev(out, torch.float32, "out"), ws_ptr, ws_bytes,
         _dev(status, torch.int32, "status") if status is not None else None, _stream())
    return out


# ------------------------------- rows, attention and logits over own pages --

# A call's checks read each tensor attribute once: they are most of a small call's time on the host.

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8


def _start(t, name, types=_TYPES):
    """(element type code, device index) of the operand that decides a call's type and device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    code = types.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be one of {list(types)}, got {t.dtype}")
    return code, t.get_device()


def _wrong(t, dtype, name, index, numel=None):
    """What keeps an operand from being a contiguous `dtype` tensor of `numel` elements on the device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must have {numel} elements, got {t.numel()}")
    raise ValueError(f"{name} must be contiguous")


def _heads(t, dtype, name, index, shape=None):
    """Address and row stride of a [rows, heads, 64] operand whose rows may be strided (a projection's columns)."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index:
        _wrong(t, dtype, name, index)
    if t.dim() != 3 or t.shape[2] != 64 or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be [rows, heads, 64]{'' if shape is None else f' = {list(shape)}'}, got {list(t.shape)}")
    rows, heads, _ = t.shape
    if t.is_contiguous():
        return t.data_ptr(), heads * 64
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != 64):
        raise ValueError(f"{name}: a row's heads and dims must be contiguous")
    return t.data_ptr(), (t.stride(0) if rows > 1 else heads * 64)


def _vec(t, dtype, name, index, numel=None):
    """Address of a contiguous operand on the device (None passes through)."""
    if t is None:
        return None
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index or not t.is_contiguous()
            or (numel is not None and t.numel() != numel)):
        _wrong(t, dtype, name, index, numel)
    return t.data_ptr()


def _pages(page_table, pool, page_bytes, layer, index):
    """The cache arguments of the C entry points from the page table [slots, max_pages] on."""
    table, bytes_ = _vec(page_table, _I32, "page_table", index), _vec(pool, _U8, "pool", index)
    if table is None or bytes_ is None or page_table.dim() != 2:
        raise ValueError("page_table must be [slots, max_pages], and a pool is needed")
    if page_bytes <= 0:
        raise ValueError(f"page_bytes {page_bytes}")
    slots, max_pages = page_table.shape
    return table, slots, max_pages, bytes_, page_bytes, pool.numel() // page_bytes, layer


def _call_on(index, name, *args):
    """The call on the device's current stream (whichever device is current)."""
    if index == torch.cuda.current_device():
        return call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def kv_append(k, v, row_slot, row_pos, page_table, pool, page_bytes, layer, status=None):
    """Rows of keys and values into the pages (ndl_kv_append).

    k, v [rows, kv_heads, 64] of one type (float32, float16, bfloat16), rows
    possibly strided; row_slot, row_pos int32 [rows] (distinct positions; a
    negative position: padding); page_table int32 [slots, max_pages], pool
    uint8 [num_pages * page_bytes]."""
    code, index = _start(k, "k")
    kp, ks = _heads(k, k.dtype, "k", index)
    rows, kv_heads, _ = k.shape
    vp, vs = _heads(v, k.dtype, "v", index, k.shape)
    _call_on(index, "ndl_kv_append", kp, ks, vp, vs, code, _vec(row_slot, _I32, "row_slot", index, rows),
             _vec(row_pos, _I32, "row_pos", index, rows), rows, kv_heads,
             *_pages(page_table, pool, page_bytes, layer, index), _vec(status, _I32, "status", index))


def kv_gather(row_slot, row_pos, kv_heads, page_table, pool, page_bytes, layer, dtype=torch.float32, k=None, v=None,
              status=None):
    """The values the pages hold for the rows (ndl_kv_gather): k and v
    [rows, kv_heads, 64] of `dtype` (or of the tensors given)."""
    _, index = _start(pool, "pool", {_U8: 0})
    rows = row_slot.numel()
    shape = (rows, kv_heads, 64)
    k = pool.new_empty(shape, dtype=dtype) if k is None else k
    v = torch.empty_like(k, memory_format=torch.contiguous_format) if v is None else v
    code, _ = _start(k, "k")
    kp, ks = _heads(k, k.dtype, "k", index, shape)
    vp, vs = _heads(v, k.dtype, "v", index, shape)
    _call_on(index, "ndl_kv_gather", _vec(row_slot, _I32, "row_slot", index),
             _vec(row_pos, _I32, "row_pos", index, rows), rows, kv_heads,
             *_pages(page_table, pool, page_bytes, layer, index), kp, ks, vp, vs, code,
             _vec(status, _I32, "status", index))
    return k, v


def attention_prompt(q, seq_rows, seq_slot, seq_pos, kv_heads, page_table, pool, page_bytes, layer, scale=0.125,
                     window=0, out=None, status=None):
    """Whole-prompt causal attention over the pages (ndl_attention_prompt).

    q [rows, heads, 64] (float32, float16, bfloat16; rows possibly strided)
    packs the sequences: rows seq_rows[s] .. seq_rows[s+1] (int32
    [sequences + 1]) are queries at positions seq_pos[s], seq_pos[s] + 1, ...
    of slot seq_slot[s], whose pages hold the keys and values up to the last
    of them.  window > 0: the last `window` positions only.  Rows of no
    sequence are left as they are in `out`."""
    code, index = _start(q, "q")
    qp, qs = _heads(q, q.dtype, "q", index)
    out = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    op, os_ = _heads(out, q.dtype, "out", index, q.shape)
    rows, heads, _ = q.shape
    sequences = seq_slot.numel()
    _call_on(index, "ndl_attention_prompt", qp, qs, code, _vec(seq_rows, _I32, "seq_rows", index, sequences + 1),
             _vec(seq_slot, _I32, "seq_slot", index), _vec(seq_pos, _I32, "seq_pos", index, sequences), sequences,
             rows, heads, kv_heads, scale, window, *_pages(page_table, pool, page_bytes, layer, index), op, os_,
             _vec(status, _I32, "status", index))
    return out


def attention_split_workspace(rows, heads, kv_heads, max_pages):
    return lib().ndl_attention_split_workspace(rows, heads, kv_heads, max_pages)


def attention_split(q, row_slot, row_len, kv_heads, page_table, pool, page_bytes, layer, scale=0.125, window=0,
                    out=None, workspace=None, status=None):
    """Attention of single tokens, each split over its cache (ndl_attention_split).

    q [rows, heads, 64] (float32, float16, bfloat16; rows possibly strided);
    row r attends to the first row_len[r] positions (with window > 0 the last
    `window` of them) of slot row_slot[r]; length 0 gives zeros.  workspace
    uint8 [attention_split_workspace(...)]: allocated for the call if none is
    given; calls that overlap need one each."""
    code, index = _start(q, "q")
    qp, qs = _heads(q, q.dtype, "q", index)
    out = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    op, os_ = _heads(out, q.dtype, "out", index, q.shape)
    rows, heads, _ = q.shape
    pages = _pages(page_table, pool, page_bytes, layer, index)
    if workspace is None:
        workspace = pool.new_empty(lib().ndl_attention_split_workspace(rows, heads, kv_heads, pages[2]))
    _call_on(index, "ndl_attention_split", qp, qs, code, _vec(row_slot, _I32, "row_slot", index, rows),
             _vec(row_len, _I32, "row_len", index, rows), rows, heads, kv_heads, scale, window, *pages, op, os_,
             _vec(workspace, _U8, "workspace", index), workspace.numel(), _vec(status, _I32, "status", index))
    return out


def logits_process(logits, out=None, tokens=None, token_offsets=None, prompt_lens=None, repetition=None,
                   frequency=None, presence=None, bias_ids=None, bias_values=None, bias_offsets=None, mask=None,
                   mask_index=None, status=None):
    """Penalties, biases and masks on logits [rows, vocab] fp32 (ndl_logits_process).

    Row r's tokens are tokens[token_offsets[r]:token_offsets[r+1]] (int32), of
    which the first prompt_lens[r] are the prompt; repetition, frequency,
    presence fp32 [rows]; its biases bias_ids / bias_values
    [bias_offsets[r]:bias_offsets[r+1]]; mask int32 [mask rows, words] (bit
    set: allowed), row mask_index[r] of it (negative: none), without
    mask_index row r.  out may be `logits` itself."""
    _, index = _start(logits, "logits", {_F32: 0})
    out = torch.empty_like(logits, memory_format=torch.contiguous_format) if out is None else out
    if logits.dim() != 2:
        raise ValueError("logits must be [rows, vocab]")
    rows, vocab = logits.shape

    def matrix(t, name):
        if not isinstance(t, torch.Tensor) or t.dtype is not _F32 or t.get_device() != index:
            _wrong(t, _F32, name, index)
        if t.shape != logits.shape or (vocab > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be [{rows}, {vocab}] with contiguous rows")
        return t.data_ptr(), (t.stride(0) if rows > 1 else vocab)

    n_bias = 0 if bias_ids is None else bias_ids.numel()
    mask_rows, words = (0, 0) if mask is None else mask.shape
    _call_on(index, "ndl_logits_process", *matrix(logits, "logits"), *matrix(out, "out"), rows, vocab,
             _vec(tokens, _I32, "tokens", index), 0 if tokens is None else tokens.numel(),
             _vec(token_offsets, _I32, "token_offsets", index, rows + 1),
             _vec(prompt_lens, _I32, "prompt_lens", index, rows), _vec(repetition, _F32, "repetition", index, rows),
             _vec(frequency, _F32, "frequency", index, rows), _vec(presence, _F32, "presence", index, rows),
             _vec(bias_ids, _I32, "bias_ids", index), _vec(bias_values, _F32, "bias_values", index, n_bias), n_bias,
             _vec(bias_offsets, _I32, "bias_offsets", index, rows + 1), _vec(mask, _I32, "mask", index), mask_rows,
             words, _vec(mask_index, _I32, "mask_index", index, rows), _vec(status, _I32, "status", index))
    return out
