"""Device-tensor wrappers of the C ABI: torch CUDA tensors in and out, work
enqueued on torch's current stream.

Every function takes 2-D tensors whose last dimension is contiguous (row
stride = tensor.stride(0)), so column bands and column slices of wider
buffers are accepted as they are -- the banded outputs of src/rowops.py:80-88
and the per-head slices of a fused QKV buffer.
"""
import ctypes
import functools

import torch

from . import _lib as L


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _mat(t, name, dtypes):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dim() != 2 or t.stride(1) != 1:
        raise ValueError(f"{name} must be 2-D with a contiguous last dimension")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} dtype {t.dtype} not in {dtypes}")
    return t


def _vec(t, n, name):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32:
        raise ValueError(f"{name} must be a float32 CUDA tensor")
    t = t.contiguous()
    if t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
    return t


def gelu_poly4(x, out=None, rounding=L.WX_ROUND_RNE):
    """GELU-poly4 of a bf16 (g4 / g4r) or fp32 (g4f) matrix into bf16 `out`."""
    _mat(x, "x", (torch.bfloat16, torch.float32))
    rows, cols = x.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=torch.bfloat16, device=x.device)
    _mat(out, "out", (torch.bfloat16,))
    if tuple(out.shape) != (rows, cols):
        raise ValueError("out shape mismatch")
    dt = L.WX_DTYPE_F32 if x.dtype == torch.float32 else L.WX_DTYPE_BF16
    L.check(L.lib().wx_gelu_poly4(_ptr(x), dt, _ptr(out), rows, cols, x.stride(0),
                                  out.stride(0), rounding, _stream()))
    return out


def softmax_rows(x, out=None, valid=0, scale=1.0, variant=4, rounding=L.WX_ROUND_TRUNC):
    """Row softmax over the first `valid` columns (all if 0) of bf16 rows."""
    _mat(x, "x", (torch.bfloat16,))
    rows, cols = x.shape
    if out is None:
        out = torch.empty(rows, cols, dtype=torch.bfloat16, device=x.device)
    _mat(out, "out", (torch.bfloat16,))
    if out.shape[0] != rows or out.shape[1] < (valid if valid > 0 else cols):
        raise ValueError("out shape mismatch")
    L.check(L.lib().wx_softmax_rows(_ptr(x), _ptr(out), rows, cols, valid, x.stride(0),
                                    out.stride(0), float(scale), variant, rounding, _stream()))
    return out


def layer_norm_rows(x, gamma=None, beta=None, out=None, eps=1e-5, mode=L.WX_LN_AIE,
                    rounding=L.WX_ROUND_TRUNC, out_dtype=None):
    """LayerNorm of each row (mode WX_LN_AIE: the reference's device kernel,
    bf16; WX_LN_FP32: fp32 two-pass, bf16 or fp32 in and out)."""
    _mat(x, "x", (torch.bfloat16, torch.float32))
    rows, cols = x.shape
    if out is None:
        od = out_dtype or (torch.bfloat16 if mode == L.WX_LN_AIE else x.dtype)
        out = torch.empty(rows, cols, dtype=od, device=x.device)
    _mat(out, "out", (torch.bfloat16, torch.float32))
    g, b = _vec(gamma, cols, "gamma"), _vec(beta, cols, "beta")
    idt = L.WX_DTYPE_F32 if x.dtype == torch.float32 else L.WX_DTYPE_BF16
    odt = L.WX_DTYPE_F32 if out.dtype == torch.float32 else L.WX_DTYPE_BF16
    L.check(L.lib().wx_layernorm_rows(_ptr(x), idt, _ptr(g), _ptr(b), _ptr(out), odt, rows,
                                      cols, x.stride(0), out.stride(0), float(eps), mode,
                                      rounding, _stream()))
    return out


def gemm(A, W, bias=None, residual=None, out=None, epilogue=None):
    """epilogue(A @ W^T) on the tensor cores: A (M, K) bf16, W (N, K) bf16.

    Default epilogue: fp32 output (+ residual when given)."""
    _mat(A, "A", (torch.bfloat16,))
    _mat(W, "W", (torch.bfloat16,))
    M, K = A.shape
    N, K2 = W.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if epilogue is None:
        epilogue = L.WX_EPI_F32_RESID if residual is not None else L.WX_EPI_F32
    f32_out = epilogue in (L.WX_EPI_F32, L.WX_EPI_F32_RESID)
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32 if f32_out else torch.bfloat16,
                          device=A.device)
    _mat(out, "out", (torch.float32,) if f32_out else (torch.bfloat16,))
    b = _vec(bias, N, "bias")
    r = None
    if residual is not None:
        r = _mat(residual, "residual", (torch.float32,))
    L.check(L.lib().wx_gemm_bf16(_ptr(A), _ptr(W), _ptr(b), _ptr(r), _ptr(out), M, N, K,
                                 A.stride(0), W.stride(0), out.stride(0),
                                 r.stride(0) if r is not None else 0, epilogue, _stream()))
    return out


def gemm_f32(A, W, bias=None, out=None):
    """A @ W^T (+ bias) in fp32 on the FMA pipe: A (M, K), W (N, K) float32
    CUDA tensors with unit column stride; each output sums k in ascending order."""
    _mat(A, "A", (torch.float32,))
    _mat(W, "W", (torch.float32,))
    M, K = A.shape
    N, K2 = W.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32, device=A.device)
    _mat(out, "out", (torch.float32,))
    b = _vec(bias, N, "bias")
    L.check(L.lib().wx_gemm_f32(_ptr(A), _ptr(W), _ptr(b), _ptr(out), M, N, K, A.stride(0),
                                W.stride(0), out.stride(0), _stream()))
    return out


def _outvec(t, n, name):
    """A float32 CUDA vector written in place: must be contiguous already."""
    _vec(t, n, name)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _dtype_code(t, name):
    if t.dtype == torch.bfloat16:
        return L.WX_DTYPE_BF16
    if t.dtype == torch.float32:
        return L.WX_DTYPE_F32
    raise TypeError(f"{name}: bf16 or fp32 expected, got {t.dtype}")


def absmax_rows(x, out=None, per_row=True):
    """max |x| per row (per_row) or over the whole matrix, folded into `out`
    (fp32, zeroed when created here)."""
    _mat(x, "x", (torch.bfloat16, torch.float32))
    rows, cols = x.shape
    if out is None:
        out = torch.zeros(rows if per_row else 1, dtype=torch.float32, device=x.device)
    _outvec(out, rows if per_row else 1, "out")
    L.check(L.lib().wx_absmax_rows(_ptr(x), _dtype_code(x, "x"), rows, cols, x.stride(0),
                                   _ptr(out), 1 if per_row else 0, _stream()))
    return out


def quantize_rows(x, rowmax=None, q=None, scale=None):
    """Per-row int8 quantisation: scale = max|row| / 127 (1 for a zero row),
    q = rint(x / scale). rowmax: precomputed maxima, one per row or a single
    value for every row. Returns (q int8 (rows, cols), scale fp32 (rows,))."""
    _mat(x, "x", (torch.bfloat16, torch.float32))
    rows, cols = x.shape
    if q is None:
        q = torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :cols]
    _mat(q, "q", (torch.int8,))
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _outvec(scale, rows, "scale")
    stride = 0
    if rowmax is not None:
        if rowmax.numel() not in (1, rows):
            raise ValueError("rowmax: one value per row or one in all")
        stride = 1 if rowmax.numel() == rows and rows > 1 else 0
        rowmax = _vec(rowmax, rowmax.numel(), "rowmax")
    L.check(L.lib().wx_quantize_rows(_ptr(x), _dtype_code(x, "x"), rows, cols, x.stride(0),
                                     _ptr(rowmax), stride, _ptr(q), q.stride(0), _ptr(scale),
                                     _stream()))
    return q, scale


def layer_norm_quant_rows(x, gamma=None, beta=None, eps=1e-5, q=None, scale=None):
    """fp32 LayerNorm of each row of x quantised per row to int8, in one pass:
    the same (q, scale) as quantize_rows(layer_norm_rows(x, ..., fp32 out))."""
    _mat(x, "x", (torch.float32,))
    rows, cols = x.shape
    if q is None:
        q = torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :cols]
    _mat(q, "q", (torch.int8,))
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    _outvec(scale, rows, "scale")
    g = _vec(gamma, cols, "gamma")
    b = _vec(beta, cols, "beta")
    L.check(L.lib().wx_layernorm_quant_rows(_ptr(x), _ptr(g), _ptr(b), _ptr(q), _ptr(scale), rows,
                                            cols, x.stride(0), q.stride(0), eps, _stream()))
    return q, scale


def gemm_i8(Aq, Wq, sa, sw, bias=None, residual=None, out=None, epilogue=None, rowmax=None):
    """epilogue((float(Aq @ Wq^T) * sa[:, None]) * sw[None, :]) on the int8
    tensor cores: Aq (M, K) and Wq (N, K) int8 with rows 16-byte aligned, sa
    (M,) and sw (N,) fp32. rowmax (M,) fp32 collects max |out| per row for the
    bf16 epilogues."""
    _mat(Aq, "Aq", (torch.int8,))
    _mat(Wq, "Wq", (torch.int8,))
    M, K = Aq.shape
    N, K2 = Wq.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    if epilogue is None:
        epilogue = L.WX_EPI_F32_RESID if residual is not None else L.WX_EPI_F32
    f32_out = epilogue in (L.WX_EPI_F32, L.WX_EPI_F32_RESID)
    if out is None:
        out = torch.empty(M, N, dtype=torch.float32 if f32_out else torch.bfloat16,
                          device=Aq.device)
    _mat(out, "out", (torch.float32,) if f32_out else (torch.bfloat16,))
    sa = _vec(sa, M, "sa")
    sw = _vec(sw, N, "sw")
    b = _vec(bias, N, "bias")
    if rowmax is not None:
        _outvec(rowmax, M, "rowmax")
    r = None
    if residual is not None:
        r = _mat(residual, "residual", (torch.float32,))
    L.check(L.lib().wx_gemm_i8(_ptr(Aq), _ptr(Wq), _ptr(sa), _ptr(sw), _ptr(b), _ptr(r),
                               _ptr(out), M, N, K, Aq.stride(0), Wq.stride(0), out.stride(0),
                               r.stride(0) if r is not None else 0, epilogue, _ptr(rowmax),
                               _stream()))
    return out


def attention(q, k, v, n_batch, n_head, scale, out=None):
    """softmax(scale * q k^T) v per (batch, head); q, k, v: (n_batch*T, n_head*64)
    bf16 (column slices of one QKV buffer are fine)."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _mat(t, n, (torch.bfloat16,))
    rows, width = q.shape
    if rows % n_batch:
        raise ValueError("rows not divisible by n_batch")
    T = rows // n_batch
    hd = width // n_head
    if out is None:
        out = torch.empty(rows, width, dtype=torch.bfloat16, device=q.device)
    _mat(out, "out", (torch.bfloat16,))
    L.check(L.lib().wx_attention(_ptr(q), _ptr(k), _ptr(v), _ptr(out), n_batch, n_head, T, hd,
                                 q.stride(0), k.stride(0), v.stride(0), out.stride(0),
                                 float(scale), _stream()))
    return out


def log_mel(audio, n_mels=80, out=None):
    """whisper's log-mel features of 16 kHz audio on the GPU: audio a CUDA
    float32 tensor (batch, n_samples) or (n_samples,), each clip zero-padded or
    trimmed to 30 s -> (batch, n_mels, 3000) float32 (or (n_mels, 3000))."""
    squeeze = audio.dim() == 1
    a = audio.unsqueeze(0) if squeeze else audio
    if not a.is_cuda or a.dtype != torch.float32 or a.dim() != 2 or a.stride(1) != 1:
        raise ValueError("audio must be a CUDA float32 tensor with contiguous rows")
    B, n = a.shape
    if out is None:
        out = torch.empty(B, n_mels, 3000, dtype=torch.float32, device=a.device)
    if out.shape != (B, n_mels, 3000) or not out.is_contiguous() or out.dtype != torch.float32:
        raise ValueError("out must be a contiguous float32 (batch, n_mels, 3000) tensor")
    L.check(L.lib().wx_log_mel(_ptr(a), B, n, a.stride(0) if B > 1 else n, int(n_mels),
                               _ptr(out), _stream()))
    return out[0] if squeeze else out


# ---------------------------------------------------------------- decoder operators
# Paged key-value cache: pools of shape (pages, page, heads, head_dim) for a
# layer, (layers, pages, page, heads, head_dim) for a whole cache, any strides
# with head_dim contiguous (a head-major pool is passed transposed). The page
# table is (n_seqs, width) int32, -1 past a sequence's last page.

_KV_DTYPES = {torch.bfloat16: L.WX_DTYPE_BF16, torch.float32: L.WX_DTYPE_F32}

# a decoder step calls these operators for every layer, so their checks are kept
# to a few microseconds
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on(dev, name, t, dtype, shape):
    """The address of t: on device `dev`, of dtype, contiguous, of the shape given."""
    if (isinstance(t, torch.Tensor) and t.get_device() == dev and t.dtype is dtype
            and t.shape == shape and t.is_contiguous()):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or t.get_device() != dev:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the others")
    raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got "
                     f"{t.dtype}, {tuple(t.shape)}, strides {t.stride()}")


def _pools(k_cache, v_cache, dim):
    """Checks a cache's two pools; returns (device, dtype code, shape, strides)."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor")
    dtype, shape, strides = k_cache.dtype, k_cache.shape, k_cache.stride()
    if len(shape) != dim:
        raise ValueError(f"the cache must have {dim} dimensions, got {len(shape)}")
    if v_cache.dtype is not dtype or v_cache.shape != shape or v_cache.stride() != strides:
        raise ValueError("k_cache and v_cache must have the same dtype, shape and strides")
    code = _KV_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"cache dtype {dtype} not in {list(_KV_DTYPES)}")
    if strides[-1] != 1:
        raise ValueError("the cache's head_dim must be contiguous")
    dev = k_cache.get_device()
    if v_cache.get_device() != dev or dev != torch.cuda.current_device():
        raise ValueError("the cache must be on the current CUDA device")
    return dev, code, shape, strides


def _rows(dev, table):
    """(sequences, width, address) of a page table."""
    shape = table.shape if isinstance(table, torch.Tensor) else ()
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError("table must be a (n_seqs, width) tensor")
    return shape[0], shape[1], _on(dev, "table", table, torch.int32, shape)


@functools.lru_cache(maxsize=1024)
def _attend_space(n_seqs, n_heads, group, head_dim, max_len, dtype):
    n = L.lib().wx_paged_attention_workspace(n_seqs, n_heads, group, head_dim, max_len, dtype)
    if n < 0:
        L.check(n)
    return n


def paged_attention(q, k_cache, v_cache, table, lens, scale=None, starts=None, max_len=None,
                    out=None, return_lse=False):
    """Attention of one new token a sequence over a paged cache: query row g of
    cache head h of sequence i attends to the keys starts[i] <= j < lens[i].

    q: (n_seqs, heads, head_dim), its heads in groups that share a cache head, or
    (n_seqs, cache heads, group, head_dim) with any strides -- for beams over one
    clip's keys, x.view(clips, beams, heads, hd).transpose(1, 2). scale: default
    head_dim ** -0.5. max_len: an upper bound of lens, by default what the table
    holds; a close one makes a better split. Returns out (q's shape and strides,
    q's dtype), with return_lse also log sum_j e^(scale q.k_j), fp32, q's shape
    without head_dim. A row without keys gives 0 and -inf."""
    dev, dt, shape, st = _pools(k_cache, v_cache, 4)
    n_pages, page, n_heads, hd = shape
    n, width, table_p = _rows(dev, table)
    lens_p = _on(dev, "lens", lens, torch.int32, (n,))
    if not isinstance(q, torch.Tensor) or q.get_device() != dev or q.dtype is not k_cache.dtype:
        raise ValueError("q must be a CUDA tensor on the cache's device, of its dtype")
    qs, qt = q.shape, q.stride()
    if len(qs) == 3:
        group, rest = divmod(qs[1], n_heads)
        if rest:
            raise ValueError(f"{qs[1]} query heads are no multiple of {n_heads} cache heads")
    elif len(qs) == 4:
        group = qs[2]
        if qs[1] != n_heads:
            raise ValueError(f"q has {qs[1]} cache heads, the cache {n_heads}")
    else:
        raise ValueError("q must have 3 or 4 dimensions")
    if qs[0] != n or qs[-1] != hd or qt[-1] != 1:
        raise ValueError(f"q of shape {tuple(qs)} does not fit {n} sequences of head_dim {hd} "
                         "(contiguous)")
    if out is None:
        out = torch.empty_like(q)
    elif (out.shape != qs or out.dtype is not q.dtype or out.get_device() != dev
          or out.stride(-1) != 1):
        raise ValueError("out must be like q, with a contiguous head_dim")
    ot = out.stride()
    if len(qs) == 3:
        qt, ot = (qt[0], qt[1] * group, qt[1]), (ot[0], ot[1] * group, ot[1])
    if max_len is None:
        max_len = width * page
    starts_p = None if starts is None else _on(dev, "starts", starts, torch.int32, (n,))
    lse = torch.empty(qs[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    space = _attend_space(n, n_heads, group, hd, max_len, dt)
    ws = torch.empty(space, dtype=torch.uint8, device=q.device) if space else None
    status = L.lib().wx_paged_attention(
        q.data_ptr(), qt[0], qt[1], qt[2], k_cache.data_ptr(), v_cache.data_ptr(), st[0], st[1],
        st[2], table_p, width, lens_p, starts_p, out.data_ptr(), ot[0], ot[1], ot[2],
        lse.data_ptr() if return_lse else None, n, n_heads, group, hd, n_pages, page, max_len,
        hd ** -0.5 if scale is None else float(scale), dt, ws.data_ptr() if space else None,
        space, _raw_stream(dev))
    if status:
        L.check(status)
    return (out, lse) if return_lse else out


def kv_append(k, v, k_cache, v_cache, table, lens, counts=None):
    """Writes new tokens into a layer's cache, in place: k, v (n_seqs, tokens,
    heads, head_dim) or, for one token each, (n_seqs, heads, head_dim), of the
    cache's dtype; row t < counts[i] (all if None) of sequence i goes to position
    lens[i] - counts[i] + t."""
    dev, dt, shape, st = _pools(k_cache, v_cache, 4)
    n_pages, page, n_heads, hd = shape
    n, width, table_p = _rows(dev, table)
    lens_p = _on(dev, "lens", lens, torch.int32, (n,))
    for t, name in ((k, "k"), (v, "v")):
        if (not isinstance(t, torch.Tensor) or t.get_device() != dev
                or t.dtype is not k_cache.dtype):
            raise ValueError(f"{name} must be a CUDA tensor on the cache's device, of its dtype")
    ks, kt = k.shape, k.stride()
    if v.shape != ks or v.stride() != kt:
        raise ValueError("k and v must have the same shape and strides")
    if len(ks) == 3:
        ks, kt = (ks[0], 1, ks[1], ks[2]), (kt[0], 0, kt[1], kt[2])
    if len(ks) != 4 or ks[0] != n or ks[2] != n_heads or ks[3] != hd or kt[3] != 1:
        raise ValueError(f"k of shape {tuple(k.shape)} does not fit {n} sequences of {n_heads} "
                         f"heads of {hd} (contiguous)")
    counts_p = _on(dev, "counts", counts, torch.int32, (n,)) if counts is not None else None
    L.check(L.lib().wx_kv_append(
        k.data_ptr(), v.data_ptr(), kt[0], kt[1], kt[2], k_cache.data_ptr(), v_cache.data_ptr(),
        st[0], st[1], st[2], table_p, width, lens_p, counts_p, n, ks[1], n_heads, hd, n_pages,
        page, dt, _raw_stream(dev)))


@functools.lru_cache(maxsize=1024)
def _plan_space(n_seqs, n_pages):
    return L.lib().wx_kv_workspace(n_seqs, n_pages)


def kv_fork(k_cache, v_cache, table, lens, refs, parents=None, grow=None):
    """One step of every sequence's pages in all layers of a cache: sequence i
    goes on as parents[i] was (-1: it starts empty; None: as itself), with room
    for grow[i] more tokens (None: no tokens). Shared pages about to be written
    are copied, pages nobody names are freed, new ones are the lowest free ones.
    Nothing waits for the GPU.

    Returns new int32 tensors (table, lens, refs, grown, status): lens counts the
    tokens granted (grown), status is (pages left free, pages short). A sequence
    whose pages the pool does not hold is not grown."""
    dev, dt, shape, st = _pools(k_cache, v_cache, 5)
    n_layers, n_pages, page, n_heads, hd = shape
    n, width, table_p = _rows(dev, table)
    lens_p = _on(dev, "lens", lens, torch.int32, (n,))
    refs_p = _on(dev, "refs", refs, torch.int32, (n_pages,))
    parents_p = _on(dev, "parents", parents, torch.int32, (n,)) if parents is not None else None
    grow_p = _on(dev, "grow", grow, torch.int32, (n,)) if grow is not None else None
    space = _plan_space(n, n_pages)
    on = table.device
    new = (torch.empty_like(table), torch.empty_like(lens), torch.empty_like(refs),
           torch.empty_like(lens), torch.empty(2, dtype=torch.int32, device=on))
    ws = torch.empty(space, dtype=torch.uint8, device=on)
    L.check(L.lib().wx_kv_fork(
        k_cache.data_ptr(), v_cache.data_ptr(), n_layers, st[0], st[1], st[2], st[3], n_heads, hd,
        n_pages, page, dt, table_p, lens_p, refs_p, parents_p, grow_p, n, width,
        *(t.data_ptr() for t in new), ws.data_ptr(), space, _raw_stream(dev)))
    return new


def kv_compact(k_cache, v_cache, table, refs):
    """Moves the pages in use to the front of the pool in all layers of a cache,
    with the fewest moves. Returns new int32 tensors (table, refs, status), status
    being (pages in use, pages moved)."""
    dev, dt, shape, st = _pools(k_cache, v_cache, 5)
    n_layers, n_pages, page, n_heads, hd = shape
    n, width, table_p = _rows(dev, table)
    refs_p = _on(dev, "refs", refs, torch.int32, (n_pages,))
    space = _plan_space(n, n_pages)
    on = table.device
    new = (torch.empty_like(table), torch.empty_like(refs),
           torch.empty(2, dtype=torch.int32, device=on))
    ws = torch.empty(space, dtype=torch.uint8, device=on)
    L.check(L.lib().wx_kv_compact(
        k_cache.data_ptr(), v_cache.data_ptr(), n_layers, st[0], st[1], st[2], st[3], n_heads, hd,
        n_pages, page, dt, table_p, refs_p, n, width, *(t.data_ptr() for t in new),
        ws.data_ptr(), space, _raw_stream(dev)))
    return new


def token_logprobs(logits, tokens, top_k=0, temperature=1.0):
    """Scores under rows of logits ((rows, vocab), bf16 or fp32, masked tokens
    -inf), with z = logits / temperature: returns (logprob, entropy, top_logprob,
    top_index) -- log softmax(z)[tokens] (tokens (rows,) int64; a token below 0 is
    none and scores 0) and the entropy in nats, fp32 (rows,), and the top_k (<= 32)
    likeliest tokens with their log probabilities, (rows, top_k) fp32 and int32,
    equal logits by the lowest token. A row that is all -inf scores -inf, with
    entropy 0."""
    _mat(logits, "logits", (torch.bfloat16, torch.float32))
    rows, vocab = logits.shape
    dev = logits.get_device()
    if dev != torch.cuda.current_device():
        raise ValueError("logits must be on the current CUDA device")
    tokens_p = _on(dev, "tokens", tokens, torch.int64, (rows,))
    if not 0 <= top_k <= min(32, vocab):
        raise ValueError(f"top_k {top_k} not in [0, min(32, vocabulary {vocab})]")
    on = logits.device
    logprob = torch.empty(rows, dtype=torch.float32, device=on)
    entropy = torch.empty_like(logprob)
    top = torch.empty((rows, top_k), dtype=torch.float32, device=on)
    index = torch.empty_like(top, dtype=torch.int32)
    status = L.lib().wx_token_logprobs(
        logits.data_ptr(), _KV_DTYPES[logits.dtype], rows, vocab, logits.stride(0), tokens_p,
        top_k, float(temperature), logprob.data_ptr(), entropy.data_ptr(),
        top.data_ptr() if top_k else None, index.data_ptr() if top_k else None,
        _raw_stream(dev))
    if status:
        L.check(status)
    return logprob, entropy, top, index
