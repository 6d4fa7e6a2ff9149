"""fp8 codes with a scale per 128 values, and what makes and reads them: the
quantizer, the products of a Linear, the root-mean-square norm in front of it.

Codes are float8_e4m3fn or float8_e5m2 tensors whose rows start at multiples of
16 bytes.  Scales are [blocks, rows]: scales[b, r] belongs to columns 128 b to
128 b + 127 of row r, as float8_e8m0fnu (powers of two, which the matrix
instructions apply by themselves) or fp32 numbers, each block's starting at a
multiple of 16 bytes.  The calls here lay both out so; :func:`block_scales`
brings scales from elsewhere into that form.
"""
from __future__ import annotations

import ctypes
import enum
import functools

from . import (Fmt, _check_gpu, _check_like, _fits, _in_dtype, _INT_MAX, _on, _plain, _ptr, _row_vector, _rows,
               _stream, _torch, call, lib, round16)

BLOCK = 128  # values that share a scale


@functools.lru_cache(1024)
def _workspace_bytes(fn: str, *sizes) -> int:
    """(0.2 us of a call where asking the library takes 1 to 2)"""
    return getattr(lib(), fn + "_workspace_bytes")(*sizes)


def _kind(fn: str, dtype) -> int:
    torch = _torch()
    if dtype is torch.float8_e8m0fnu:
        return 1  # DF_SCALE_E8M0
    if dtype is torch.float32:
        return 0
    raise TypeError(f"{fn}: scales are float8_e8m0fnu or float32, not {dtype}")


def _code_dtype(fmt):
    torch = _torch()
    return torch.float8_e4m3fn if Fmt(fmt) == Fmt.E4M3 else torch.float8_e5m2


def _new_scales(like, blocks: int, rows: int, dtype):
    """[blocks, rows], each block's at a multiple of 16 bytes, and the leading
    dimension."""
    step = 15 if dtype.itemsize == 1 else 3
    ld = (rows + step) & ~step
    s = like.new_empty((blocks, ld), dtype=dtype)
    return (s if ld == rows else s.as_strided((blocks, rows), (ld, 1))), ld


def _scales_ld(fn: str, name: str, s, blocks: int, rows: int, dtype) -> int:
    """The leading dimension of scales, checked to lie as the library reads
    them: 16 bytes at a time, the last ones of a block too."""
    if s.shape != (blocks, rows) or s.dtype is not dtype:
        raise ValueError(f"{fn}: {name} is {tuple(s.shape)} {s.dtype}, not {(blocks, rows)} {dtype}")
    step, size = (15, 1) if dtype.itemsize == 1 else (3, 4)
    need = (rows + step) & ~step  # of one block
    ld, one = s.stride()
    if blocks <= 1 or rows == 0:
        ld = need
    if (one != 1 and rows > 1 or ld < rows or ld & step or s.data_ptr() & 15
            or need != rows and (s.storage_offset() + (blocks - 1) * ld + need) * size > s.untyped_storage().nbytes()):
        raise ValueError(f"{fn}: {name} with strides {s.stride()} does not lie as block_scales() leaves it")
    return ld


def block_scales(scales, rows: int | None = None):
    """Scales as others keep them, [rows, blocks], or for codes of ``rows``
    rows [ceil(rows / 128), blocks] (one per 128 x 128 square), as the products
    read them: [blocks, rows].  A copy, made once when weights are loaded."""
    fn, torch = "block_scales", _torch()
    _kind(fn, scales.dtype)
    if scales.dim() != 2:
        raise ValueError(f"{fn}: scales of {scales.dim()} dimensions, not 2")
    raw = scales.view(torch.uint8) if scales.dtype.itemsize == 1 else scales
    if rows is not None:
        if raw.shape[0] != -(-rows // BLOCK):
            raise ValueError(f"{fn}: {raw.shape[0]} rows of scales for {rows} rows of codes, 128 to a scale")
        raw = raw.repeat_interleave(BLOCK, 0)[:rows]
    out, _ = _new_scales(scales, raw.shape[1], raw.shape[0], scales.dtype)
    out.view(raw.dtype).copy_(raw.t())
    return out


def quantize_blocks(x, fmt: Fmt = Fmt.E4M3, want_q=True, want_qt=False, square=False, scale_dtype=None):
    """A 2-D fp32/bf16/f16 tensor [R, C] to fp8 codes with a scale per 128 values
    (df_quantize_blocks): returns (q [R, ceil16(C)], s [ceil(C/128), R], qt [C,
    ceil16(R)], st [ceil(R/128), C]), None where not wanted.  q shares a scale
    among 128 columns of a row, qt among 128 rows of a column; with ``square``
    (weights) both have one scale per 128 x 128.  Scales are powers of two
    (float8_e8m0fnu) unless ``scale_dtype`` is float32."""
    fn, torch = "quantize_blocks", _torch()
    if x.dim() != 2:
        raise ValueError(f"{fn}: x has {x.dim()} dimensions, not 2")
    if not (want_q or want_qt):
        raise ValueError(f"{fn}: no codes wanted")
    scale_dtype = scale_dtype or torch.float8_e8m0fnu
    kind, codes = _kind(fn, scale_dtype), _code_dtype(fmt)
    rows, cols = x.shape
    if (rows | cols) > _INT_MAX:
        _fits(fn, rows, cols)
    if not x.is_cuda:
        raise ValueError(f"{fn}: x is on {x.device}, not on a GPU")
    ldx = cols if x.is_contiguous() else _rows(fn, "x", x, x.shape, x.dtype)
    dt = _in_dtype(x)
    with _on(x):
        q = s = qt = st = None
        ldq = lds = ldqt = ldst = 0
        step, nb, nbt = (15 if kind else 3), -(-cols // BLOCK), -(-rows // BLOCK)
        if want_q:
            ldq, lds = (cols + 15) & ~15, (rows + step) & ~step
            q = x.new_empty((rows, ldq), dtype=codes)
        if want_qt:
            ldqt, ldst = (rows + 15) & ~15, (cols + step) & ~step
            qt = x.new_empty((cols, ldqt), dtype=codes)
        # both kinds of scales in one allocation: an allocation is 1.4 us of a call, a view 0.7
        scales = x.new_empty(nb * lds + nbt * ldst, dtype=scale_dtype)
        if want_q:
            s = scales.as_strided((nb, rows), (lds, 1))
        if want_qt:
            st = scales.as_strided((nbt, cols), (ldst, 1), nb * lds)
        if rows and cols:
            call("df_quantize_blocks", dt, x.data_ptr(), rows, cols, ldx, int(fmt), kind, int(bool(square)), _ptr(q), ldq,
                 _ptr(s), lds, _ptr(qt), ldqt, _ptr(st), ldst, _stream())
    return q, s, qt, st


def _rows_ld(t, rows: int, ld: int, red: int) -> int:
    """The leading dimension of ``rows`` rows of codes ``ld`` apart, which are read up to
    the next multiple of 16 behind ``red``; -1 where the last one's do not lie in the
    tensor's memory."""
    width, need = t.shape[-1], (red + 15) & ~15
    if width < need and rows:  # (the rows' own width holds them else)
        return -1 if t.storage_offset() + (rows - 1) * ld + need > t.untyped_storage().nbytes() else ld
    # the stride of one row, or of rows without codes, is arbitrary and says nothing
    return (width + 15) & ~15 if rows <= 1 or width == 0 else ld


def _codes(fn: str, name: str, t, red: int, ok: bool):
    """The leading dimension of an operand's codes (``ok``: their type is right)."""
    if not ok or t.dim() != 2:
        raise ValueError(f"{fn}: {name} {tuple(t.shape)} {t.dtype} is not a matrix of codes in its format")
    rows, width = t.shape
    ld, one = t.stride()
    if rows <= 1 or not width or width < (red + 15) & ~15:  # (the usual codes are asked no more)
        ld = _rows_ld(t, rows, ld, red)
    if width < red or one != 1 and width > 1 or ld < width or ld & 15 or t.data_ptr() & 15:
        raise ValueError(f"{fn}: {name} {tuple(t.shape)} with strides {t.stride()} has no rows of {red} codes at "
                         "multiples of 16 bytes, readable up to the next")
    return ld


def gemm_blocks(a_q, sa, b_q, sb, K: int, bias=None, out_dtype=None, out=None):
    """C [M, N] = A . B^T with a scale per 128 of K (df_fp8_gemm_blocks): a_q [M,
    >=K] e4m3 or e5m2 codes with scales sa [ceil(K/128), M], b_q [N, >=K] e4m3
    codes with scales sb [ceil(K/128), N], both zero from K to the next multiple
    of 16; plus bias [N] (fp32, bf16 or f16).  A new C is bf16 unless ``out_dtype``
    says otherwise; ``out`` is a C to write.  With :func:`quantize_blocks`' results
    of x [M, K], w [N, K] (square) and dy [M, N]:
    y = gemm_blocks(xq, sx, wq, sw, K), dx = gemm_blocks(dyq, sdy, wqt, swt, N),
    dw = gemm_blocks(dyqt, sdyt, xqt, sxt, M)."""
    fn, torch = "gemm_blocks", _torch()
    if K < 0:
        raise ValueError(f"{fn}: K = {K}")
    ta, kinds = a_q.dtype, sa.dtype
    e4 = ta is torch.float8_e4m3fn
    lda = _codes(fn, "a_q", a_q, K, e4 or ta is torch.float8_e5m2)
    ldb = _codes(fn, "b_q", b_q, K, b_q.dtype is torch.float8_e4m3fn)
    M, N, blocks = a_q.shape[0], b_q.shape[0], -(-K // BLOCK)
    kind = _kind(fn, kinds)
    ldsa, ldsb = _scales_ld(fn, "sa", sa, blocks, M, kinds), _scales_ld(fn, "sb", sb, blocks, N, kinds)
    at = a_q.get_device()
    if at < 0 or not (sa.get_device() == b_q.get_device() == sb.get_device() == at):
        _check_gpu(fn, a_q=a_q, sa=sa, b_q=b_q, sb=sb)
    if (M | N | K | lda | ldb | ldsa | ldsb) > _INT_MAX:
        _fits(fn, M, N, K, lda, ldb, ldsa, ldsb)
    bias_dt = 0
    if bias is not None:
        bias_dt = _in_dtype(bias)
        if not _plain(bias, (N,), bias.dtype, at):
            _check_gpu(fn, a_q=a_q, bias=bias)
            _row_vector(fn, "bias", bias, N, bias.dtype)
    with _on(a_q):
        if out is None:
            out, ldc = a_q.new_empty((M, N), dtype=out_dtype or torch.bfloat16), N
        else:
            _check_gpu(fn, a_q=a_q, out=out)
            ldc = _rows(fn, "out", out, (M, N), out_dtype or out.dtype)
        call("df_fp8_gemm_blocks", 0 if e4 else 1, a_q.data_ptr(), lda, b_q.data_ptr(), ldb, M, N, K, kind, sa.data_ptr(),
             ldsa, sb.data_ptr(), ldsb, bias_dt, None if bias is None else bias.data_ptr(), _in_dtype(out), out.data_ptr(),
             ldc, _stream())
    return out


class BlocksKernel(enum.IntEnum):
    """DF_BLOCKS_KERNEL_* of include/df_capi.h: by tiles."""
    T16 = 0
    T16X32 = 1
    T32 = 2
    T32_LONG = 3
    T64 = 4
    T128 = 5
    T256X128 = 6
    T256 = 7


def gemm_blocks_plan(M: int, N: int, K: int, scale_dtype=None, out_dtype=None) -> BlocksKernel:
    """The kernel that :func:`gemm_blocks` takes for these sizes on the current GPU
    (df_fp8_gemm_blocks_plan)."""
    fn, torch = "gemm_blocks_plan", _torch()
    kind = _kind(fn, scale_dtype or torch.float8_e8m0fnu)
    out = ctypes.c_int()
    call("df_fp8_gemm_blocks_plan", M, N, K, kind, _in_dtype(torch.empty(0, dtype=out_dtype or torch.bfloat16)),
         ctypes.byref(out))
    return BlocksKernel(out.value)


# ----------------------------------------------------------------------------
# a mixture-of-experts layer for a few tokens
# ----------------------------------------------------------------------------
ACTIVATIONS = {"swiglu": 0, "geglu": 1, "gelu": 2}  # df_activation


def quantize_experts_blocks(w, scale_dtype=None):
    """Experts' weights w [experts, R, C] (fp32, bf16 or float16) to e4m3 codes with a
    scale per 128 x 128: returns (q [experts, R, ceil16(C)], s [experts, ceil(C/128),
    R]), as :func:`moe_layer` takes them."""
    fn, torch = "quantize_experts_blocks", _torch()
    if w.dim() != 3 or not w.is_contiguous():
        raise ValueError(f"{fn}: w {tuple(w.shape)} is not [experts, R, C] and contiguous")
    scale_dtype = scale_dtype or torch.float8_e8m0fnu
    kind = _kind(fn, scale_dtype)
    _check_gpu(fn, w=w)
    E, R, C = w.shape
    _fits(fn, E, R, C)
    dt = _in_dtype(w)
    with _on(w):
        q = w.new_empty((E, R, round16(C)), dtype=torch.float8_e4m3fn)
        step = 16 // scale_dtype.itemsize
        ld = -(-R // step) * step
        s = w.new_empty((E, -(-C // BLOCK), ld), dtype=scale_dtype)
        for e in range(E if R and C else 0):
            call("df_quantize_blocks", dt, w[e].data_ptr(), R, C, C, int(Fmt.E4M3), kind, 1, q[e].data_ptr(), q.shape[2],
                 s[e].data_ptr(), ld, None, 0, None, 0, _stream())
    return q, s[:, :, :R]


def _expert_weights(fn: str, n: int, w, s, rows: int, cols: int, experts: int):
    """Leading dimensions of experts' codes and scales, checked."""
    blocks, shape = -(-cols // BLOCK), tuple(w.shape)
    if len(shape) != 3 or w.dtype is not _torch().float8_e4m3fn or shape[:2] != (experts, rows) or shape[2] < cols:
        raise ValueError(f"{fn}: w{n} is {shape} {w.dtype}, not e4m3 codes of {(experts, rows, cols)}")
    width, (each, ldw, one) = shape[2], w.stride()
    if rows <= 1 and experts > 1:
        ldw = each
    ldw = _rows_ld(w, experts * rows, ldw, cols)
    if one != 1 and width > 1 or ldw < width or ldw & 15 or w.data_ptr() & 15 or experts > 1 and each != rows * ldw:
        raise ValueError(f"{fn}: w{n} with strides {w.stride()} has no rows at multiples of 16 bytes, readable up to "
                         "the next, expert behind expert")
    if s.shape != (experts, blocks, rows):
        raise ValueError(f"{fn}: s{n} is {tuple(s.shape)}, not {(experts, blocks, rows)}")
    step, size = (3, 4) if s.dtype is _torch().float32 else (15, 1)
    need = (rows + step) & ~step
    each, lds, one = s.stride()
    if blocks <= 1:
        lds = each if experts > 1 else need
    if (one != 1 and rows > 1 or lds < rows or lds & step or s.data_ptr() & 15 or experts > 1 and each != blocks * lds
            or need != rows
            and (s.storage_offset() + (experts * blocks - 1) * lds + need) * size > s.untyped_storage().nbytes()):
        raise ValueError(f"{fn}: s{n} with strides {s.stride()} does not lie as quantize_experts_blocks() leaves it")
    return ldw, lds


def moe_layer(x, logits, w1, s1, w2, s2, top_k: int, activation: str = "swiglu", renormalize: bool = True):
    """A whole mixture-of-experts layer for a few tokens (df_moe_layer): x [T, H] bf16
    or float16, T <= 64, logits [T, experts] of the router (fp32, bf16 or float16), w1
    [experts, 2 N, >=H] (gate's rows, then up's; [experts, N, >=H] for "gelu") and w2
    [experts, H, >=N] e4m3 codes with scales s1, s2 (:func:`quantize_experts_blocks`).
    Each token goes to the ``top_k`` experts of its largest logits, weighted by the
    softmax over them (over all experts without ``renormalize``); a logit of -inf or NaN
    is never chosen.  Returns (y [T, H], ids int32 [T, top_k], weights fp32 [T, top_k]);
    an id is -1 where no expert was left."""
    fn, torch = "moe_layer", _torch()
    if x.dim() != 2 or logits.dim() != 2 or logits.shape[0] != x.shape[0]:
        raise ValueError(f"{fn}: x {tuple(x.shape)} and logits {tuple(logits.shape)} are not [tokens, H] and [tokens, experts]")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{fn}: x is {x.dtype}, not bfloat16 or float16")
    if activation not in ACTIVATIONS:
        raise ValueError(f"{fn}: activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    (tokens, H), experts = x.shape, logits.shape[1]
    if not 1 <= top_k <= experts:
        raise ValueError(f"{fn}: top_k = {top_k} of {experts} experts")
    if H == 0 and tokens:
        raise ValueError(f"{fn}: x has no columns")
    N = w2.shape[-1] if w2.dim() == 3 else 0
    if w1.dim() == 3:  # w2's rows may be padded, w1's are not
        N = w1.shape[1] if activation == "gelu" else w1.shape[1] // 2
    at = x.get_device()
    if at < 0 or not (logits.get_device() == w1.get_device() == s1.get_device() == w2.get_device() == s2.get_device() == at):
        _check_gpu(fn, x=x, logits=logits, w1=w1, s1=s1, w2=w2, s2=s2)
    kind = _kind(fn, s1.dtype)
    if s2.dtype is not s1.dtype:
        raise ValueError(f"{fn}: s1 is {s1.dtype} and s2 {s2.dtype}")
    ldw1, lds1 = _expert_weights(fn, 1, w1, s1, N if activation == "gelu" else 2 * N, H, experts)
    ldw2, lds2 = _expert_weights(fn, 2, w2, s2, H, N, experts)
    ldx = H if x.is_contiguous() else _rows(fn, "x", x, x.shape, x.dtype)
    ldl = experts if logits.is_contiguous() else _rows(fn, "logits", logits, logits.shape, logits.dtype)
    dt, lt = _in_dtype(x), _in_dtype(logits)
    if max(H, 2 * N, ldw1, ldw2, lds1, lds2) > _INT_MAX:
        _fits(fn, H, 2 * N, ldw1, ldw2, lds1, lds2)
    with _on(x):
        y = x.new_empty((tokens, H))
        ids = x.new_empty((tokens, top_k), dtype=torch.int32)
        weights = x.new_empty((tokens, top_k), dtype=torch.float32)
        # not a cached one: a captured graph keeps the workspace it was given
        nws = _workspace_bytes("df_moe_layer", tokens, H, N, experts, top_k)
        ws = x.new_empty(nws, dtype=torch.uint8)
        call("df_moe_layer", dt, x.data_ptr(), ldx, tokens, H, N, experts, top_k, lt, logits.data_ptr(), ldl,
             int(bool(renormalize)), ACTIVATIONS[activation], w1.data_ptr(), ldw1, w2.data_ptr(), ldw2, kind, s1.data_ptr(),
             lds1, s2.data_ptr(), lds2, y.data_ptr(), H, ids.data_ptr(), weights.data_ptr(), ws.data_ptr(), nws, _stream())
    return y, ids, weights


# ----------------------------------------------------------------------------
# root-mean-square norm
# ----------------------------------------------------------------------------
def _norm_args(fn: str, x, gamma, residual):
    if x.dim() != 2:
        raise ValueError(f"{fn}: x has {x.dim()} dimensions, not 2")
    shape, dtype, at = x.shape, x.dtype, x.get_device()
    rows, cols = shape
    if (rows | cols) > _INT_MAX:
        _fits(fn, rows, cols)
    ldx = ldr = cols
    if not (at >= 0 and x.is_contiguous() and _plain(residual, shape, dtype, at) and _plain(gamma, (cols,), dtype, at)):
        _check_gpu(fn, x=x, gamma=gamma, residual=residual)
        ldx = _rows(fn, "x", x, shape, dtype)
        ldr = cols if residual is None else _rows(fn, "residual", residual, shape, dtype)
        _row_vector(fn, "gamma", gamma, cols, dtype)
    return rows, cols, ldx, ldr


def rmsnorm_forward(x, gamma=None, eps=1e-5, residual=None):
    """Root-mean-square norm over the last dim of a 2-D fp32/bf16/f16 tensor
    (df_rmsnorm_forward): returns (y, s, rstd), where s = x + residual is what the
    norm saw (x itself without a residual) and rstd its rows' fp32 statistic: what
    :func:`rmsnorm_backward` takes."""
    fn, torch = "rmsnorm_forward", _torch()
    rows, cols, ldx, ldr = _norm_args(fn, x, gamma, residual)
    dt = _in_dtype(x)
    with _on(x):
        y = x.new_empty((rows, cols))
        s = x if residual is None else x.new_empty((rows, cols))
        rstd = x.new_empty(rows, dtype=torch.float32)
        if cols == 0:  # the library writes nothing; a mean over no values is none
            rstd.fill_(float("nan"))
        call("df_rmsnorm_forward", dt, x.data_ptr(), rows, cols, ldx, _ptr(residual), ldr,
             None if residual is None else s.data_ptr(), cols, _ptr(gamma), float(eps), y.data_ptr(), cols,
             rstd.data_ptr(), _stream())
    return y, s, rstd


def rmsnorm_quantize(x, gamma=None, eps=1e-5, residual=None, fmt: Fmt = Fmt.E4M3, want_y=False, scale_dtype=None):
    """:func:`rmsnorm_forward` whose output is fp8 codes with a scale per 128
    columns, the operand of :func:`gemm_blocks` (df_rmsnorm_quantize): returns (q
    [R, ceil16(C)], scales [ceil(C/128), R], s, rstd), with ``want_y`` y in x's type
    behind them.  Codes come from y in fp32, not from y as rounded."""
    fn, torch = "rmsnorm_quantize", _torch()
    rows, cols, ldx, ldr = _norm_args(fn, x, gamma, residual)
    scale_dtype = scale_dtype or torch.float8_e8m0fnu
    kind, codes, dt = _kind(fn, scale_dtype), _code_dtype(fmt), _in_dtype(x)
    ldq = round16(cols)
    with _on(x):
        q = x.new_empty((rows, ldq), dtype=codes)
        sc, ldsc = _new_scales(x, -(-cols // BLOCK), rows, scale_dtype)
        s = x if residual is None else x.new_empty((rows, cols))
        y = x.new_empty((rows, cols)) if want_y else None
        rstd = x.new_empty(rows, dtype=torch.float32)
        if cols == 0:
            rstd.fill_(float("nan"))
        call("df_rmsnorm_quantize", dt, x.data_ptr(), rows, cols, ldx, _ptr(residual), ldr,
             None if residual is None else s.data_ptr(), cols, _ptr(gamma), float(eps), _ptr(y), cols, rstd.data_ptr(),
             int(fmt), q.data_ptr(), ldq, kind, sc.data_ptr(), ldsc, _stream())
    return (q, sc, s, rstd, y) if want_y else (q, sc, s, rstd)


def rmsnorm_backward(dy, x, gamma=None, rstd=None, eps=1e-5, dresidual=None, sums=True):
    """The gradients of :func:`rmsnorm_forward` (df_rmsnorm_backward), x being what
    the norm saw: returns (dx, dgamma), the last in fp32 (None with
    ``sums=False``).  Without rstd it is taken from x at eps again.  ``dresidual``
    (the gradient that reaches the residual stream past the norm) is added to dx."""
    fn, torch = "rmsnorm_backward", _torch()
    if x.dim() != 2:
        raise ValueError(f"{fn}: x has {x.dim()} dimensions, not 2")
    shape, dtype, at = x.shape, x.dtype, x.get_device()
    rows, cols = shape
    if (rows | cols) > _INT_MAX:
        _fits(fn, rows, cols)
    ldx = lddy = lddr = cols
    if not (at >= 0 and x.is_contiguous() and _plain(dy, shape, dtype, at) and _plain(dresidual, shape, dtype, at)
            and _plain(gamma, (cols,), dtype, at) and _plain(rstd, (rows,), torch.float32, at)):
        _check_gpu(fn, dy=dy, x=x, gamma=gamma, rstd=rstd, dresidual=dresidual)
        ldx, lddy = _rows(fn, "x", x, shape, dtype), _rows(fn, "dy", dy, shape, dtype)
        lddr = cols if dresidual is None else _rows(fn, "dresidual", dresidual, shape, dtype)
        _row_vector(fn, "gamma", gamma, cols, dtype)
        _row_vector(fn, "rstd", rstd, rows, torch.float32)
    dt = _in_dtype(x)
    with _on(x):
        dx = x.new_empty(shape)
        dg = x.new_empty(cols, dtype=torch.float32) if sums else None
        # not a cached one: a captured graph keeps the workspace it was given
        nws = _workspace_bytes("df_rmsnorm_backward", rows, cols)
        ws = x.new_empty(nws, dtype=torch.uint8)
        call("df_rmsnorm_backward", dt, dy.data_ptr(), lddy, x.data_ptr(), ldx, rows, cols, _ptr(gamma), _ptr(rstd),
             float(eps), _ptr(dresidual), lddr, dx.data_ptr(), cols, _ptr(dg), ws.data_ptr(), nws, _stream())
    return dx, dg
