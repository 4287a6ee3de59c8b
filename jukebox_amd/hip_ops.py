"""Thin tensor-level wrappers over the C ABI (include/jukebox_hip.h).

torch supplies device memory and the current HIP stream only; every computation below happens
in libjukebox_hip.so.  Tensors must live on the GPU and be contiguous unless a function says
otherwise; there is no CPU path.
"""
import ctypes as C
import math
from array import array

import torch

from . import _lib as L


def _chk_cuda(*ts):
    for t in ts:
        if t is not None and (not t.is_cuda or not t.is_contiguous()):
            raise L.JukeboxHipError("expected contiguous GPU tensors")


class PackedWeight:
    """A K x J matrix in MFMA fragment order (see csrc/gemm.hip) plus its logical dims.
    `taps` > 1 holds the per-tap matrices of a (transposed) convolution back to back."""

    def __init__(self, data, K, J, dtype, taps=1, split=False, unscale=1.0):
        self.data, self.K, self.J, self.dtype, self.taps = data, K, J, dtype, taps
        self.tap_stride = data.numel() // taps
        self.split = split              # fp32 matrix as hi / lo f16 images (jb_gemm_args.w_split); `data` holds the raw words
        self.unscale = unscale          # split images hold s * W for a power of two s: 1 / s (jb_gemm_args.w_split_unscale)

    @property
    def ptr(self):
        return self.data.data_ptr()


def pack_weight(w, K, J, stride_k, stride_j, dtype, out=None, offset_elems=0):
    """Pack logical matrix M[k, j] = w.flatten()[offset + k*stride_k + j*stride_j] into `dtype`."""
    _chk_cuda(w)
    code = L.dtype_code(dtype)
    nbytes = L.lib().jb_packed_weight_bytes(K, J, code)
    if out is None:
        out = torch.empty(nbytes // (2 if code == L.F16 else 4), dtype=dtype, device=w.device)
    src = w.data_ptr() + offset_elems * w.element_size()
    L.check(L.lib().jb_pack_weight(src, L.dtype_code(w.dtype), stride_k, stride_j, K, J, out.data_ptr(), code, L.stream()))
    return out


def pack_conv1d_w(w, dtype):
    """Conv1D.w (n_in, n_out) (jukebox/transformer/ops.py:89-95)."""
    K, J = w.shape
    return PackedWeight(pack_weight(w, K, J, J, 1, dtype), K, J, dtype)


class FoldedLN:
    """LayerNorm folded into the Conv1D that follows it (jb_gemv_args.ln_fold_c1): LN(x)·W + b is evaluated as
    rstd·(x·W' - mean·c1) + b' with W' = diag(gamma)·W (packed, engine dtype), c1 = column sums of W' as stored,
    b' = beta·W + b.  `w` is Conv1D.w (n_in, n_out); W is first rounded to the engine dtype, as the reference's
    `w.type_as(x)` does (jukebox/transformer/ops.py:99)."""

    def __init__(self, w, b, gamma, beta, dtype):
        K, J = w.shape
        w_used = w.to(dtype).double()
        wf = (gamma.double()[:, None] * w_used).to(dtype).contiguous()
        self.wf = wf                                           # unpacked diag(gamma)·W
        self.pw = PackedWeight(pack_weight(wf, K, J, J, 1, dtype), K, J, dtype)
        self.c1 = wf.double().sum(0).float().contiguous()
        self.bias = (beta.double() @ w_used + b.double()).float().contiguous()


def ln_fold_supported(dtype, K, J, n_rows):
    return bool(L.lib().jb_gemv_ln_fold_supported(L.dtype_code(dtype), K, J, n_rows))


def pack_linear_w(w, dtype):
    """nn.Linear.weight (out, in): logical [k=in][j=out]."""
    J, K = w.shape
    return PackedWeight(pack_weight(w, K, J, 1, K, dtype), K, J, dtype)


def pack_conv_taps(w, dtype, transposed=False, split=False):
    """nn.Conv1d weight (Cout, Cin, k) or nn.ConvTranspose1d weight (Cin, Cout, k): one K=Cin x J=Cout
    matrix per tap.  split (fp32 only, Cin a multiple of 32): every tap as the hi / lo pair of f16 images that lets the
    fp32 conv stacks run on the f16 matrix cores at fp32 accuracy (jb_gemm_args.w_split) -- the same bytes per tap."""
    w = w.contiguous()
    unscale = 1.0
    if split:
        assert dtype == torch.float32 and w.shape[0 if transposed else 1] % 32 == 0
        # (once per layer, at pack time) the image holds s * w with the power of two s that puts max |w| into [128, 256): every
        # weight down to 2^-22 of the largest keeps a NORMAL hi half, i.e. 2^-22 relative precision after the split, whatever the
        # layer's scale -- unscaled, a trained layer with |w| < 6e-5 would have subnormal hi halves (exact: powers of two)
        amax = float(w.abs().max())
        assert math.isfinite(amax), "f16-split weight image: weights must be finite"
        if amax > 0.0:
            scale = 2.0 ** (8 - math.frexp(amax)[1])
            w, unscale = (w.float() * scale).contiguous(), 1.0 / scale
    if transposed:
        Cin, Cout, k = w.shape
        sk, sj = Cout * k, k
    else:
        Cout, Cin, k = w.shape
        sk, sj = k, Cin * k
    code = L.F16_SPLIT if split else L.dtype_code(dtype)
    per = L.lib().jb_packed_weight_bytes(Cin, Cout, code) // (2 if code == L.F16 else 4)
    out = torch.empty(per * k, dtype=dtype, device=w.device)
    for tap in range(k):
        dst = out[tap * per:(tap + 1) * per]
        if split:
            L.check(L.lib().jb_pack_weight(w.data_ptr() + tap * w.element_size(), L.dtype_code(w.dtype), sk, sj, Cin, Cout,
                                           dst.data_ptr(), code, L.stream()))
        else:
            pack_weight(w, Cin, Cout, sk, sj, dtype, out=dst, offset_elems=tap)
    return PackedWeight(out, Cin, Cout, dtype, taps=k, split=split, unscale=unscale)


def layernorm(x, gamma, beta, eps=1e-5, out_dtype=None):
    """ops.LayerNorm.forward (jukebox/transformer/ops.py:14-24)."""
    _chk_cuda(x, gamma, beta)
    W = x.shape[-1]
    y = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    L.check(L.lib().jb_layernorm_fwd(x.data_ptr(), L.dtype_code(x.dtype), y.data_ptr(), L.dtype_code(y.dtype),
                                     gamma.data_ptr(), beta.data_ptr(), x.numel() // W, W, eps, L.stream()))
    return y


def gemm(A, pw, bias=None, out=None, res=None, n_seq=1, t_in=None, t_out=None, shifts=(0,), in_stride=1,
         out_stride=1, out_offset=0, out_rows_per_seq=None, pre_relu=False, act=L.ACT_NONE, res_scale=1.0, in_seq_pitch=None):
    """Sequence/tap GEMM (see jb_gemm).  A: (n_seq*t_in, lda>=K); returns (n_seq*out_rows_per_seq, J).
    in_seq_pitch: rows between the starts of two sequences in A when they are not packed (t_in must then be given)."""
    _chk_cuda(A, bias, out, res)
    rows_in = A.shape[0]
    assert in_seq_pitch is None or t_in is not None
    t_in = t_in if t_in is not None else rows_in // n_seq
    t_out = t_out if t_out is not None else t_in
    orps = out_rows_per_seq if out_rows_per_seq is not None else t_out * out_stride
    if out is None:
        out = torch.empty((n_seq * orps, pw.J), dtype=A.dtype, device=A.device)
    a = L.GemmArgs()
    a.dtype = L.dtype_code(A.dtype)
    a.A, a.lda = A.data_ptr(), A.stride(0)
    a.W, a.tap_stride = pw.ptr, pw.tap_stride
    a.bias = L.ptr(bias)
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.res, a.ldr = L.ptr(res), (res.stride(0) if res is not None else 0)
    a.n_seq, a.t_in, a.t_out = n_seq, t_in, t_out
    a.in_seq_stride, a.out_seq_stride = (t_in if in_seq_pitch is None else in_seq_pitch), orps
    a.K, a.J = pw.K, pw.J
    if len(shifts) != pw.taps:
        raise L.JukeboxHipError(f"{len(shifts)} shifts for a weight with {pw.taps} taps")
    a.n_taps, a.in_stride = len(shifts), in_stride
    for i, s in enumerate(shifts):
        a.shift[i] = s
    a.out_stride, a.out_offset = out_stride, out_offset
    a.pre_relu, a.act, a.res_scale = int(pre_relu), act, res_scale
    a.w_split = int(pw.split)
    a.w_split_unscale = float(pw.unscale)
    if pw.split:            # scratch for the activations' hi / lo images (same bytes as the fp32 rows); the caching allocator recycles it
        scratch = torch.empty(n_seq * t_in * pw.K, dtype=torch.float32, device=A.device)
        a.a_split, a.a_split_bytes = scratch.data_ptr(), scratch.numel() * 4
    L.check(L.lib().jb_gemm(C.byref(a), L.stream()))
    return out


def check_split_overflow(wait=True):
    """Raise if a conv-stack launch on the f16-split path (jb_gemm_args.w_split) has seen an activation outside the half range
    (or a NaN) since the last check: its output is not the convolution.  The flag is a host-coherent word, so reading it costs
    nothing and waits for nothing: wait=True synchronises the device first (end of a job, tests: the launches just enqueued
    count), wait=False looks at what has FINISHED so far -- the sampler's look after every window, which must not stall the
    other levels' streams (a window's conv stacks ran seconds before its last token)."""
    if wait:
        torch.cuda.synchronize()
    rc = L.lib().jb_gemm_split_overflow(1)
    if rc < 0:
        L.check(rc)
    if rc:
        raise L.JukeboxHipError("a convolution on the f16-split path was given activations outside the half range (|x| > 65504 or "
                                "NaN): its output is invalid (jukebox_amd.vqvae.rows.SPLIT_F16 = False selects the exact-fp32 kernel)")


def gemm_qkv(h, pw, bias, n_seq, n_q, S, kcache, vcache, t0):
    """c_attn projection of a chunk with the k/v parts written into the caches at positions t0.. (jb_gemm
    qkv_split).  h: (n_seq*n_q, K).  Returns q: (n_seq*n_q, S)."""
    _chk_cuda(h, bias, kcache, vcache)
    q = torch.empty((n_seq * n_q, S), dtype=h.dtype, device=h.device)
    a = L.GemmArgs()
    a.dtype = L.dtype_code(h.dtype)
    a.A, a.lda = h.data_ptr(), h.stride(0)
    a.W, a.tap_stride, a.bias = pw.ptr, pw.tap_stride, L.ptr(bias)
    a.out, a.ldo = q.data_ptr(), S
    a.n_seq, a.t_in, a.t_out = n_seq, n_q, n_q
    a.in_seq_stride, a.out_seq_stride = n_q, n_q
    a.K, a.J = pw.K, pw.J
    a.n_taps, a.in_stride, a.out_stride, a.res_scale = 1, 1, 1, 1.0
    a.qkv_split, a.S = 1, S
    a.kcache, a.vcache, a.cache_cap, a.cache_t0 = kcache.data_ptr(), vcache.data_ptr(), kcache.shape[1], t0
    L.check(L.lib().jb_gemm(C.byref(a), L.stream()))
    return q


def tap_view(pw, taps):
    """PackedWeight holding only the listed taps (must be equally spaced) -- for transposed-conv phases."""
    step = taps[1] - taps[0] if len(taps) > 1 else 1
    assert all(taps[i] == taps[0] + i * step for i in range(len(taps)))
    base = pw.data[taps[0] * pw.tap_stride:]
    v = PackedWeight(base, pw.K, pw.J, pw.dtype, taps=1, split=pw.split, unscale=pw.unscale)
    v.tap_stride = pw.tap_stride * step
    v.taps = len(taps)
    return v


def gemv(x, pw, bias=None, ln=None, res=None, act=L.ACT_NONE, out=None, eps=1e-5, ln_fold=None, parts=None, out2=None,
         add2=None, t_dev=None, qkv=None):
    """Decode-step skinny GEMM (see jb_gemv).  x: (n_rows<=64, K).  ln = (gamma, beta): normalise the rows in the
    kernel; ln_fold = FoldedLN: the folded form (pw / bias are taken from it); parts = (x_parts (N, P, K) f16,
    ml (N, H, P, 2) fp32): the operand is the merge of the key-split attention's partial states (x must be None);
    out2 (N, J) fp32 [+ add2 (N, T, J) fp32 read at row *t_dev]: the second, fp32 output of the plain projection;
    qkv = (S, kcache, vcache or None, vcache_wide or None): c_attn of the decode step -- columns q | k | v | v' with the
    cache rows written at *t_dev; returns q (N, S)."""
    if ln_fold is not None:
        assert ln is None and bias is None and pw is None
        pw, bias = ln_fold.pw, ln_fold.bias
    _chk_cuda(x, bias, res, out, out2, add2)
    src = x if x is not None else parts[0]
    if out is None:
        out = torch.empty((src.shape[0], qkv[0] if qkv is not None else pw.J), dtype=src.dtype, device=src.device)
    a = L.GemvArgs()
    if qkv is not None:
        S, kc, vc, vw = qkv
        _chk_cuda(kc, vc, vw, t_dev)
        a.qkv_split, a.S, a.kcache, a.vcache, a.cache_cap = 1, S, kc.data_ptr(), L.ptr(vc), kc.shape[1]
        if vw is not None:
            a.vcache_wide, a.wide = vw.data_ptr(), vw.shape[2]
        a.t_dev = L.ptr(t_dev)
    a.dtype = L.dtype_code(src.dtype)
    a.n_rows = src.shape[0]
    if x is not None:
        a.x, a.ldx = x.data_ptr(), x.stride(0)
    else:
        xp, ml = parts
        _chk_cuda(xp, ml)
        a.x_parts, a.x_ml, a.n_parts, a.n_head = xp.data_ptr(), ml.data_ptr(), xp.shape[1], ml.shape[1]
        a.d_head, a.ldx = xp.shape[2] // ml.shape[1], xp.shape[2]
    if out2 is not None:
        a.out2, a.ldo2 = out2.data_ptr(), out2.stride(0)
        if add2 is not None:
            a.add2, a.add2_n_stride, a.add2_t_stride = add2.data_ptr(), add2.stride(0), add2.stride(1)
        a.t_dev = L.ptr(t_dev)
    if ln is not None:
        a.ln_gamma, a.ln_beta, a.ln_eps = ln[0].data_ptr(), ln[1].data_ptr(), eps
    if ln_fold is not None:
        a.ln_fold_c1, a.ln_eps = ln_fold.c1.data_ptr(), eps
    a.W, a.bias, a.K, a.J = pw.ptr, L.ptr(bias), pw.K, pw.J
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.res, a.ldr = L.ptr(res), (res.stride(0) if res is not None else 0)
    a.act = act
    L.check(L.lib().jb_gemv(C.byref(a), L.stream()))
    return out


def attn_decode(func, q, kcache, vcache, n_head, block_ctx, t_dev, max_len):
    """q (N, S); caches (N, cap, S); returns (N, S)."""
    _chk_cuda(q, kcache, vcache, t_dev)
    N, S = q.shape
    out = torch.empty_like(q)
    L.check(L.lib().jb_attn_decode(L.dtype_code(q.dtype), func, q.data_ptr(), q.stride(0), kcache.data_ptr(),
                                   vcache.data_ptr(), kcache.shape[1], out.data_ptr(), out.stride(0), N, n_head,
                                   S // n_head, block_ctx or 0, t_dev.data_ptr(), max_len, L.stream()))
    return out


def attn_decode_wide(func, q, kcache, vcache_w, res, bias, block_ctx, t_dev, max_len):
    """Wide-value decode attention of a single-head fp16 layer (jb_attn_decode_wide): q (N, S); kcache (N, cap, S);
    vcache_w (N, cap, W) rows v' = v·Wp; returns x_out (N, W) = res + (sum_k p_k v'_k + bias)."""
    _chk_cuda(q, kcache, vcache_w, res, bias, t_dev)
    N, S = q.shape
    W = vcache_w.shape[2]
    out = torch.empty_like(res)
    L.check(L.lib().jb_attn_decode_wide(func, q.data_ptr(), q.stride(0), kcache.data_ptr(), vcache_w.data_ptr(),
                                        kcache.shape[1], res.data_ptr(), res.stride(0), bias.data_ptr(), out.data_ptr(),
                                        out.stride(0), N, S, W, block_ctx or 0, t_dev.data_ptr(), max_len, L.stream()))
    return out


def attn_decode_split(func, q, kcache, vcache, n_head, block_ctx, t_dev, max_keys, n_parts):
    """Key-split decode attention (fp16): returns (parts (N, n_parts, S) f16, ml (N, n_head, n_parts, 2) fp32)."""
    _chk_cuda(q, kcache, vcache, t_dev)
    N, S = q.shape
    parts = torch.empty((N, n_parts, S), dtype=q.dtype, device=q.device)
    ml = torch.empty((N, n_head, n_parts, 2), dtype=torch.float32, device=q.device)
    L.check(L.lib().jb_attn_decode_split(func, q.data_ptr(), q.stride(0), kcache.data_ptr(), vcache.data_ptr(),
                                         kcache.shape[1], parts.data_ptr(), ml.data_ptr(), N, n_head, S // n_head,
                                         block_ctx or 0, t_dev.data_ptr(), max_keys, n_parts, L.stream()))
    return parts, ml


def attn_prefill(func, q, kcache, vcache, n_head, block_ctx, t0):
    """q (N, n_q, S) for positions t0..t0+n_q-1; caches (N, cap, S) already hold them."""
    _chk_cuda(q, kcache, vcache)
    N, nq, S = q.shape
    out = torch.empty_like(q)
    L.check(L.lib().jb_attn_prefill(L.dtype_code(q.dtype), func, q.data_ptr(), kcache.data_ptr(), vcache.data_ptr(),
                                    kcache.shape[1], out.data_ptr(), N, n_head, S // n_head, block_ctx or 0, t0, nq,
                                    L.stream()))
    return out


# ---- keys and values in pages ---------------------------------------------------------------------------------------------

_INT_MAX = 0x7fffffff
_PAGED_TYPES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}


def _paged_type(t, *ts):
    """dtype code of the paged cache's operators (single, half and bfloat16) for tensors that must share it."""
    dtype = t.dtype
    code = _PAGED_TYPES.get(dtype)
    for x in ts:
        if x.dtype != dtype:
            code = None
    if code is None:
        raise L.JukeboxHipError(f"expected one type of float32, float16, bfloat16; got {', '.join(str(x.dtype) for x in (t, *ts))}")
    return code


def _chk_paged(first, *ts):
    """Every tensor on the first one's GPU."""
    if not first.is_cuda:
        raise L.JukeboxHipError("expected GPU tensors")
    i = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != i:
            raise L.JukeboxHipError("expected tensors on one GPU")


def _chk_int(name, t, n=None):
    """A contiguous int32 array (of n elements)."""
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
        raise L.JukeboxHipError(f"{name}: expected a contiguous int32 array" + ("" if n is None else f" of {n} elements"))


def _chk_table(table):
    if table.dtype != torch.int32 or table.dim() != 2:
        raise L.JukeboxHipError("table: expected int32 rows of page numbers")
    n, width = table.shape
    stride, one = table.stride()
    if width == 0 or (width > 1 and one != 1):
        raise L.JukeboxHipError("table: expected int32 rows of page numbers")
    if n < 2:           # the row of a table of one row may carry any stride
        stride = width
    elif stride < width:
        raise L.JukeboxHipError("table: rows overlap")
    return n, width, stride


def _launch(fn, t, *args):
    """A call of the library on the current stream of tensor t's own GPU."""
    i = t.get_device()
    # (the raw handles: a Stream object and its device index cost more than the rest of a small call)
    if i == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        L.check(rc)


def attn_paged(q, kpool, vpool, table, lens, cu_q, max_q=None, max_len=None, func=0, block_ctx=0, window=0, scale=None, out=None):
    """Attention of every sequence's newest tokens over keys and values in pages (jb_attn_paged).

    q (n_tokens, n_head, d_head): rows cu_q[i] .. cu_q[i + 1] - 1 are the last positions of sequence i, whose keys and values
    the cache holds already.  kpool, vpool (n_pages, page_size, n_kv_head, d_head), any strides that both share, channels
    contiguous.  table (n_seq, max_pages), lens (n_seq), cu_q (n_seq + 1): int32 on the GPU.  max_q, max_len: the most queries
    / tokens of a sequence, which shape the launch and choose the kernel.  Default: all of the table's pages; all rows of q, but 1
    where q has a row a sequence.  func, block_ctx: the
    pattern (dense, block, transpose, prev); window: the query at position p sees p - window + 1 .. p (dense).  scale:
    1 / sqrt(d_head) by default.  Returns (n_tokens, n_head, d_head); `out` overlaps no input, and its rows outside every sequence
    stay as they are.

    In 16 bits, calls with max_q * n_head / n_kv_head >= 64, heads of up to 256 channels and no transpose pattern go to the kernel of
    chunks, which rounds the probabilities to the type once; all others carry them in two parts (jb_attn_paged has the bounds)."""
    code = _paged_type(q, kpool, vpool)
    _chk_paged(q, kpool, vpool, table, lens, cu_q, out)
    if q.dim() != 3 or kpool.dim() != 4 or kpool.shape != vpool.shape or kpool.stride() != vpool.stride() or q.shape[2] != kpool.shape[3]:
        raise L.JukeboxHipError("expected q (n_tokens, n_head, d_head) and kpool, vpool (n_pages, page_size, n_kv_head, d_head) of equal strides")
    T, H, D = q.shape
    P, page, KV, _ = kpool.shape
    n, width, table_stride = _chk_table(table)
    _chk_int("lens", lens, n)
    _chk_int("cu_q", cu_q, n + 1)
    if out is None:
        out = torch.empty((T, H, D), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise L.JukeboxHipError("out: expected q's shape and type")
    if q.stride(2) != 1 or kpool.stride(3) != 1 or out.stride(2) != 1:
        raise L.JukeboxHipError("expected contiguous channels")
    ps, rs, hs = kpool.stride()[:3]
    if max_q is None:   # as many rows as sequences: a step of one token each (64 of 4000 tokens, 32 heads on 8: 213 us; as a chunk 339)
        max_q = 1 if T == n else T
    a = L.AttnPagedArgs(code, func, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0) if T > 1 else H * D,
                        out.stride(1) if H > 1 else D, kpool.data_ptr(), vpool.data_ptr(), ps, rs, hs, P, page, table.data_ptr(),
                        table_stride, width, lens.data_ptr(), cu_q.data_ptr(), T, n, H, KV, D, min(max_q or 1, T),
                        min(width * page if max_len is None else max_len, _INT_MAX), min(block_ctx or 0, _INT_MAX), min(window or 0, _INT_MAX),
                        1.0 / math.sqrt(D) if scale is None else scale, None, 0)
    lib = L.lib()
    need = lib.jb_attn_paged_workspace(C.byref(a))
    if need < 0:
        L.check(need)
    if need:            # the caching allocator keeps it for this stream (or this captured graph) until the launches have run
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _launch(lib.jb_attn_paged, q, C.byref(a))
    return out


def kv_write(k, v, kpool, vpool, slots):
    """New key / value rows into pages (jb_kv_write): k, v (n_tokens, n_kv_head, d_head) to the cache rows slots (n_tokens,
    int64: page * page_size + row in the page; pages_extend makes them) of kpool, vpool (n_pages, page_size, n_kv_head, d_head).
    Rows whose slot is -1 are left out."""
    code = _paged_type(k, v, kpool, vpool)
    _chk_paged(k, v, kpool, vpool, slots)
    if k.dim() != 3 or kpool.dim() != 4 or k.shape != v.shape or kpool.shape != vpool.shape or k.shape[1:] != kpool.shape[2:]:
        raise L.JukeboxHipError("expected k, v (n_tokens, n_kv_head, d_head) and kpool, vpool (n_pages, page_size, n_kv_head, d_head)")
    if k.stride() != v.stride() or kpool.stride() != vpool.stride() or k.stride(2) != 1 or kpool.stride(3) != 1:
        raise L.JukeboxHipError("expected equal strides of k and v and of kpool and vpool, and contiguous channels")
    T, KV, D = k.shape
    if slots.dtype != torch.int64 or slots.shape != (T,) or not slots.is_contiguous():
        raise L.JukeboxHipError("slots: expected a contiguous int64 array with an entry per token")
    ts, hs = k.stride()[:2]
    ps, rs, phs = kpool.stride()[:3]
    if KV == 1:         # a single head's stride is anything
        hs = phs = D
    a = L.KvWriteArgs(code, k.data_ptr(), v.data_ptr(), ts, hs, kpool.data_ptr(), vpool.data_ptr(), ps, rs, phs, kpool.shape[0],
                      kpool.shape[1], slots.data_ptr(), T, KV, D)
    _launch(L.lib().jb_kv_write, k, C.byref(a))


def _page_table(table, lens, ref, page_size, status=None):
    n, width, stride = _chk_table(table)
    if lens is not None:
        _chk_int("lens", lens, n)
    _chk_int("ref", ref)
    if status is not None:
        _chk_int("status", status, 1)
    _chk_paged(table, lens, ref, status)
    return L.PageTable(table.data_ptr(), stride, n, width, L.ptr(lens), ref.data_ptr(), ref.shape[0], page_size)


def _page_pools(pools, n_pages, device):
    """Pools of equal shape and strides, (n_pages, ...) with contiguous pages; any type."""
    if len(pools) == 0:
        return L.PagePools(None, 0, n_pages, 1, 1)
    p = pools[0]
    if p.dim() == 0:
        raise L.JukeboxHipError("pools: expected arrays of pages")
    shape, stride, dtype, size, gpu = p.shape, p.stride(), p.dtype, p.element_size(), device.index
    n = 1
    for m, st in zip(reversed(shape[1:]), reversed(stride[1:])):
        if m > 1 and st != n:
            raise L.JukeboxHipError("pools: expected contiguous pages")
        n *= m
    if shape[0] != n_pages or n == 0 or (n_pages > 1 and stride[0] < n):
        raise L.JukeboxHipError(f"pools: expected {n_pages} pages that do not overlap")
    for x in pools:
        if x.shape != shape or x.stride() != stride or x.dtype != dtype or x.get_device() != gpu:
            raise L.JukeboxHipError("pools: expected equal shapes, strides and types on the table's GPU")
    base = (C.c_uint64 * len(pools)).from_buffer(array("Q", [x.data_ptr() for x in pools]))
    return L.PagePools(C.cast(base, C.POINTER(L.vp)), len(pools), n_pages, n * size, (stride[0] if n_pages > 1 else n) * size)


def pages_extend(table, lens, ref, cu_new, page_size, n_tokens, status):
    """Room for cu_new[i + 1] - cu_new[i] more tokens of every sequence (jb_pages_extend): takes free pages from the lowest on,
    adds to lens, and returns the cache row of each of the n_tokens new tokens (int64; -1 behind the last).  Without enough free
    pages nothing changes, all slots are -1 and status (one int32, which the caller clears) says so."""
    t = _page_table(table, lens, ref, page_size, status)
    if not 0 <= n_tokens <= _INT_MAX:
        raise L.JukeboxHipError("n_tokens: expected 0 to 2^31 - 1")
    _chk_int("cu_new", cu_new, t.n_seq + 1)
    _chk_paged(table, cu_new)
    slots = torch.empty(n_tokens, dtype=torch.int64, device=table.device)
    work = torch.empty(1 + 2 * t.n_seq + t.n_pages, dtype=torch.int32, device=table.device)
    _launch(L.lib().jb_pages_extend, table, C.byref(t), cu_new.data_ptr(), n_tokens, slots.data_ptr(), work.data_ptr(), status.data_ptr())
    return slots


def pages_free(table, lens, ref, rows, status):
    """The sequences in these rows (int32) of the table end (jb_pages_free): references given back, rows -1, lengths 0."""
    t = _page_table(table, lens, ref, 1, status)
    _chk_int("rows", rows)
    _chk_paged(table, rows)
    _launch(L.lib().jb_pages_free, table, C.byref(t), rows.data_ptr(), rows.shape[0], status.data_ptr())


def pages_fork(pools, table, lens, ref, src, dst, page_size, status):
    """Row dst[i] of the table becomes a fork of row src[i] (jb_pages_fork): shares the full pages and gets a copy of the last,
    part-filled one in every pool.  pools: a list of (n_pages, ...) tensors -- every layer's keys and values -- with contiguous
    pages.  The rows dst are empty before (pages_free), and no source."""
    t = _page_table(table, lens, ref, page_size, status)
    p = _page_pools(pools, t.n_pages, table.device)
    _chk_int("src", src)
    _chk_int("dst", dst, src.shape[0])
    _chk_paged(table, src, dst)
    work = torch.empty(2 + 4 * src.shape[0], dtype=torch.int32, device=table.device)
    _launch(L.lib().jb_pages_fork, table, C.byref(t), C.byref(p), src.data_ptr(), dst.data_ptr(), src.shape[0], work.data_ptr(), status.data_ptr())


def pages_compact(pools, table, ref):
    """Live pages (ref > 0) moved to the lowest numbers in every pool (jb_pages_compact).  Returns the table and the reference
    counts that go with the moved pages; the ones given stay as they are."""
    t = _page_table(table, None, ref, 1)
    p = _page_pools(pools, t.n_pages, table.device)
    table_out, ref_out = torch.empty(table.shape, dtype=torch.int32, device=table.device), torch.empty_like(ref)
    work = torch.empty(2 + 3 * t.n_pages, dtype=torch.int32, device=table.device)
    _launch(L.lib().jb_pages_compact, table, C.byref(t), C.byref(p), table_out.data_ptr(), ref_out.data_ptr(), work.data_ptr())
    return table_out, ref_out


def pages_copy(pools, src, dst):
    """Page src[i] of every pool to page dst[i] (jb_pages_copy; int32 arrays).  No target twice, no target that is a source."""
    if len(pools) == 0:
        return
    p = _page_pools(pools, pools[0].shape[0] if pools[0].dim() else 0, pools[0].device)
    _chk_int("src", src)
    _chk_int("dst", dst, src.shape[0])
    _chk_paged(pools[0], src, dst)
    _launch(L.lib().jb_pages_copy, src, C.byref(p), src.data_ptr(), dst.data_ptr(), src.shape[0])


def vq_gather(codes, codebook):
    """(N, T) int64 -> (N, T, emb) fp32 (BottleneckBlock.decode, channels-last)."""
    _chk_cuda(codes, codebook)
    out = torch.empty((*codes.shape, codebook.shape[1]), dtype=torch.float32, device=codes.device)
    L.check(L.lib().jb_vq_gather(codes.data_ptr(), codebook.data_ptr(), out.data_ptr(), codes.numel(),
                                 codebook.shape[1], codebook.shape[0], L.stream()))
    return out


def vq_argmin(x, xk, codebook):
    _chk_cuda(x, xk, codebook)
    codes = torch.empty(x.shape[0], dtype=torch.int64, device=x.device)
    L.check(L.lib().jb_vq_argmin(x.data_ptr(), xk.data_ptr(), codebook.data_ptr(), codes.data_ptr(), x.shape[0],
                                 x.shape[1], codebook.shape[0], L.stream()))
    return codes


def sample_logits(logits, params_dev, tokens, t_dev, preds=None):
    _chk_cuda(logits, tokens, t_dev, preds)
    L.check(L.lib().jb_sample_logits(logits.data_ptr(), logits.shape[0], logits.shape[1], params_dev.data_ptr(),
                                     tokens.data_ptr(), tokens.stride(0), t_dev.data_ptr(), L.ptr(preds),
                                     preds.stride(0) if preds is not None else 0, L.stream()))


def make_sample_params(temp=1.0, top_k=0, top_p=0.0, seed=0, sample_base=0, pos_base=0, stream_id=0, device="cuda"):
    """Device copy of jb_sample_params."""
    p = L.SampleParams(temp, top_k, top_p, sample_base, seed & 0xFFFFFFFFFFFFFFFF, pos_base, stream_id)
    raw = bytes(p)
    return torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(device)


def sample_filtered(logits, u, temp=1.0, top_k=0, top_p=0.0, min_p=0.0, out=None):
    """One token a row (int64) from given uniform numbers after temperature, top-k, top-p and min-p (jb_sample_filtered has the
    definition, which the answer equals whatever the sizes).  logits (rows, bins), float32, float16 or bfloat16, rows of any
    pitch that does not overlap them, or one row expanded to many; u (rows) float32 in [0, 1).  temp, top_k, top_p, min_p: a number for all rows or an array with one for each (int32 for
    top_k, float32 for the others).  temp <= 0: the largest logit; top_k <= 0, top_p <= 0 or >= 1, min_p <= 0: off.  -inf and NaN
    are forbidden tokens; a row without any other gives -1."""
    code = _paged_type(logits)
    if logits.dim() != 2 or logits.shape[1] == 0 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise L.JukeboxHipError("logits: expected rows of contiguous values")
    n, bins = logits.shape
    if out is None:
        out = torch.empty(n, dtype=torch.int64, device=logits.device)
    elif out.dtype != torch.int64 or out.shape != (n,) or not out.is_contiguous():
        raise L.JukeboxHipError("out: expected a contiguous int64 array with an entry per row")
    ptrs, vals, each = [], [], []
    for name, x, dtype in (("u", u, torch.float32), ("temp", temp, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if torch.is_tensor(x):
            if x.dtype != dtype or x.shape != (n,) or not x.is_contiguous():
                raise L.JukeboxHipError(f"{name}: expected a contiguous {dtype} array with an entry per row")
            ptrs.append(x.data_ptr())
            vals.append(0)
            each.append(x)
        elif name == "u":
            raise L.JukeboxHipError("u: expected an array with a uniform number per row")
        else:
            ptrs.append(None)
            vals.append(max(min(x, _INT_MAX), 0) if name == "top_k" else x)
    _chk_paged(logits, out, *each)
    a = L.SampleFilteredArgs(code, logits.data_ptr(), logits.stride(0) if n > 1 else bins, n, bins, *ptrs, *vals[1:], out.data_ptr())
    _launch(L.lib().jb_sample_filtered, logits, C.byref(a))
    return out
