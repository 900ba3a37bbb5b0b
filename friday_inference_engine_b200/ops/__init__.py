"""The library's operations, callable on torch tensors: what the tests of single kernels
and the measurements use.  Every function marshals its arguments to the C++ operation of
the same name (ops/ops.cpp, include/friday/ops.h), which chooses and launches this
library's own CUDA kernels; nothing is computed here, and there is no CPU path.

Kernels run on the legacy default stream, which is also torch's default, so they are
ordered with the torch operations around them.  (rotate_axes, rope_axes_kv_write and
attention_shared run on torch's current stream instead, may be captured into a CUDA graph
there, and may be called from several threads at once.)
"""
from ctypes import byref, c_int, c_int64, c_void_p
from functools import lru_cache

from .. import native

_CODES = None


def _codes():
    global _CODES
    if _CODES is None:
        import torch
        _CODES = {torch.float32: 0, torch.bfloat16: 1, torch.int32: 2}
    return _CODES


def _t(t):
    """FridayTensor for a torch tensor (None -> a null pointer)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise native.KernelError("tensor on %s: this library runs on CUDA devices only, it has no CPU path" % t.device)
    try:
        code = _codes()[t.dtype]
    except KeyError:
        raise native.KernelError("no kernel for dtype %s (float32 and bfloat16 only)" % t.dtype) from None
    if t.dim() > 4 or t.dim() < 1 or t.stride(-1) != 1:
        raise native.KernelError("tensors must have 1 to 4 dimensions and unit inner stride, got shape %s strides %s"
                          % (tuple(t.shape), t.stride()))
    if t.dim() > 2 and not t.is_contiguous():
        raise native.KernelError("tensors of more than two dimensions must be contiguous")
    d = native.Tensor()
    d.data, d.dtype, d.ndim = t.data_ptr(), code, t.dim()
    for i, s in enumerate(t.shape):
        d.shape[i] = s
    d.ld = t.stride(0) if t.dim() == 2 else t.shape[-1]
    return d


def _p(t):
    return None if t is None else c_void_p(t.data_ptr())


def _ref(struct):
    return None if struct is None else byref(struct)


_ROW_CODES = None


def _row_codes():
    """dtypes of rows -> the kernels' numbers for them"""
    global _ROW_CODES
    if _ROW_CODES is None:
        import torch
        _ROW_CODES = {torch.float32: 0, torch.bfloat16: 1}
    return _ROW_CODES


def _current_stream(device):
    global _current_stream
    import torch
    _current_stream = torch._C._cuda_getCurrentRawStream
    return _current_stream(device)


@lru_cache(maxsize=256)
def _sections_of(values):
    import torch
    s = tuple(map(int, values))
    if not 1 <= len(s) <= 4 or min(s) < 0 or sum(s) < 1:
        raise ValueError
    return (c_int * len(s))(*s), len(s), sum(s), torch.int32, torch.float32


def _sections(sections):
    """(host array, number of sections, pairs in all, and the dtypes of positions and denominators)"""
    try:
        return _sections_of(tuple(sections))
    except (TypeError, ValueError):
        raise native.KernelError("1 to 4 sections (pairs per axis) with at least one pair between them are wanted, got %r" % (sections,)) from None


class DeferredNorm:
    """Rows whose RMSNorm is half done by the product that made them (friday::Rows): `scaled` holds weight (*) x
    rounded to bf16, `ssq` [parts, rows] each part's share of the rows' sums of squares."""

    def __init__(self, scaled, ssq, eps, source, weight):
        self.scaled, self.ssq, self.eps, self.source, self.weight = scaled, ssq, float(eps), source, weight
        self.shape, self.dtype, self.device = scaled.shape, scaled.dtype, scaled.device

    def materialize(self):
        return rmsnorm(self.source, self.weight, self.eps)


def materialize(h):
    return h.materialize() if isinstance(h, DeferredNorm) else h


def _rows(x):
    """(tensor, ssq or None, eps, source, weight) of plain or deferred rows."""
    if isinstance(x, DeferredNorm):
        return x.scaled, x.ssq, x.eps, x.source, x.weight
    return x, None, 0.0, None, None


def _kv(k_pool, v_pool, block_table, page_size, window=None, write=True):
    if k_pool is None:
        return None
    kv = native.KV()
    kv.k_pool, kv.v_pool = k_pool.data_ptr(), v_pool.data_ptr()
    kv.pool_pages = k_pool.shape[0]
    kv.block_table = block_table.data_ptr()
    kv.table_width = block_table.shape[1]
    kv.page_size = int(page_size)
    kv.window = int(window or 0)
    kv.n_kv_heads, kv.head_dim = k_pool.shape[-2], k_pool.shape[-1]
    kv.dtype = _codes()[k_pool.dtype]
    kv.write = 1 if write else 0
    return kv


class CudaOps:
    """The handle of the library's operations on one device."""

    name = "cuda"

    def __init__(self, device=0):
        self.device = int(device)
        self._floats_of = {}                       # attention_shared: floats of scratch by a call's sizes
        self._h = c_void_p()
        native.call("friday_ops_new", int(device), None, byref(self._h))

    def __del__(self):
        if getattr(self, "_h", None) and native is not None and native._lib is not None:      # None at interpreter exit
            native._lib.friday_ops_free(self._h)
            self._h = None

    def info(self):
        return native.call_json("friday_ops_info", self._h)

    def check_status(self):
        native.call("friday_ops_check_status", self._h)

    # -- row-wise ---------------------------------------------------------
    def embedding(self, tokens, table, out=None):
        import torch
        if out is None:
            out = torch.empty((tokens.numel(), table.shape[1]), dtype=table.dtype, device=table.device)
        native.call("friday_ops_embedding", self._h, _p(tokens), tokens.numel(), _t(table), _t(out))
        return out

    def gather_rows(self, rows, src):
        import torch
        out = torch.empty((rows.numel(), src.shape[1]), dtype=src.dtype, device=src.device)
        native.call("friday_ops_gather_rows", self._h, _p(rows), rows.numel(), _t(src), _t(out))
        return out

    def rmsnorm(self, x, weight, eps, out=None):
        import torch
        if out is None:
            out = torch.empty_like(x)
        native.call("friday_ops_rmsnorm", self._h, _t(x), _t(weight), float(eps), _t(out))
        return out

    def swiglu(self, gate_up):
        import torch
        out = torch.empty((gate_up.shape[0], gate_up.shape[1] // 2), dtype=gate_up.dtype, device=gate_up.device)
        native.call("friday_ops_swiglu", self._h, _t(gate_up), _t(out))
        return out

    def rope_kv_write(self, qkv, row_seq, row_pos, denom, rotary_dim, n_heads, n_kv_heads, head_dim, k_pool=None,
                      v_pool=None, block_table=None, page_size=0):
        kv = _kv(k_pool, v_pool, block_table, page_size)
        native.call("friday_ops_rope_kv_write", self._h, _t(qkv), _p(row_seq), _p(row_pos), _p(denom), int(rotary_dim),
                    n_heads, n_kv_heads, head_dim, _ref(kv))

    def advance(self, tokens, sampled, row_pos, kv_len, row_seq, draws=None):
        native.call("friday_ops_advance", self._h, _p(tokens), _p(sampled), _p(row_pos), _p(kv_len), _p(row_seq),
                    _p(draws), tokens.numel())

    def scale_rows(self, x, scale):
        native.call("friday_ops_scale_rows", self._h, _t(x), float(scale))
        return x

    def finish_logits(self, logits, bias=None, scale=1.0, softcap=0.0):
        native.call("friday_ops_finish_logits", self._h, _t(logits), _t(bias), float(scale), float(softcap))
        return logits

    # -- matrix products --------------------------------------------------
    def linear(self, x, weight, bias=None, residual=None, out_dtype=None, out=None):
        import torch
        xt, ssq, eps, source, nw = _rows(x)
        if out is None:
            out = torch.empty((xt.shape[0], weight.shape[0]), dtype=out_dtype or xt.dtype, device=xt.device)
        native.call("friday_ops_linear", self._h, _t(xt), _t(ssq), float(eps), _t(source), _t(nw), _t(weight), _t(bias),
                    _t(residual), _t(out))
        return out

    def _linear_tc(self, x, weight, bias, residual, out, swap=-1, bn=-1, splits=-1, act=0):
        native.call("friday_ops_linear_tc", self._h, _t(x), _t(weight), _t(bias), _t(residual), _t(out), swap, bn, splits, act)
        return out

    def _linear_simt(self, x, weight, bias, residual, out):
        native.call("friday_ops_linear_simt", self._h, _t(x), _t(weight), _t(bias), _t(residual), _t(out))
        return out

    def linear_norm(self, x, weight, norm_weight, eps, bias=None, residual=None):
        import torch
        xt, ssq, in_eps, _, _ = _rows(x)
        rows, n = xt.shape[0], weight.shape[0]
        out = torch.empty((rows, n), dtype=xt.dtype, device=xt.device)
        normed = torch.empty_like(out)
        parts = torch.empty((max(n // 16, 1), rows), dtype=torch.float32, device=xt.device)
        parts_d = _t(parts)
        deferred = c_int()
        native.call("friday_ops_linear_norm", self._h, _t(xt), _t(ssq), float(in_eps), _t(weight), _t(norm_weight),
                    float(eps), _t(bias), _t(residual), _t(out), _t(normed), parts_d, byref(deferred))
        if deferred.value:
            return out, DeferredNorm(normed, parts[:parts_d.shape[0]], eps, out, norm_weight)
        return out, normed

    def qkv_rope_write(self, x, weight, bias, row_seq, row_pos, denom, rotary_dim, n_heads, n_kv_heads, head_dim,
                       k_pool=None, v_pool=None, block_table=None, page_size=0):
        import torch
        xt, ssq, in_eps, _, _ = _rows(x)
        out = torch.empty((xt.shape[0], weight.shape[0]), dtype=xt.dtype, device=xt.device)
        kv = _kv(k_pool, v_pool, block_table, page_size)
        native.call("friday_ops_qkv_rope_write", self._h, _t(xt), _t(ssq), float(in_eps), _t(weight), _t(bias),
                    _p(row_seq), _p(row_pos), _p(denom), int(rotary_dim), n_heads, n_kv_heads, head_dim, _ref(kv), _t(out))
        return out

    def linear_swiglu(self, x, weight_pairs):
        import torch
        xt, ssq, in_eps, _, _ = _rows(x)
        out = torch.empty((xt.shape[0], weight_pairs.shape[0] // 2), dtype=xt.dtype, device=xt.device)
        native.call("friday_ops_linear_swiglu", self._h, _t(xt), _t(ssq), float(in_eps), _t(weight_pairs), _t(out))
        return out

    def tensor_core_ok(self, x, weight, out, residual=None):
        ok = c_int()
        native.call("friday_ops_tensor_core_ok", self._h, _t(x), _t(weight), _t(out), byref(ok))
        return bool(ok.value)

    def plan(self, rows, n, k):
        """(operands swapped, tile width, splits of k) that the tensor-core product chooses for a shape."""
        s, bn, sp = c_int(), c_int(), c_int()
        native.call("friday_ops_plan", self._h, rows, n, k, byref(s), byref(bn), byref(sp))
        return bool(s.value), bn.value, sp.value

    # -- attention --------------------------------------------------------
    def attention(self, q, q_stride, out, k_pool, v_pool, block_table, page_size, row_seq, row_pos, n_heads, n_kv_heads,
                  head_dim, window, scale, geometry):
        """geometry: an object with max_kv_len and, for the tensor-core kernels, n_seqs, max_q_len, decode and the
        per-sequence arrays seq_start, seq_qlen, seq_pos0 (int32, device)."""
        g = native.Geometry()
        g.rows = out.shape[0]
        g.n_seqs = int(getattr(geometry, "n_seqs", 0))
        g.max_q_len = int(getattr(geometry, "max_q_len", 0))
        g.max_kv_len = int(geometry.max_kv_len)
        g.decode = 1 if getattr(geometry, "decode", False) else 0
        g.row_seq, g.row_pos = row_seq.data_ptr(), row_pos.data_ptr()
        for name in ("seq_start", "seq_qlen", "seq_pos0"):
            t = getattr(geometry, name, None)
            setattr(g, name, None if t is None else t.data_ptr())
        kv = _kv(k_pool, v_pool, block_table, page_size, window, write=False)
        native.call("friday_ops_attention", self._h, _t(q), int(q_stride), _t(out), byref(kv), byref(g), n_heads,
                    n_kv_heads, head_dim, int(window or 0), float(scale))

    def decode_splits(self, n_seqs, n_heads, n_kv_heads, head_dim, max_kv_len):
        s = c_int()
        native.call("friday_ops_decode_splits", self._h, n_seqs, n_heads, n_kv_heads, head_dim, max_kv_len, byref(s))
        return s.value

    def attention_splits(self, rows, n_heads, max_kv_len):
        s = c_int()
        native.call("friday_ops_attention_splits", self._h, rows, n_heads, max_kv_len, byref(s))
        return s.value

    # -- a batch that shares a long prefix, positions with several axes ----
    # These run on torch's current stream; what a call needs of scratch is torch's, so that a captured graph has its own.  A step of a
    # few rows is over in the time of some thirty Python calls: every check is part of one condition, and what is wrong is looked for
    # only once that fails.
    def _rows_wrong(self, what, **tensors):
        for name, t in tensors.items():
            if t.get_device() != self.device:
                raise native.KernelError("%s: %s is on %s, these operations are cuda:%d's" % (what, name, t.device, self.device))
            if t.dtype not in _row_codes() or t.dim() != 2:
                raise native.KernelError("%s: %s must be rows of float32 or bfloat16, got %s %s" % (what, name, t.dtype, tuple(t.shape)))
            if (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
                raise native.KernelError("%s: %s needs unit inner stride and rows apart, got strides %s" % (what, name, t.stride()))

    def _numbers_wrong(self, what, **arrays):
        import torch
        for name, (t, shape) in arrays.items():
            whole = isinstance(shape, tuple)
            if (t.dtype != torch.int32 or t.get_device() != self.device or not t.is_contiguous() or (tuple(t.shape) != shape if whole else t.numel() < shape)):
                raise native.KernelError("%s: %s must be %s contiguous int32 numbers on cuda:%d, got %s %s with strides %s on %s"
                                         % (what, name, list(shape) if whole else "at least %d" % shape, self.device, t.dtype, tuple(t.shape),
                                            t.stride(), t.device))

    def _axes_wrong(self, what, rows, positions, denom, axes, pairs):
        self._numbers_wrong(what, positions=(positions, (rows, axes)))
        raise native.KernelError("%s: denom must be %d contiguous float32 numbers on cuda:%d, one per pair, got %s %s on %s"
                                 % (what, pairs, self.device, denom.dtype, tuple(denom.shape), denom.device))

    def _cache_wrong(self, what, k_pool, v_pool, block_table, shape):
        self._numbers_wrong(what, block_table=(block_table, 0))
        if block_table.dim() != 2:
            raise native.KernelError("%s: the block table is [sequences, pages], got %s" % (what, tuple(block_table.shape)))
        raise native.KernelError("%s: keys and values need pools of their own, contiguous [pages, %d, %d, %d] of float32 or bfloat16 on cuda:%d, "
                                 "got %s %s and %s %s" % ((what,) + shape + (self.device, k_pool.dtype, tuple(k_pool.shape), v_pool.dtype, tuple(v_pool.shape))))

    def rotate_axes(self, x, positions, denom, sections, heads, head_dim, interleaved=False, neighbours=False, out=None):
        """The first `heads` heads of every row of x [rows, >= heads * head_dim], turned: pair i of a head by
        positions[row][axis of i] / denom[i].  sections: pairs per axis (time, height, width; up to 4), one axis after another, or
        with `interleaved` in turn: pair i belongs to axis i mod n if i < n * sections[i mod n], else to axis 0.  A pair is
        (i, i + pairs), with `neighbours` (2i, 2i + 1); dimensions behind the pairs stay.  out [rows, heads * head_dim] may be x's own
        columns (None: a new tensor).  positions int32 [rows, axes], denom float32 [pairs], not zero.  -> out"""
        array, axes, pairs, i32, f32 = _sections(sections)
        if out is None:
            out = x.new_empty((x.shape[0], max(int(heads), 0) * max(int(head_dim), 0)))
        device, codes, shape, at, to, place = self.device, _row_codes(), x.shape, x.stride(), out.stride(), out.shape
        if not (x.get_device() == device == out.get_device() and x.dtype in codes and out.dtype is x.dtype and len(shape) == 2 == len(place)
                and (at[1] == 1 or shape[1] < 2) and (to[1] == 1 or place[1] < 2) and (shape[0] < 2 or (at[0] >= shape[1] and to[0] >= place[1]))):
            self._rows_wrong("rotate_axes", x=x, out=out)
            raise native.KernelError("rotate_axes: x and out are of one dtype, got %s and %s" % (x.dtype, out.dtype))
        rows = shape[0]
        if not (positions.dtype is i32 and positions.shape == (rows, axes) and positions.get_device() == device == denom.get_device()
                and positions.is_contiguous() and denom.dtype is f32 and denom.numel() == pairs and denom.is_contiguous()):
            self._axes_wrong("rotate_axes", rows, positions, denom, axes, pairs)
        if rows == 0:
            return out
        native.check(native.lib().friday_ops_rotate_axes(
            self._h, x.data_ptr(), rows, shape[1], at[0], out.data_ptr(), place[0], place[1], to[0], codes[x.dtype], positions.data_ptr(),
            denom.data_ptr(), array, axes, interleaved, neighbours, heads, head_dim, _current_stream(device)))
        return out

    def rope_axes_kv_write(self, qkv, row_seq, row_pos, positions, denom, sections, n_heads, n_kv_heads, head_dim, k_pool, v_pool,
                           block_table, page_size, interleaved=False, neighbours=False, q_out=None):
        """Rows [queries | keys | values] of qkv: the queries turned (see rotate_axes) into q_out [rows, n_heads * head_dim] (may be
        qkv's own query columns; None: a new tensor), keys turned and values as they are to the cache's row of (row_seq, row_pos):
        page block_table[row_seq][row_pos / page_size], row row_pos mod page_size.  Nothing else of qkv changes.  Rows whose row_seq
        is negative are left alone; a row whose place the table does not name only gets its queries.  No two rows of a call may name
        the same place.  -> q_out"""
        what = "rope_axes_kv_write"
        array, axes, pairs, i32, f32 = _sections(sections)
        if q_out is None:
            q_out = qkv.new_empty((qkv.shape[0], max(int(n_heads), 0) * max(int(head_dim), 0)))
        device, codes, shape, at, to, place = self.device, _row_codes(), qkv.shape, qkv.stride(), q_out.stride(), q_out.shape
        if not (qkv.get_device() == device == q_out.get_device() and qkv.dtype in codes and q_out.dtype is qkv.dtype and len(shape) == 2 == len(place)
                and (at[1] == 1 or shape[1] < 2) and (to[1] == 1 or place[1] < 2) and (shape[0] < 2 or (at[0] >= shape[1] and to[0] >= place[1]))):
            self._rows_wrong(what, qkv=qkv, q_out=q_out)
            raise native.KernelError("%s: qkv and q_out are of one dtype, got %s and %s" % (what, qkv.dtype, q_out.dtype))
        rows = shape[0]
        if not (positions.dtype is i32 and positions.shape == (rows, axes) and positions.get_device() == device == denom.get_device()
                and positions.is_contiguous() and denom.dtype is f32 and denom.numel() == pairs and denom.is_contiguous()):
            self._axes_wrong(what, rows, positions, denom, axes, pairs)
        if not (row_seq.dtype is i32 and row_pos.dtype is i32 and row_seq.get_device() == device == row_pos.get_device() and row_seq.is_contiguous()
                and row_pos.is_contiguous() and row_seq.numel() >= rows and row_pos.numel() >= rows):
            self._numbers_wrong(what, row_seq=(row_seq, rows), row_pos=(row_pos, rows))
        k, v, pages, table, seqs, width = self._cache(what, k_pool, v_pool, block_table, page_size, n_kv_heads, head_dim)
        if k_pool.dtype is not qkv.dtype:
            raise native.KernelError("%s: the cache's dtype differs from the rows'" % what)
        if rows == 0 or seqs == 0:
            return q_out
        if width == 0:
            raise native.KernelError("%s: the block table is empty" % what)
        native.check(native.lib().friday_ops_rope_axes_kv_write(
            self._h, qkv.data_ptr(), rows, shape[1], at[0], q_out.data_ptr() if n_heads > 0 else None, place[0], place[1], to[0], codes[qkv.dtype],
            row_seq.data_ptr(), row_pos.data_ptr(), positions.data_ptr(), denom.data_ptr(), array, axes, interleaved, neighbours, n_heads,
            n_kv_heads, head_dim, k, v, pages, page_size, table, seqs, width, _current_stream(device)))
        return q_out

    def _cache(self, what, k_pool, v_pool, block_table, page_size, n_kv_heads, head_dim):
        shape, device, dtype, k, v = k_pool.shape, self.device, k_pool.dtype, k_pool.data_ptr(), v_pool.data_ptr()
        table = block_table.shape
        if not (dtype in _row_codes() and v_pool.dtype is dtype and v_pool.shape == shape and len(shape) == 4 and shape[1:] == (page_size, n_kv_heads, head_dim)
                and shape[0] > 0 and k != v and k_pool.is_contiguous() and v_pool.is_contiguous() and k_pool.get_device() == device == v_pool.get_device()
                and _codes().get(block_table.dtype) == 2 and len(table) == 2 and block_table.is_contiguous() and block_table.get_device() == device):
            self._cache_wrong(what, k_pool, v_pool, block_table, (page_size, n_kv_heads, head_dim))
        return k, v, shape[0], block_table.data_ptr(), table[0], table[1]

    def attention_shared(self, q, q_stride, out, k_pool, v_pool, prefix_table, prefix_len, block_table, page_size, row_seq, row_pos,
                         n_heads, n_kv_heads, head_dim, window, scale, geometry):
        """attention() for sequences that all begin with the same prefix_len positions.  Their keys and values lie in the pages of
        prefix_table (int32, may be None without a prefix); block_table [sequences, pages] names each sequence's own pages, its
        position prefix_len being the first row of the first of them.  A row at position p (row_pos, prefix included) sees position j
        if p - window < j <= p (window 0 or None: every j <= p) and a table has room for it; a page that a table leaves out reads as
        zeros.  A row that sees nothing gives zeros; a row whose row_seq is negative is not written.  Values of positions that some row
        sees must be finite.

        geometry: an object with n_seqs, max_q_len, max_kv_len (prefix included) and the arrays seq_start and seq_qlen (int32,
        device): the rows of sequence s are seq_start[s] and the seq_qlen[s] - 1 after it, row_seq says so too.  max_q_len bounds
        seq_qlen; max_kv_len is a bound on the positions that only shares the work out.  prefix_len is a number of the host's: a
        captured graph keeps it."""
        what = "attention_shared"
        device, codes, shape, at, to, place = self.device, _row_codes(), q.shape, q.stride(), out.stride(), out.shape
        if not (q.get_device() == device == out.get_device() and q.dtype in codes and out.dtype is q.dtype and len(shape) == 2 == len(place)
                and (at[1] == 1 or shape[1] < 2) and (to[1] == 1 or place[1] < 2) and (shape[0] < 2 or (at[0] >= shape[1] and at[0] == q_stride))
                and (place[0] < 2 or to[0] == place[1])):
            self._rows_wrong(what, q=q, out=out)
            raise native.KernelError("%s: queries and results of one dtype, queries q_stride apart and results contiguous are wanted, got %s with strides %s, "
                                     "q_stride %s, and %s with strides %s" % (what, q.dtype, at, q_stride, out.dtype, to))
        rows, window, prefix_len = place[0], int(window or 0), int(prefix_len)
        k, v, pages, table, seqs, width = self._cache(what, k_pool, v_pool, block_table, page_size, n_kv_heads, head_dim)
        if k_pool.dtype is not q.dtype:
            raise native.KernelError("%s: the cache's dtype differs from the queries'" % what)
        n_seqs, max_q_len, max_kv_len, starts, lens = geometry.n_seqs, geometry.max_q_len, geometry.max_kv_len, geometry.seq_start, geometry.seq_qlen
        i32 = row_seq.dtype
        if not (i32 is block_table.dtype and row_pos.dtype is i32 and starts.dtype is i32 and lens.dtype is i32
                and row_seq.get_device() == row_pos.get_device() == starts.get_device() == lens.get_device() == device
                and row_seq.is_contiguous() and row_pos.is_contiguous() and starts.is_contiguous() and lens.is_contiguous()
                and row_seq.numel() >= rows and row_pos.numel() >= rows and starts.numel() >= n_seqs and lens.numel() >= n_seqs):
            self._numbers_wrong(what, row_seq=(row_seq, rows), row_pos=(row_pos, rows), seq_start=(starts, n_seqs), seq_qlen=(lens, n_seqs))
        if seqs < n_seqs:
            raise native.KernelError("%s: %d sequences, a block table of %d" % (what, n_seqs, seqs))
        prefix = None
        if prefix_len > 0:
            if prefix_table is None:
                raise native.KernelError("%s: a prefix of %d needs its pages" % (what, prefix_len))
            if not (prefix_table.dtype is i32 and prefix_table.get_device() == device and prefix_table.is_contiguous()
                    and prefix_table.numel() * page_size >= prefix_len):
                self._numbers_wrong(what, prefix_table=(prefix_table, -(-prefix_len // page_size)))
            prefix = prefix_table.data_ptr()
        if rows == 0 or n_seqs <= 0:
            return
        code = codes[q.dtype]
        floats = self._shared_floats(rows, n_seqs, max_q_len, max_kv_len, prefix_len, n_heads, n_kv_heads, head_dim, page_size, window, code)
        scratch = q.new_empty(floats * (4 // q.element_size())) if floats else None
        native.check(native.lib().friday_ops_attention_shared(
            self._h, q.data_ptr(), shape[0], shape[1], q_stride, out.data_ptr(), rows, place[1], code, k, v, pages, page_size, prefix, prefix_len,
            table, n_seqs, width, row_seq.data_ptr(), row_pos.data_ptr(), starts.data_ptr(), lens.data_ptr(), max_q_len, max_kv_len, n_heads,
            n_kv_heads, head_dim, window, scale, scratch.data_ptr() if floats else None, floats, _current_stream(device)))

    def _shared_floats(self, *sizes):
        got = self._floats_of.get(sizes)
        if got is None:
            n = c_int64()
            native.call("friday_ops_attention_shared_floats", self._h, *sizes, byref(n))
            if len(self._floats_of) >= 4096:                  # (sizes of a step: a few of them come again and again)
                self._floats_of.clear()
            got = self._floats_of[sizes] = n.value
        return got

    # -- one attention kernel's launcher, called directly with chosen arguments (tests of that kernel alone) -----
    def _test_buffers(self, device):
        import torch
        if getattr(self, "_tb", None) is None:
            self._tb = (torch.zeros((1 << 16,), dtype=torch.int32, device=device),
                        torch.zeros((4,), dtype=torch.int32, device=device))
        return self._tb

    def attention_tc(self, q, q_stride, out, k_pool, v_pool, block_table, seq_start, seq_qlen, seq_pos0, seq_live,
                     n_seqs, max_q_len, n_heads, n_kv_heads, head_dim, window, scale):
        from . import lib
        status = self._test_buffers(q.device)[1]
        lib.family("attention_tc").call(
            "attention_tc", q.data_ptr(), q_stride, q.shape[0], out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
            k_pool.shape[0], block_table.data_ptr(), block_table.shape[1], seq_start.data_ptr(), seq_qlen.data_ptr(),
            seq_pos0.data_ptr(), 0 if seq_live is None else seq_live.data_ptr(), n_seqs, max_q_len, n_heads, n_kv_heads,
            head_dim, window or 0, float(scale), status.data_ptr(), None)
        if int(status[0].item()):
            status.zero_()
            raise native.KernelError("the tcgen05 attention kernel gave up on one of its bounded waits")

    def attention_mma(self, q, q_stride, out, k_pool, v_pool, block_table, seq_start, seq_qlen, seq_pos0, seq_live,
                      n_seqs, max_q_len, n_heads, n_kv_heads, head_dim, window, scale, keys_mode, splits, geometry=None):
        import torch
        from . import lib
        rows = out.shape[0]
        counters, status = self._test_buffers(q.device)
        scratch = None
        if splits > 1:
            scratch = torch.empty((rows * n_heads * splits * (head_dim + 2),), dtype=torch.float32, device=q.device)
        lib.family("attention_mma").call(
            "attention_mma", q.data_ptr(), q_stride, out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_pool.shape[0],
            block_table.data_ptr(), block_table.shape[1], 64, seq_start.data_ptr(), seq_qlen.data_ptr(),
            seq_pos0.data_ptr(), 0 if seq_live is None else seq_live.data_ptr(), n_seqs, rows, max_q_len, n_heads,
            n_kv_heads, head_dim, window or 0, float(scale), 1 if keys_mode else 0, splits,
            0 if scratch is None else scratch.data_ptr(), counters.data_ptr(), counters.numel(), status.data_ptr(), None)

    # -- sampling ---------------------------------------------------------
    def sample(self, logits, temperature, streams, steps, seed, row_live=None, out=None):
        import torch
        if out is None:
            out = torch.empty((logits.shape[0],), dtype=torch.int32, device=logits.device)
        native.call("friday_ops_sample", self._h, _t(logits), _p(temperature), _p(streams), _p(steps),
                    int(seed) & 0xFFFFFFFFFFFFFFFF, _p(row_live), _p(out))
        return out


_backend = None


def backend():
    global _backend
    if _backend is None:
        _backend = CudaOps()
    return _backend


def fusion_enabled():
    """FRIDAY_FUSE=0 keeps norms, rotation and cache write in kernels of their own (for comparison)."""
    return backend().info()["fusion"]


def launch_count():
    return backend().info()["launches"]


def __getattr__(name):
    if name == "lib":          # direct access to the kernel libraries' C entry points, for tests of those
        import importlib
        return importlib.import_module(".lib", __name__)
    raise AttributeError(name)


def embedding(*a, **k):
    return backend().embedding(*a, **k)


def gather_rows(*a, **k):
    return backend().gather_rows(*a, **k)


def rmsnorm(*a, **k):
    return backend().rmsnorm(*a, **k)


def swiglu(*a, **k):
    return backend().swiglu(*a, **k)


def linear_swiglu(*a, **k):
    return backend().linear_swiglu(*a, **k)


def rope_kv_write(*a, **k):
    return backend().rope_kv_write(*a, **k)


def advance(*a, **k):
    return backend().advance(*a, **k)


def linear(*a, **k):
    return backend().linear(*a, **k)


def linear_norm(*a, **k):
    return backend().linear_norm(*a, **k)


def qkv_rope_write(*a, **k):
    return backend().qkv_rope_write(*a, **k)


def attention(*a, **k):
    return backend().attention(*a, **k)


def rotate_axes(*a, **k):
    return backend().rotate_axes(*a, **k)


def rope_axes_kv_write(*a, **k):
    return backend().rope_axes_kv_write(*a, **k)


def attention_shared(*a, **k):
    return backend().attention_shared(*a, **k)


def sample(*a, **k):
    return backend().sample(*a, **k)
