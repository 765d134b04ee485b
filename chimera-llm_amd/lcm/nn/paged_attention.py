"""A paged key/value cache and the attention that reads it, for ragged batches with grouped key heads.

The reference keeps one growing key / value tensor per document (lcm/nn/incremental_state.py:14-43) and attends with fairseq2's
SDPA (lcm/nn/transformer/attention.py:201-298).  These operators are for a server that holds many sequences of different
lengths: the cache of a layer is a pool of pages (`KVPages`), a batch is a list of sequences with a page table (`PagedBatch`),
and between a layer's q / k / v products and its output product stand

    q = paged_append(pages, batch, k, v, q=q, rope=rope, norm=norm)      # or head_norm_rope + paged_append
    o = paged_attention(q, pages, batch)                                   # or shared_prefix_attention

`pages` differ from layer to layer, `batch` (and `SharedPrefix`) is made once for a step and used by every layer.

All of it runs on the HIP library only (float32 and bfloat16, head widths 64 and 128) and on the current stream of the
tensors' device.  There is no derivative: a tensor of a call (inputs, pages, norm weights, rotary
tables, given outputs) that requires a gradient while gradients are recorded, or that carries a forward-mode tangent, is refused.  Index tensors
(page tables, lengths, row starts, positions) are int32 tensors on the same device which the kernels read when they run; a
captured graph can be replayed on new contents of the same tensors.  What they hold is not checked on the host (that would
wait for the GPU), but it cannot make a kernel leave its buffers: see include/lcmhip.h for what a wrong entry does.
"""

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import forward_ad

from lcm import _hip
from lcm.nn.normalization import norm_kind

_lib = _hip.lib
_NO_BACKWARD = "the paged cache operators have no backward: call them under torch.no_grad() or detach the inputs"
_MOST = 2**30                             # of positions and rows: the structs hold 32-bit numbers, and ctypes cuts what does not fit
_NO_TANGENT = "the paged cache operators have no forward-mode derivative: detach the inputs"


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _index(t: Tensor, what: str, dims: int, device: Optional[torch.device] = None) -> int:
    """Device pointer of an int32 index tensor."""
    _hip.require_gpu(t, what)
    _require(t.dtype == torch.int32 and t.dim() == dims and t.is_contiguous(), f"{what} must be a contiguous int32 tensor of {dims} dimension(s)")
    _require(device is None or t.device == device, f"{what} lives on {t.device}, not on {device}")
    return t.data_ptr()


class RotaryTable:
    """Cosines and sines of the rotation, fp32 (positions, rotary_dim / 2); `style`: "pairs" rotates the dimensions (2i, 2i + 1)
    of a head together (the pairing of fairseq2's rotary encoder), "halves" (i, i + rotary_dim / 2).  Dimensions from
    rotary_dim on stay as they are."""

    def __init__(self, cos: Tensor, sin: Tensor, style: str = "pairs") -> None:
        _hip.require_gpu(cos, "rotary table")
        _require(cos.dtype == torch.float32 and sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape
                 and cos.device == sin.device and cos.is_contiguous() and sin.is_contiguous(),
                 "cos and sin must be contiguous float32 tensors of the same shape (positions, rotary_dim / 2)")
        _require(style in _hip.ROTARY, f"unknown rotary style {style!r}: one of {sorted(_hip.ROTARY)}")
        self.cos, self.sin, self.style, self.device = cos, sin, style, cos.device
        self._c = _hip.Rotary(cos.data_ptr(), sin.data_ptr(), cos.shape[0], 2 * cos.shape[1], _hip.ROTARY[style])
        self._ref = C.byref(self._c)

    @classmethod
    def create(cls, max_positions: int, rotary_dim: int, *, theta: float = 10000.0, style: str = "pairs", device=None) -> "RotaryTable":
        """The table of angles p * theta^(-2 i / rotary_dim), computed in 64 bits; rotary_dim a multiple of 16."""
        _require(rotary_dim >= 16 and rotary_dim % 16 == 0, f"rotary_dim {rotary_dim} is not a positive multiple of 16")
        half = rotary_dim // 2
        freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq[None, :]
        return cls(angle.cos().float().to(device or "cuda"), angle.sin().float().to(device or "cuda"), style)


class HeadNorm:
    """Norm over the values of every head: `kind` is a style of lcm.nn.normalization ("rms", "standard", "fp32", "unit"); one
    weight (and, for "standard", optionally one bias) vector of head_dim for all query heads and one for all key heads."""

    def __init__(self, kind: str, q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None,
                 q_bias: Optional[Tensor] = None, k_bias: Optional[Tensor] = None, eps: float = 1e-5) -> None:
        self.kind, self.eps = kind, float(eps)
        self.tensors = (q_weight, q_bias, k_weight, k_bias)
        given = [t for t in self.tensors if t is not None]
        for t in given:
            _hip.require_gpu(t, "head norm weight")
            _require(t.dim() == 1 and t.is_contiguous() and t.shape == given[0].shape and t.dtype == given[0].dtype
                     and t.device == given[0].device, "head norm weights and biases must be alike, contiguous (head_dim,)")
        self._given = given
        self._head_dim, self._dtype, self._device = (given[0].shape[0], given[0].dtype, given[0].device) if given else (None,) * 3
        self._c = _hip.HeadNorm(*(None if t is None else t.data_ptr() for t in self.tensors), norm_kind(kind), self.eps)
        self._ref = C.byref(self._c)

    def _check(self, head_dim: int, dtype: torch.dtype, device: torch.device) -> None:
        if self._given and (self._head_dim != head_dim or self._dtype is not dtype or self._device != device):
            raise ValueError(f"head norm weights are {(self._head_dim, self._dtype, self._device)}, the heads {(head_dim, dtype, device)}")
        _grad_free(*self._given)


class KVPages:
    """The page pool of one layer: k, v (pages, key heads, page_size, head_dim), contiguous; page_size a power of two from 16 to 65536."""

    def __init__(self, k: Tensor, v: Tensor) -> None:
        _hip.require_gpu(k, "key pages")
        _require(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device and k.is_contiguous()
                 and v.is_contiguous(), "k and v must be contiguous tensors of the same shape (pages, heads, page_size, head_dim)")
        self.k, self.v = k, v
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self._c = _hip.KVPages(k.data_ptr(), v.data_ptr(), self.num_pages, self.page_size, self.num_kv_heads, self.head_dim,
                               _hip.dtype_code(k.dtype))
        self._ref = C.byref(self._c)

    @classmethod
    def create(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *, dtype=torch.bfloat16, device=None) -> "KVPages":
        """A pool of `num_pages` pages (contents undefined)."""
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device or "cuda"), torch.empty(shape, dtype=dtype, device=device or "cuda"))


class PagedBatch:
    """The sequences of one step.  Sequence b owns the rows [q_starts[b], q_starts[b + 1]) of the q / k / v tensors (q_starts None:
    row b), its newest positions; seq_lens[b] counts its positions including them, and position c lies in page
    page_table[b, c // page_size].  `max_q` is the most rows of one sequence, `max_keys` an upper bound of seq_lens (None: what
    the table can hold, at most 2^30); both choose how the work is split.  Positions from max_keys on are not there: a row of such a position is
    not stored, and no row sees one."""

    def __init__(self, page_table: Tensor, seq_lens: Tensor, q_starts: Optional[Tensor] = None, max_q: int = 1,
                 max_keys: Optional[int] = None) -> None:
        table = _index(page_table, "page_table", 2)
        self.device = page_table.device
        lens = _index(seq_lens, "seq_lens", 1, self.device)
        n = page_table.shape[0]
        _require(seq_lens.shape[0] == n, "page_table and seq_lens must have one entry for every sequence")
        starts = None
        if q_starts is not None:
            starts = _index(q_starts, "q_starts", 1, self.device)
            _require(q_starts.shape[0] == n + 1, "q_starts must have one entry more than there are sequences")
        _require(max_q >= 1, "max_q must be positive")
        _require(q_starts is not None or max_q == 1, "without q_starts every sequence has one row")
        self.page_table, self.seq_lens, self.q_starts = page_table, seq_lens, q_starts
        self.num_seqs, self.max_pages, self.max_q, self.max_keys = n, page_table.shape[1], min(int(max_q), _MOST), max_keys
        self._fields, self._refs = (table, lens, starts, n, self.max_pages, self.max_q), {}

    def _bind(self, pages: KVPages, rows: int):
        """The C struct for this page size."""
        if self.device != pages.device:
            raise ValueError(f"the batch lives on {self.device}, the pages on {pages.device}")
        if self.q_starts is None and rows != self.num_seqs:
            raise ValueError("without q_starts there is one row for every sequence")
        ref = self._refs.get(pages.page_size)
        if ref is None:
            ref = C.byref(_hip.PagedBatch(*self._fields, _reach(self.max_keys, self.max_pages, pages)))
            self._refs[pages.page_size] = ref
        return ref


class SharedPrefix:
    """Common beginnings: the sequences [group_starts[g], group_starts[g + 1]) of a batch continue the lens[g] positions of the
    pages page_table[g].  `max_keys`: an upper bound of lens (None: what the table can hold)."""

    def __init__(self, page_table: Tensor, lens: Tensor, group_starts: Tensor, max_keys: Optional[int] = None) -> None:
        table = _index(page_table, "prefix page_table", 2)
        self.device = page_table.device
        n = page_table.shape[0]
        lens_p = _index(lens, "prefix lens", 1, self.device)
        starts = _index(group_starts, "group_starts", 1, self.device)
        _require(n >= 1 and lens.shape[0] == n and group_starts.shape[0] == n + 1,
                 "a shared prefix needs one table row and length for every group and one start more")
        self.page_table, self.lens, self.group_starts = page_table, lens, group_starts
        self.max_pages, self.max_keys = page_table.shape[1], max_keys
        self._fields, self._refs = (table, lens_p, starts, n, self.max_pages), {}

    def _bind(self, pages: KVPages):
        if self.device != pages.device:
            raise ValueError(f"the prefix lives on {self.device}, the pages on {pages.device}")
        ref = self._refs.get(pages.page_size)
        if ref is None:
            ref = C.byref(_hip.SharedPrefix(*self._fields, _reach(self.max_keys, self.max_pages, pages)))
            self._refs[pages.page_size] = ref
        return ref


def _reach(max_keys: Optional[int], max_pages: int, pages: KVPages) -> int:
    reach = min(max_pages * pages.page_size, _MOST)
    if max_keys is None:
        return reach
    if not 1 <= max_keys <= reach:
        raise ValueError(f"max_keys {max_keys} is not in [1, {reach}], what the page table holds and no more than 2^30")
    return max_keys


def _grad_free(*tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(_NO_BACKWARD)
    if forward_ad._current_level >= 0:     # inside forward_ad.dual_level(); torch.no_grad() does not end it
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(_NO_TANGENT)


def _new(like: Tensor) -> Tensor:
    out = torch.empty_like(like)           # keeps the order of a permuted dense tensor's dimensions
    return out if out.is_contiguous() else torch.empty(like.shape, dtype=like.dtype, device=like.device)


def _heads(t: Tensor, what: str, dtype: torch.dtype, device: torch.device, rows: Optional[int], heads: Optional[int],
           head_dim: int) -> Tuple[int, int, int]:
    """(pointer, row stride, head stride) of a row tensor (rows, heads, head_dim) with a dense last dimension; None: any number.
    These checks stand in front of kernels of a few microseconds: they build no message before they fail."""
    shape, stride = t.shape, t.stride()
    if (len(shape) == 3 and stride[2] == 1 and shape[2] == head_dim and t.dtype is dtype and t.device == device
            and (heads is None or shape[1] == heads) and (rows is None or shape[0] == rows)):
        return t.data_ptr(), stride[0], stride[1]
    _hip.require_gpu(t, what)
    raise ValueError(f"{what} is {tuple(shape)} with strides {stride}, {t.dtype} on {t.device}; expected "
                     f"({'any' if rows is None else rows}, {'any' if heads is None else heads}, {head_dim}) with a dense last "
                     f"dimension, {dtype} on {device}")


def _call(device: torch.device, fn, *args) -> None:
    """Runs a library entry point on the current stream of `device`."""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        _hip.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _hip.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))


def _transform(rope: Optional[RotaryTable], norm: Optional[HeadNorm], positions: Optional[Tensor], like: Tensor):
    rows, _, head_dim = like.shape
    device = like.device
    if norm is not None:
        norm._check(head_dim, like.dtype, device)
    if rope is not None:
        _grad_free(rope.cos, rope.sin)
        if rope.device != device:
            raise ValueError(f"the rotary table lives on {rope.device}, not on {device}")
    pos = None
    if positions is not None:
        if positions.dtype is not torch.int32 or positions.shape != (rows,) or positions.device != device or not positions.is_contiguous():
            raise ValueError(f"positions must be a contiguous int32 tensor with one entry for every row on {device}")
        pos = positions.data_ptr()
    return None if norm is None else norm._ref, None if rope is None else rope._ref, pos


def head_norm_rope(q: Optional[Tensor], k: Optional[Tensor], *, positions: Optional[Tensor] = None, rope: Optional[RotaryTable] = None,
                   norm: Optional[HeadNorm] = None, q_out: Optional[Tensor] = None, k_out: Optional[Tensor] = None):
    """Norm of every query and key head and the position rotation behind it, in one pass: returns (q_out, k_out).

    q (rows, heads, head_dim), k (rows, key heads, head_dim), either may be None, may be slices of one stacked product.
    `positions` (rows,) int32, needed with `rope`: a row of a negative position is skipped (padding: q_out and k_out keep what
    they hold there), one beyond the table gives NaN.  q_out / k_out default to new contiguous tensors and may be q / k themselves."""
    like = q if q is not None else k
    if like is None:
        raise ValueError("head_norm_rope needs queries or keys")
    dtype, device, shape = like.dtype, like.device, like.shape
    if len(shape) != 3:
        raise ValueError("queries and keys must be (rows, heads, head_dim)")
    if not like.is_cuda:
        _hip.require_gpu(like, "heads")
    rows, _, head_dim = shape
    _grad_free(q, k, q_out, k_out)
    q_args = k_args = qo_args = ko_args = (None, 0, 0)
    q_heads = k_heads = 0
    if q is not None:
        q_args, q_heads = _heads(q, "q", dtype, device, rows, None, head_dim), shape[1]
        if q_out is None:
            q_out = _new(q)
            qo_args = q_out.data_ptr(), q_heads * head_dim, head_dim
        else:
            qo_args = _heads(q_out, "q_out", dtype, device, rows, q_heads, head_dim)
    elif q_out is not None:
        raise ValueError("q_out without q")
    if k is not None:
        k_args, k_heads = _heads(k, "k", dtype, device, rows, None, head_dim), k.shape[1]
        if k_out is None:
            k_out = _new(k)
            ko_args = k_out.data_ptr(), k_heads * head_dim, head_dim
        else:
            ko_args = _heads(k_out, "k_out", dtype, device, rows, k_heads, head_dim)
    elif k_out is not None:
        raise ValueError("k_out without k")
    if rope is not None and positions is None:
        raise ValueError("a rotation needs positions")
    norm_ref, rope_ref, pos = _transform(rope, norm, positions, like)
    if rows == 0:                          # an empty tensor has no address
        return q_out, k_out
    _call(device, _lib.lcmhip_head_norm_rope, *q_args, *k_args, *qo_args, *ko_args, rows, q_heads, k_heads, head_dim, norm_ref,
          rope_ref, pos, _hip.dtype_code(dtype))
    return q_out, k_out


def paged_append(pages: KVPages, batch: PagedBatch, k: Tensor, v: Tensor, *, q: Optional[Tensor] = None,
                 positions: Optional[Tensor] = None, rope: Optional[RotaryTable] = None, norm: Optional[HeadNorm] = None,
                 q_out: Optional[Tensor] = None) -> Optional[Tensor]:
    """Stores the rows of k (normed and rotated on the way) and v in the pages of their sequences; q, when given, goes through
    the same norm and rotation into q_out (default: a new tensor), which is returned.

    k, v (rows, key heads, head_dim), q (rows, heads, head_dim), strided.  Row t of sequence b becomes position
    seq_lens[b] - (q_starts[b + 1] - t) of the sequence and is rotated by positions[t] (int32), or by that position when
    `positions` is None.  Rows without a place (before the sequence's beginning, from the batch's max_keys on, of no sequence, or of a
    negative position) are skipped: nothing is stored, and q_out keeps what it holds there (undefined without `q_out`)."""
    _grad_free(k, v, q, q_out, pages.k, pages.v)
    dtype, device, head_dim, kv_heads = pages.dtype, pages.device, pages.head_dim, pages.num_kv_heads
    kp = _heads(k, "k", dtype, device, None, kv_heads, head_dim)
    rows = k.shape[0]
    vp = _heads(v, "v", dtype, device, rows, kv_heads, head_dim)
    qp, heads, qo = (None, 0, 0), 0, None
    if q is not None:
        qp, heads = _heads(q, "q", dtype, device, rows, None, head_dim), q.shape[1]
        if q_out is None:
            q_out = _new(q)
        else:
            _heads(q_out, "q_out", dtype, device, rows, heads, head_dim)
            _require(q_out.is_contiguous(), "q_out must be contiguous")
        qo = q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    norm_ref, rope_ref, pos = _transform(rope, norm, positions, k)
    batch_ref = batch._bind(pages, rows)
    if rows and batch.num_seqs:            # an empty tensor has no address
        _call(device, _lib.lcmhip_paged_append, pages._ref, batch_ref, *kp, *vp, *qp, qo, rows, heads, norm_ref, rope_ref, pos)
    return q_out


def _attend(q: Tensor, pages: KVPages, batch: PagedBatch, prefix: Optional[SharedPrefix], causal: bool, scale: Optional[float],
            out: Optional[Tensor]) -> Tensor:
    _grad_free(q, out, pages.k, pages.v)
    qp = _heads(q, "q", pages.dtype, pages.device, None, None, pages.head_dim)
    rows, heads, head_dim = q.shape
    if out is None:
        out = _new(q)
    else:
        _heads(out, "out", pages.dtype, pages.device, rows, heads, head_dim)
        _require(out.is_contiguous(), "out must be contiguous")
    if prefix is None:
        refs, fn, size_fn = (pages._ref, batch._bind(pages, rows)), _lib.lcmhip_paged_attention, _lib.lcmhip_paged_attention_workspace
    else:
        refs, fn, size_fn = ((pages._ref, batch._bind(pages, rows), prefix._bind(pages)), _lib.lcmhip_shared_prefix_attention,
                             _lib.lcmhip_shared_prefix_attention_workspace)
    if rows == 0 or batch.num_seqs == 0:
        return out
    need = C.c_size_t()
    _hip.check(size_fn(*refs, rows, heads, C.byref(need)))
    size = need.value
    # partial results live as long as the call's kernels: the allocator orders the memory's next use behind them
    ws = q.new_empty(size, dtype=torch.uint8) if size else None
    _call(pages.device, fn, *refs, *qp, out.data_ptr(), rows, heads, head_dim ** -0.5 if scale is None else scale, int(causal),
          None if ws is None else ws.data_ptr(), size)
    return out


def paged_attention(q: Tensor, pages: KVPages, batch: PagedBatch, *, causal: bool = True, scale: Optional[float] = None,
                    out: Optional[Tensor] = None) -> Tensor:
    """softmax(scale q K^T) V over the pages of every row's sequence: (rows, heads, head_dim), contiguous.

    With `causal` a row sees its sequence up to its own position, otherwise all seq_lens positions.  Query head h reads key head
    h // (heads // key heads).  `scale` defaults to head_dim ** -0.5 and must lie in [1e-20, 1e20].  A row that sees no position gives
    zeros; rows of no sequence keep what `out` holds there (undefined without `out`).  `out` must not overlap q."""
    return _attend(q, pages, batch, None, causal, scale, out)


def shared_prefix_attention(q: Tensor, pages: KVPages, batch: PagedBatch, prefix: SharedPrefix, *, causal: bool = True,
                            scale: Optional[float] = None, out: Optional[Tensor] = None) -> Tensor:
    """`paged_attention` for sequences that continue common prefixes: every row sees all positions of its group's prefix, then
    its own sequence as above (seq_lens and the batch's table count the sequence's own positions only).  The prefix is read once
    for all rows of a group."""
    return _attend(q, pages, batch, prefix, causal, scale, out)
