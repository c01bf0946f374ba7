"""A serving step over a paged compressed cache: the pages, slots and positions
of a step's tokens from the requests' lengths (`paged_plan`), the norm of each
query and key head with the position rotation (`qk_norm_rope`), keys and
values into and out of their pages (`paged_store`, `paged_load`), attention of
one new token per request (`paged_decode_attention`), and `PagedCache`, which
runs them together.

Everything is queued on the current stream of the current device, where all
tensors of a call have to be; nothing is read back to the host, so a step can
be captured into a graph.  Layouts: include/turboquant_amd.h.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Tuple

import torch

from ._lib import TQ_NORM_MAXNORM, TQ_OUTLIER_ALL, check, lib
from .cache import _DT, DEFAULT_QJL_SEED, CacheConfig, _cur_device, _stream


def _device() -> int:
    return _cur_device() if _cur_device is not None else torch.cuda.current_device()


def _refuse(t: torch.Tensor, dtype: torch.dtype, shape, what: str) -> None:
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{what} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
    if t.get_device() < 0 or t.get_device() != _device():
        raise ValueError(f"{what} must be on the current device")
    raise ValueError(f"{what} must be contiguous")


# A call's checks are most of its host time (a launch takes 3 us, a comparison
# of a tensor's attribute 0.1): one condition for a good tensor, its address
# with it, and what is wrong with a bad one found out afterwards.
def _ptr(t: torch.Tensor, dtype: torch.dtype, shape, what: str, dev: int) -> int:
    """The address of a contiguous tensor of this type and shape on the current device `dev`."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _refuse(t, dtype, shape, what)


def _addr(t: torch.Tensor, dtype: torch.dtype, what: str, dev: int) -> int:
    """The same for a tensor whose shape is right already."""
    if t.dtype is dtype and t.get_device() == dev and t.is_contiguous():
        return t.data_ptr()
    _refuse(t, dtype, t.shape, what)


def _rows(t: torch.Tensor, dtype: torch.dtype, shape, what: str, dev: int) -> Tuple[int, int]:
    """Address and row stride (elements) of t [tokens, heads, head_dim], heads adjacent, likewise."""
    n, h, d = shape
    s0, s1, s2 = t.stride()
    if t.dtype is dtype and t.shape == shape and t.get_device() == dev:
        if s2 == 1 and (s1 == d or h == 1):
            return t.data_ptr(), s0 if n > 1 else h * d
        raise ValueError(f"{what}'s heads must be adjacent (strides {t.stride()} of {list(t.shape)})")
    _refuse(t, dtype, shape, what)


def _current() -> int:
    """The current device; -2 without one (no tensor is there)."""
    try:
        return _device()
    except RuntimeError:
        return -2


class PagedLayer:
    """One layer's pages: codes u8 [num_pages, num_kv_heads, page_size,
    head_dim * bits / 8] and scales int16 (f16 bits) [..., head_dim / 32] of
    keys and values; for TQ records also the keys' signs u8 [..., head_dim / 8]
    and norms int16 [num_pages, num_kv_heads, page_size].  The shapes are
    checked here, once."""

    __slots__ = ("k_idx", "k_sc", "v_idx", "v_sc", "signs", "norms", "num_pages", "num_kv_heads", "page_size",
                 "head_dim", "packed_dim", "device", "_ptrs", "_sketch")

    def __init__(self, k_idx: torch.Tensor, k_sc: torch.Tensor, v_idx: torch.Tensor, v_sc: torch.Tensor,
                 signs: Optional[torch.Tensor] = None, norms: Optional[torch.Tensor] = None):
        if k_idx.dim() != 4 or k_sc.dim() != 4:
            raise ValueError("pools must be [num_pages, num_kv_heads, page_size, bytes or blocks]")
        base = k_idx.shape[:3]
        self.num_pages, self.num_kv_heads, self.page_size = base
        self.packed_dim, self.head_dim = k_idx.shape[3], 32 * k_sc.shape[3]
        self.k_idx, self.k_sc, self.v_idx, self.v_sc, self.signs, self.norms = k_idx, k_sc, v_idx, v_sc, signs, norms
        idx, sc = (*base, self.packed_dim), (*base, self.head_dim // 32)
        self.device = dev = _current()
        self._ptrs = (_ptr(k_idx, torch.uint8, idx, "k_idx", dev), _ptr(k_sc, torch.int16, sc, "k_sc", dev),
                      _ptr(v_idx, torch.uint8, idx, "v_idx", dev), _ptr(v_sc, torch.int16, sc, "v_sc", dev))
        self._sketch = (None, None)
        if (signs is None) != (norms is None):
            raise ValueError("signs and norms come together")
        if signs is not None:
            self._sketch = (_ptr(signs, torch.uint8, (*base, self.head_dim // 8), "signs", dev),
                            _ptr(norms, torch.int16, base, "norms", dev))

    @staticmethod
    def empty(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, bits: int, qjl: bool = False,
              device="cuda") -> "PagedLayer":
        """Zeroed pages."""
        base = (num_pages, num_kv_heads, page_size)

        def make(width, dtype):
            return torch.zeros((*base, width), dtype=dtype, device=device)

        pools = [make(w, t) for _ in range(2) for w, t in ((head_dim * bits // 8, torch.uint8),
                                                           (head_dim // 32, torch.int16))]
        sketch = (make(head_dim // 8, torch.uint8), torch.zeros(base, dtype=torch.int16, device=device)) if qjl else ()
        return PagedLayer(*pools, *sketch)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_idx, self.k_sc, self.v_idx, self.v_sc, self.signs,
                                                          self.norms) if t is not None)

    def _check(self, bits: int, sign_matrix: Optional[torch.Tensor], dev: int):
        """(signs, norms, sign matrix) addresses of a call; a sign matrix selects TQ."""
        if self.device != dev:
            raise ValueError("the layer's pages must be on the current device")
        if 8 * self.packed_dim != self.head_dim * bits:
            raise ValueError(f"the layer holds records of {self.packed_dim} bytes, not {bits}-bit ones of head_dim "
                             f"{self.head_dim}")
        if sign_matrix is None:
            return None, None, None
        if self.signs is None:
            raise ValueError("a sign matrix needs pages with signs and norms")
        words = self.head_dim * self.head_dim // 32
        return (*self._sketch, _ptr(sign_matrix, torch.int32, (words,), "sign_matrix", dev))


class PagePlan(NamedTuple):
    """One step's tokens: slots int64 [num_tokens] and positions int32
    [num_tokens] (-1 in rows without a token), starts int32 [batch + 1] (request
    b's rows are starts[b] .. starts[b + 1] - 1), appended int32 [batch] (tokens
    that each request got: all of its own, or none where they do not fit),
    kv_lens int32 [batch] and free_count int32 [1] after the step."""
    slots: torch.Tensor
    positions: torch.Tensor
    starts: torch.Tensor
    appended: torch.Tensor
    kv_lens: torch.Tensor
    free_count: torch.Tensor


def paged_plan(kv_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
               free_count: torch.Tensor, page_size: int, num_tokens: int, kv_lens_out: Optional[torch.Tensor] = None,
               free_count_out: Optional[torch.Tensor] = None) -> PagePlan:
    """Pages, slots and positions of one step's tokens from the requests'
    lengths.  kv_lens, new_lens int32 [batch] (new_lens < 0: the request is done
    and its pages go back), block_table int32 [batch, width] and free_pages
    int32 [capacity] (written), free_count int32 [1].  kv_lens_out and
    free_count_out may be the inputs; new tensors by default."""
    lens, table, pages, i32, dev = kv_lens.shape, block_table.shape, free_pages.shape, torch.int32, _current()
    if len(lens) != 1 or len(table) != 2 or len(pages) != 1 or table[0] != lens[0]:
        raise ValueError("kv_lens [batch], block_table [batch, width] and free_pages [capacity] are expected")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    b = lens[0]
    ins = (_addr(kv_lens, i32, "kv_lens", dev), _ptr(new_lens, i32, lens, "new_lens", dev), b,
           _addr(block_table, i32, "block_table", dev), table[1], _addr(free_pages, i32, "free_pages", dev), pages[0],
           _ptr(free_count, i32, (1,), "free_count", dev))
    slots = kv_lens.new_empty(num_tokens, dtype=torch.int64)
    rows = kv_lens.new_empty(num_tokens + 2 * b + 1)
    first = rows.data_ptr()
    positions, starts, appended = rows.split((num_tokens, b + 1, b))
    if kv_lens_out is None:
        kv_lens_out = torch.empty_like(kv_lens)
    if free_count_out is None:
        free_count_out = torch.empty_like(free_count)
    check(lib.tq_paged_plan(*ins, page_size, num_tokens, slots.data_ptr(), first, first + 4 * num_tokens,
                            first + 4 * (num_tokens + b + 1), _ptr(kv_lens_out, i32, lens, "kv_lens_out", dev),
                            _ptr(free_count_out, i32, (1,), "free_count_out", dev), _stream()))
    return PagePlan(slots, positions, starts, appended, kv_lens_out, free_count_out)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """RMS norm of each head (none where its weight is None), then the position
    rotation of its first 2 * len(inv_freq) elements.  q [tokens, heads,
    head_dim] and k [tokens, kv_heads, head_dim] of one type, rows at any stride
    (views of a fused projection); positions int32 [tokens], rows of negative
    ones left as they are in the outputs; inv_freq f32 [rot_dim / 2].  Returns
    (q, k) in new contiguous tensors, or `out` (which may be (q, k))."""
    qs, ks, dt = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or qs[0] != ks[0] or qs[2] != ks[2] or k.dtype is not dt or dt not in _DT:
        raise ValueError("q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] of one type (f32/bf16/f16) "
                         "are expected")
    (t, h, d), hk, dev = qs, ks[1], _current()
    qp, q0 = _rows(q, dt, qs, "q", dev)
    kp, k0 = _rows(k, dt, ks, "k", dev)
    if out is None:
        qo, ko = q.new_empty(qs), k.new_empty(ks)
        qop, qo0, kop, ko0 = qo.data_ptr(), h * d, ko.data_ptr(), hk * d
    else:
        qo, ko = out
        qop, qo0 = _rows(qo, dt, qs, "out[0]", dev)
        kop, ko0 = _rows(ko, dt, ks, "out[1]", dev)
    half = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if half < 0:
        raise ValueError("inv_freq must be [rot_dim / 2]")
    wq = None if q_weight is None else _ptr(q_weight, dt, (d,), "q_weight", dev)
    wk = None if k_weight is None else _ptr(k_weight, dt, (d,), "k_weight", dev)
    check(lib.tq_qk_norm_rope(qp, q0, kp, k0, _DT[dt], _ptr(positions, torch.int32, (t,), "positions", dev), t, h, hk,
                              d, _addr(inv_freq, torch.float32, "inv_freq", dev), 2 * half,
                              1 if interleaved else 0, wq, wk, eps, qop, qo0, kop, ko0, _stream()))
    return qo, ko


def paged_store(layer: PagedLayer, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bits: int,
                outlier_blocks: int = TQ_OUTLIER_ALL, norm_mode: int = TQ_NORM_MAXNORM,
                sign_matrix: Optional[torch.Tensor] = None) -> None:
    """Quantizes k and v [tokens, num_kv_heads, head_dim] (rows at any stride)
    into the records of slots int64 [tokens]; rows whose slot is outside the
    pages are skipped, the others' slots are distinct.  sign_matrix: TQ records,
    whose keys are sketched too."""
    t, hk, d, dt, dev = slots.shape[0], layer.num_kv_heads, layer.head_dim, k.dtype, _current()
    if dt not in _DT or k.dim() != 3 or v.dim() != 3 or slots.dim() != 1:
        raise ValueError("slots [tokens], k and v [tokens, num_kv_heads, head_dim] (f32/bf16/f16) are expected")
    sg, nm, rm = layer._check(bits, sign_matrix, dev)
    shape = (t, hk, d)
    kp, k0 = _rows(k, dt, shape, "k", dev)
    vp, v0 = _rows(v, dt, shape, "v", dev)
    check(lib.tq_paged_store(kp, k0, vp, v0, _DT[dt], _addr(slots, torch.int64, "slots", dev), t, *layer._ptrs,
                             sg, nm, rm, layer.num_pages, hk, layer.page_size, d, bits, outlier_blocks, norm_mode,
                             _stream()))


def paged_load(layer: PagedLayer, slots: torch.Tensor, bits: int, outlier_blocks: int = TQ_OUTLIER_ALL,
               norm_mode: int = TQ_NORM_MAXNORM, out_dtype: torch.dtype = torch.float32,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """The records of slots int64 [tokens] as activations: (k, v) [tokens,
    num_kv_heads, head_dim] in out_dtype, or into `out`; rows whose slot is
    outside the pages are left as they are."""
    shape, dev = (slots.shape[0], layer.num_kv_heads, layer.head_dim), _current()
    if slots.dim() != 1:
        raise ValueError("slots [tokens] are expected")
    layer._check(bits, None, dev)
    if out is None:
        out = slots.new_empty(shape, dtype=out_dtype), slots.new_empty(shape, dtype=out_dtype)
    k, v = out
    dt = k.dtype
    if dt not in _DT:
        raise ValueError("out must be f32/bf16/f16")
    check(lib.tq_paged_load(*layer._ptrs, _addr(slots, torch.int64, "slots", dev), shape[0], layer.num_pages,
                            shape[1], layer.page_size, shape[2], bits, outlier_blocks, norm_mode,
                            _ptr(k, dt, shape, "out[0]", dev), _ptr(v, dt, shape, "out[1]", dev), _DT[dt], _stream()))
    return k, v


def paged_decode_attention(q: torch.Tensor, layer: PagedLayer, block_table: torch.Tensor, kv_lens: torch.Tensor,
                           bits: int, max_kv_len: int, softmax_scale: float, workspace,
                           outlier_blocks: int = TQ_OUTLIER_ALL, norm_mode: int = TQ_NORM_MAXNORM,
                           sign_matrix: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per request: q [batch, heads, head_dim] over
    the first kv_lens[b] (int32, at most max_kv_len) tokens of the pages in row
    b of block_table (int32 [batch, width]).  sign_matrix: TQ records, with the
    QJL correction of the logits.  workspace: an AttentionWorkspace of at least
    this batch, heads and max_kv_len; one call at a time uses it.  Returns
    [batch, heads, head_dim] in out_dtype (q's by default)."""
    shape, dt, dev = q.shape, q.dtype, _current()
    table = block_table.shape
    if len(shape) != 3 or shape[2] != layer.head_dim or len(table) != 2 or table[0] != shape[0]:
        raise ValueError(f"q [batch, heads, {layer.head_dim}] and block_table [batch, width] are expected")
    b, h, d = shape
    if out is None:
        out = torch.empty_like(q) if out_dtype is None or out_dtype is dt else torch.empty_like(q, dtype=out_dtype)
    elif out.shape != shape:
        raise ValueError(f"out must be {list(shape)}, got {list(out.shape)}")
    odt, ws = out.dtype, workspace.buf
    if dt not in _DT or odt not in _DT:
        raise ValueError("q and out must be f32/bf16/f16")
    sg, nm, rm = layer._check(bits, sign_matrix, dev)
    check(lib.tq_paged_decode_attention(
        _addr(q, dt, "q", dev), _DT[dt], *layer._ptrs, sg, nm, rm, _addr(block_table, torch.int32, "block_table", dev),
        table[1], _ptr(kv_lens, torch.int32, (b,), "kv_lens", dev), b, h, layer.num_kv_heads, d, bits, outlier_blocks,
        norm_mode, layer.page_size, layer.num_pages, max_kv_len, softmax_scale, _addr(out, odt, "out", dev), _DT[odt],
        _addr(ws, torch.uint8, "workspace", dev), workspace.nbytes, _stream()))
    return out


class QkNormRope(NamedTuple):
    """The norm and rotation of a layer's heads (`qk_norm_rope`)."""
    inv_freq: torch.Tensor
    q_weight: Optional[torch.Tensor] = None
    k_weight: Optional[torch.Tensor] = None
    eps: float = 1e-6
    interleaved: bool = False


class PagedCache:
    """Pages of every layer for up to max_requests requests of up to
    max_kv_len tokens, with the block table and the free list on the device.
    The layers share one table: page p of a layer holds the same tokens in all.

        plan = cache.plan(new_lens, num_tokens)          # once a step
        out = cache.step(layer, plan, q, k, v, scale, rope)   # decode, each layer

    Calls are ordered on one stream; graphs captured from them share the cache
    and its workspaces, and are replayed in order.  The first `attend` or `step`
    with a number of heads makes its workspace, outside of a capture; it stays
    for as long as the cache, which outlives its graphs."""

    def __init__(self, config: CacheConfig, num_pages: int, max_requests: int, max_kv_len: int, page_size: int = 64,
                 qjl: bool = False, device="cuda"):
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} is no power of two from 16 to 1024")
        if qjl and config.outlier_blocks != 0:
            raise ValueError("the QJL sketch needs outlier_blocks 0")
        if num_pages <= 0 or max_requests <= 0 or max_kv_len <= 0:
            raise ValueError("num_pages, max_requests and max_kv_len must be positive")
        self.config, self.page_size, self.max_requests = config, page_size, max_requests
        self.layers: List[PagedLayer] = [
            PagedLayer.empty(num_pages, page_size, config.num_kv_heads, config.head_dim, config.bits, qjl, device)
            for _ in range(config.num_layers)]
        width = -(-max_kv_len // page_size)
        self.max_kv_len = width * page_size
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(max_requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(num_pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), num_pages, dtype=torch.int32, device=device)
        self.sign_matrix = None
        if qjl:
            from . import qjl_sign_matrix
            self.sign_matrix = qjl_sign_matrix(config.head_dim, DEFAULT_QJL_SEED, device)
        self._ws = {}  # by number of heads; none is replaced, graphs hold their addresses

    def plan(self, new_lens: torch.Tensor, num_tokens: int) -> PagePlan:
        """One step's pages and slots (`paged_plan`); the cache's lengths, table
        and free list move on.  A request whose tokens would pass max_kv_len's
        pages, or find no pages, gets none of them (appended is 0)."""
        return paged_plan(self.kv_lens, new_lens, self.block_table, self.free_pages, self.free_count, self.page_size,
                          num_tokens, kv_lens_out=self.kv_lens, free_count_out=self.free_count)

    def _mode(self):
        return self.config.bits, self.config.outlier_blocks, int(self.config.norm_mode)

    def store(self, layer: int, plan: PagePlan, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's keys and values [num_tokens, num_kv_heads, head_dim] into their pages."""
        paged_store(self.layers[layer], plan.slots, k, v, *self._mode(), sign_matrix=self.sign_matrix)

    def load(self, layer: int, slots: torch.Tensor, out_dtype: torch.dtype = torch.float32):
        """Records back as activations (`paged_load`)."""
        return paged_load(self.layers[layer], slots, *self._mode(), out_dtype=out_dtype)

    def attend(self, layer: int, q: torch.Tensor, softmax_scale: float,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """q [max_requests, heads, head_dim], a row per request, over all of its tokens."""
        if q.dim() != 3 or q.shape[0] != self.max_requests:
            raise ValueError(f"q must be [{self.max_requests}, heads, head_dim]")
        ws = self._ws.get(q.shape[1])
        if ws is None:
            from . import AttentionWorkspace
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"the first call with {q.shape[1]} heads makes a workspace: call once before the "
                                   "capture")
            ws = self._ws[q.shape[1]] = AttentionWorkspace(self.max_requests, q.shape[1], self.config.num_kv_heads,
                                                           self.config.head_dim, self.max_kv_len, q.device)
        bits, outlier_blocks, norm_mode = self._mode()
        return paged_decode_attention(q, self.layers[layer], self.block_table, self.kv_lens, bits, self.max_kv_len,
                                      softmax_scale, ws, outlier_blocks, norm_mode, self.sign_matrix, out_dtype)

    def step(self, layer: int, plan: PagePlan, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             softmax_scale: float, rope: Optional[QkNormRope] = None) -> torch.Tensor:
        """A decode step of a layer: norm and rotation of q and k [num_tokens,
        heads, head_dim], the new records, and the attention of each request's
        last token: [max_requests, heads, head_dim].  Rows of requests to which
        the plan appended nothing hold nothing of use."""
        if q.dim() != 3 or q.shape[0] == 0 or q.shape[0] != plan.slots.shape[0]:
            raise ValueError(f"q must be [{plan.slots.shape[0]}, heads, head_dim], a row for each of the plan's tokens "
                             "(at least one)")
        if rope is not None:
            q, k = qk_norm_rope(q, k, plan.positions, *rope)
        self.store(layer, plan, k, v)
        rows = (plan.starts[1:] - 1).clamp_(0, q.shape[0] - 1)
        return self.attend(layer, q.index_select(0, rows), softmax_scale)

    def memory_usage(self) -> int:
        return sum(layer.nbytes() for layer in self.layers)
