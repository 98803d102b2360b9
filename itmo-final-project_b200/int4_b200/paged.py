"""Serving over a paged key-value cache: sequences of different lengths, bounded memory.

``decode`` runs a batch at one position over a static cache.  Here every sequence has its own length, and its keys and
values lie in fixed-size pages that a block table names:

* ``paged_kv_append``         rotary embedding of a step's (or a prompt's) tokens, keys and values into their pages;
* ``paged_decode_attention``  one query token per sequence over its pages, grouped-query, split over the length and
  joined; on request it adds up the attention weight that every cached slot receives;
* ``paged_evict``             the slots of highest accumulated weight and the most recent ones, copied into new pages;
* ``PagedKVCache``            the pages of every layer of a model with their bookkeeping, for ``decode.LlamaTP``.

The caches are views ``[pages, kv_heads, page_size, head_dim]`` of any strides that keep a row's ``head_dim`` values
together (so ``[pages, page_size, kv_heads, head_dim]`` memory transposed will do), bf16 or fp16, head_dim 64 or 128,
page_size a multiple of 8.  All indices and lengths are int32 tensors on the device: nothing here waits for the GPU,
and every call can be captured in a CUDA graph.  The functions have no backward pass.  No counterpart in the
reference, whose decode benchmark uses transformers' StaticCache (``benchmarks/eval_llama.py:121-183``).
"""
from __future__ import annotations

import functools

import torch

from . import _lib

_HALF = (torch.bfloat16, torch.float16)
_I32, _F32 = torch.int32, torch.float32
EVICT_MAX_SLOTS = 393216  # I4B_EVICT_MAX_SLOTS


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


@functools.lru_cache(maxsize=1024)
def _attention_workspace(B: int, nq: int, nkv: int, dim: int, capacity: int, weights: bool, device: int) -> int:
    """Bytes of workspace: a matter of the sizes (and of the device's SMs) alone."""
    with torch.cuda.device(device):
        return _lib.lib().i4b_paged_attention_workspace_size(B, nq, nkv, dim, capacity, weights)


def _on_gpu(device: torch.device, *tensors) -> None:
    """Every tensor on the one CUDA device."""
    if device.type != "cuda":
        raise ValueError("int4_b200 computes on the GPU only: the tensors must be CUDA tensors")
    index = device.index
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"tensors on {t.device} and {device}: one call works on one device")


def _indices(t: torch.Tensor, name: str, n: int) -> None:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} values")


def _table(t: torch.Tensor, name: str) -> None:
    if t.dtype is not _I32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be an int32 tensor [sequences, pages] with unit stride along the pages")


def _cache(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor):
    """The cache as the C ABI takes it, and (kv_heads, page_size, head_dim, sequences, pages per sequence)."""
    shape = k.shape
    if len(shape) != 4 or shape != v.shape:
        raise ValueError("k_cache and v_cache must both be [pages, kv_heads, page_size, head_dim]")
    dtype = k.dtype
    if dtype not in _HALF or v.dtype is not dtype:
        raise ValueError("k_cache and v_cache must both be bfloat16 or both float16")
    _table(table, "block_table")
    pages, heads, page, dim = shape
    if dim not in (64, 128):
        raise ValueError(f"head_dim {dim}: 64 and 128 are supported")
    if page <= 0 or page % 8:
        raise ValueError(f"page size {page}: a multiple of 8 is needed")
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if k3 != 1 or v3 != 1:
        raise ValueError("the caches' last dimension must have unit stride")
    seqs, width = table.shape
    return _lib.PAGED_CACHE.pack(k.data_ptr(), v.data_ptr(), k0, k1, k2, v0, v1, v2, table.data_ptr(), table.stride(0),
                                 pages, heads, page, dim, seqs, width, _lib.DTYPE_CODE[dtype]), heads, page, dim, seqs, width


def _accumulator(t: torch.Tensor, B: int, nkv: int, slots: int) -> None:
    shape = t.shape
    if t.dtype is not _F32 or len(shape) != 3 or shape[0] != B or shape[1] != nkv or shape[2] < slots \
            or (shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"weights must be float32 [{B}, {nkv}, at least {slots}] with unit stride along the slots")
    if (B > 1 and t.stride(0) == 0) or (nkv > 1 and t.stride(1) == 0):
        raise ValueError("weights of different sequences or kv heads must not be the same memory")


def _starts(t: torch.Tensor) -> torch.Tensor:
    """Where the rows t[b, h] begin in memory, in elements of 4 bytes, in order."""
    (B, nkv), (s0, s1) = t.shape[:2], t.stride()[:2]
    at = torch.arange(B)[:, None] * s0 + torch.arange(nkv) * s1 + t.data_ptr() // 4
    return at.flatten().sort().values


def _rows_meet(t: torch.Tensor, n: int) -> bool:
    """Whether two of the rows t[b, h, :n] have memory in common."""
    (B, nkv), (s0, s1) = t.shape[:2], t.stride()[:2]
    if (nkv == 1 or s1 >= n) and (B == 1 or s0 >= (nkv - 1) * s1 + n):
        return False
    if (B == 1 or s0 >= n) and (nkv == 1 or s1 >= (B - 1) * s0 + n):
        return False
    return B * nkv > 1 and n > 0 and int(_starts(t).diff().min()) < n


def _output_meets(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether a row of ``out`` has memory in common with any of ``t`` (of the same shape) but its own counterpart."""
    (B, nkv, n), p, q = t.shape, out.data_ptr(), t.data_ptr()
    a, b = out.stride(), t.stride()
    if p == q and (B == 1 or a[0] == b[0]) and (nkv == 1 or a[1] == b[1]):
        return False
    if B * nkv * n == 0 or p >= q + 4 * ((B - 1) * b[0] + (nkv - 1) * b[1] + n) \
            or q >= p + 4 * ((B - 1) * a[0] + (nkv - 1) * a[1] + n):
        return False
    x, y = _starts(out), _starts(t)
    return bool((torch.searchsorted(y, x + n) > torch.searchsorted(y, x - n, right=True)).any())


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy of it if not every row of the last dimension (a multiple of 64 two-byte elements) starts on a
    16-byte boundary."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t
        s = t.stride()
        if s[-1] == 1 and all(x % 8 == 0 or n <= 1 for x, n in zip(s[:-1], t.shape)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def paged_kv_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                    slots: torch.Tensor, block_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                    seqs: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary embedding of the tokens ``qkv[T, (nq + 2 nkv) * head_dim]`` (q, k and v heads in that order); keys and
    values go into the cache, the rotated queries ``[T, nq, head_dim]`` are returned.

    Token i takes its angle from row ``positions[i]`` of ``cos`` / ``sin`` ``[max_pos, head_dim]`` (the cache's dtype
    or float32) and goes to slot ``slots[i]`` of sequence ``seqs[i]`` (without ``seqs``: sequence i).  A slot or
    sequence outside ``block_table``, or a page outside the cache, writes nothing (padding); a position outside the
    tables gives a zero query and writes nothing.  Two tokens of a call must not name the same slot of a sequence."""
    c, nkv, _, dim, n_seqs, _ = _cache(k_cache, v_cache, block_table)
    dtype = k_cache.dtype
    if qkv.dim() != 2 or qkv.dtype is not dtype:
        raise ValueError("qkv must be [tokens, (nq + 2 nkv) * head_dim] of the caches' dtype")
    T, width = qkv.shape
    nq = width // dim - 2 * nkv
    if not (width % dim == 0 and nq > 0):
        raise ValueError(f"qkv rows of {width} values do not hold {nkv} key and value heads of {dim} and queries")
    angles = cos.shape
    if not (len(angles) == 2 and angles == sin.shape and angles[1] == dim and angles[0] > 0 and cos.dtype is sin.dtype
            and (cos.dtype is dtype or cos.dtype is _F32) and cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous [max_pos, head_dim], of the caches' dtype or float32")
    _indices(positions, "positions", T)
    _indices(slots, "slots", T)
    if seqs is not None:
        _indices(seqs, "seqs", T)
    else:
        if T > n_seqs:
            raise ValueError(f"{T} tokens without seqs, and a block table of {n_seqs} sequences")
    if out is None:
        out = qkv.new_empty((T, nq, dim))
    else:
        if out.shape != (T, nq, dim) or out.dtype is not dtype or not out.is_contiguous():
            raise ValueError("out must be a contiguous [tokens, nq, head_dim] of the caches' dtype")
    dev = qkv.device
    _on_gpu(dev, k_cache, v_cache, block_table, cos, sin, positions, slots, seqs, out)
    qkv = _rows16(qkv)
    with _lib.on_device(dev):
        st = _lib.lib().i4b_paged_kv_append(c, qkv.data_ptr(), qkv.stride(0), T, nq, cos.data_ptr(),
                                            sin.data_ptr(), _lib.DTYPE_CODE[cos.dtype], angles[0],
                                            positions.data_ptr(), slots.data_ptr(),
                                            None if seqs is None else seqs.data_ptr(), out.data_ptr(),
                                            _lib.stream_handle(dev))
    _lib.check(st, "paged_kv_append")
    return out


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                           lens: torch.Tensor, *, scale: float | None = None, weights: torch.Tensor | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query token per sequence, ``q[B, nq, head_dim]``, over slots ``0..lens[b]-1`` of its pages;
    query head h reads kv head ``h // (nq // nkv)``.  Returns ``[B, nq, head_dim]`` (zeros for an empty sequence).

    ``scale`` is head_dim ** -0.5 unless given.  ``weights`` (float32 ``[B, nkv, >= pages * page_size]``) is added to
    in place: slot j of a sequence gets its probability summed over the query heads of the kv head, which is what
    ``paged_evict`` selects by.  Lengths are clamped to what the block table's rows can hold.  A NaN or infinite value
    within a length makes its outputs NaN or infinite.

    The call takes workspace from torch's allocator.  With ``weights`` that holds a float32 score for every slot that the
    table can name, ``4 * B * nq * pages * page_size`` bytes whatever the lengths are (32 sequences of 32 heads and 131072
    slots: 537 MB); a captured graph keeps it."""
    c, nkv, page, dim, B, width = _cache(k_cache, v_cache, block_table)
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != dim or q.dtype is not k_cache.dtype:
        raise ValueError("q must be [sequences, nq, head_dim] of the caches' dtype")
    nq = shape[1]
    if nq <= 0 or nq % nkv:
        raise ValueError(f"{nq} query heads do not divide over {nkv} kv heads")
    _indices(lens, "lens", B)
    if weights is not None:
        _accumulator(weights, B, nkv, width * page)
        if _rows_meet(weights, width * page):
            raise ValueError("weights of different sequences or kv heads must not be the same memory")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        if out.shape != shape or out.dtype is not q.dtype or not out.is_contiguous():
            raise ValueError("out must be a contiguous [sequences, nq, head_dim] of the caches' dtype")
    dev = q.device
    _on_gpu(dev, k_cache, v_cache, block_table, lens, weights, out)
    q = _rows16(q)
    need = _attention_workspace(B, nq, nkv, dim, width * page, weights is not None, dev.index)
    # from torch's allocator each time: two captured graphs never share it, and eager streams do not either
    ws = lens.new_empty(need, dtype=torch.uint8) if need else None
    with _lib.on_device(dev):
        st = _lib.lib().i4b_paged_decode_attention(
            c, q.data_ptr(), q.stride(0), q.stride(1), nq, lens.data_ptr(), dim ** -0.5 if scale is None else scale,
            out.data_ptr(), None if weights is None else weights.data_ptr(),
            0 if weights is None else weights.stride(0), 0 if weights is None else weights.stride(1),
            None if ws is None else ws.data_ptr(), need, _lib.stream_handle(dev))
    _lib.check(st, "paged_decode_attention")
    return out


def paged_evict(weights: torch.Tensor, lens: torch.Tensor, block_table: torch.Tensor, k_cache: torch.Tensor,
                v_cache: torch.Tensor, new_table: torch.Tensor, budget: int, *, recent: int = 0,
                weights_out: torch.Tensor | None = None):
    """Keep at most ``budget`` slots of every sequence and copy their keys and values, in order, into the pages of
    ``new_table[B, >= ceil(budget / page_size)]``.

    A sequence longer than the budget keeps, for each kv head by itself, its last ``recent`` slots and the
    ``budget - recent`` of largest ``weights[B, nkv, W]`` among the others (ties: the lower slot); a shorter one keeps
    all of them.  The new pages must not be pages that this call reads.  Returns ``(new_lens[B], kept[B, nkv, budget],
    weights_out[B, nkv, W])``: the lengths afterwards, the slots kept (-1 behind the last one) and their weights (zeros
    behind the last; ``weights_out`` may be ``weights`` itself, else its rows lie apart from those of ``weights``)."""
    c, nkv, page, _, B, width = _cache(k_cache, v_cache, block_table)
    _accumulator(weights, B, nkv, width * page)
    if not (width * page <= EVICT_MAX_SLOTS):
        raise ValueError(f"{width * page} slots per sequence: eviction selects from at most {EVICT_MAX_SLOTS}")
    _indices(lens, "lens", B)
    _table(new_table, "new_table")
    if not (budget >= 1 and 0 <= recent <= budget):
        raise ValueError(f"budget {budget} and recent {recent}: 0 <= recent <= budget, budget >= 1")
    if not (new_table.shape[0] == B and new_table.shape[1] * page >= budget):
        raise ValueError(f"new_table must hold {-(-budget // page)} pages for each of {B} sequences")
    dev = weights.device
    if weights_out is None:
        weights_out = torch.empty_like(weights, memory_format=torch.contiguous_format)
    else:
        if not (weights_out.shape == weights.shape and weights_out.dtype == torch.float32
                and (weights.shape[2] <= 1 or weights_out.stride(2) == 1)):
            raise ValueError("weights_out must be float32 of the weights' shape")
        if _rows_meet(weights_out, weights.shape[2]) or _output_meets(weights_out, weights):
            raise ValueError("weights_out: rows must not be the same memory as each other or, but for `weights` itself, as "
                             "rows of weights")
    _on_gpu(dev, k_cache, v_cache, block_table, lens, new_table, weights_out)
    new_lens = torch.empty_like(lens)
    kept = lens.new_empty((B, nkv, budget))
    with _lib.on_device(dev):
        st = _lib.lib().i4b_paged_evict(c, weights.data_ptr(), weights.stride(0), weights.stride(1),
                                        weights.shape[2], lens.data_ptr(), new_table.data_ptr(), new_table.stride(0),
                                        new_table.shape[1], budget, recent, new_lens.data_ptr(), kept.data_ptr(),
                                        weights_out.data_ptr(), weights_out.stride(0), weights_out.stride(1),
                                        _lib.stream_handle(dev))
    _lib.check(st, "paged_evict")
    return new_lens, kept, weights_out


def _upload(values: list, device: torch.device) -> torch.Tensor:
    """Whole numbers as an int64 tensor on the device, behind what its stream holds already: the host does not wait (torch
    keeps the pinned copy until the transfer has run)."""
    t = torch.tensor(values, dtype=torch.int64)
    return t if device.type == "cpu" else t.pin_memory().to(device, non_blocking=True)


class PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences, of up to ``max_len`` slots each, in pages of every layer.

    ``k[layer]`` / ``v[layer]`` are ``[num_pages, kv_heads, page_size, head_dim]``; one block table serves all layers.
    ``lens`` counts a sequence's slots, ``positions`` the tokens that it has seen (its next rotary position); they
    differ once something was evicted; ``max_positions`` bounds them (the rotary tables' length).  Which pages are free is kept on the host; the tensors that the kernels read
    (``table``, ``lens``, ``positions``, ``live``) keep their addresses, so a captured step stays valid.
    ``weights`` takes ``4 * layers * max_seqs * kv_heads`` bytes per slot of ``max_len``, and a step's workspace grows with
    ``max_seqs * max_len`` too (``paged_decode_attention``), whatever ``num_pages`` is.  A prompt adds nothing to the
    weights: slots are ranked by the steps that followed, and before any step all of them weigh 0.
    The host waits for nothing: what it changes in those tensors is queued on the current stream, which has to be the one
    that the steps (or their graphs' replays) run on, or be ordered before them.  With
    ``track_weights`` every decode step adds the attention weights up in ``weights[layer]`` ``[max_seqs, kv_heads,
    slots]`` and ``evict`` can bound the sequences.  ``decode.LlamaTP.paged_cache`` builds one for a model."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, *, num_pages: int, max_seqs: int, max_len: int,
                 page_size: int = 64, dtype: torch.dtype = torch.bfloat16, device: torch.device | None = None,
                 track_weights: bool = False, max_positions: int | None = None):
        _need(dtype in _HALF, "a paged cache holds bfloat16 or float16")
        _need(head_dim in (64, 128), f"head_dim {head_dim}: 64 and 128 are supported")
        _need(page_size > 0 and page_size % 8 == 0, f"page size {page_size}: a multiple of 8 is needed")
        _need(layers > 0 and kv_heads > 0 and num_pages > 0 and 0 < max_seqs <= 4096 and max_len > 0,
              "layers, kv_heads, num_pages, max_len and max_seqs (at most 4096) must be positive")
        width = -(-max_len // page_size)
        _need(not track_weights or width * page_size <= EVICT_MAX_SLOTS,
              f"max_len {max_len}: eviction selects from at most {EVICT_MAX_SLOTS} slots")
        dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.max_len, self.max_seqs, self.max_positions = page_size, max_len, max_seqs, max_positions
        self.k = torch.empty(layers, num_pages, kv_heads, page_size, head_dim, dtype=dtype, device=dev)
        self.v = torch.empty_like(self.k)
        self.table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.positions = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.live = torch.zeros(max_seqs, dtype=torch.int32, device=dev)  # 1: takes part in decode steps
        self.weights = torch.zeros(layers, max_seqs, kv_heads, width * page_size, device=dev) if track_weights else None
        self.free_pages = list(range(num_pages - 1, -1, -1))
        self.lengths = [0] * max_seqs  # of the host: what `lens` holds
        self.seen = [0] * max_seqs     # and what `positions` holds
        self.pages: list[list[int]] = [[] for _ in range(max_seqs)]

    def _missing(self, seq: int, n: int) -> int:
        _need(0 <= seq < self.max_seqs, f"sequence {seq} of a cache for {self.max_seqs}")
        if self.lengths[seq] + n > self.max_len:
            raise _lib.Int4B200Error(f"paged cache: sequence {seq} would hold {self.lengths[seq] + n} slots of {self.max_len}")
        if self.max_positions is not None and self.seen[seq] + n > self.max_positions:
            raise _lib.Int4B200Error(f"paged cache: sequence {seq} would reach position {self.seen[seq] + n} of {self.max_positions}")
        return max(0, -(-(self.lengths[seq] + n) // self.page_size) - len(self.pages[seq]))

    def reserve(self, want: dict[int, int]) -> None:
        """Pages for ``want[seq]`` more slots of each sequence; all of them, or an error and none."""
        missing = {seq: self._missing(seq, n) for seq, n in want.items()}
        if sum(missing.values()) > len(self.free_pages):
            raise _lib.Int4B200Error(f"paged cache: {sum(missing.values())} pages wanted, {len(self.free_pages)} free")
        new = []
        for seq, m in missing.items():
            at = len(self.pages[seq])
            self.pages[seq] += [self.free_pages.pop() for _ in range(m)]
            new += [(seq, at + i, page) for i, page in enumerate(self.pages[seq][at:])]
        if new:
            rows, columns, pages = _upload(new, self.table.device).unbind(1)
            self.table.index_put_((rows, columns), pages.to(torch.int32))

    def reserve_step(self) -> None:
        """Host side of a decode step: a slot for every live sequence (before the step, or before its graph replays)."""
        live = [seq for seq in range(self.max_seqs) if self.lengths[seq] > 0]
        self.reserve({seq: 1 for seq in live})
        for seq in live:
            self.lengths[seq] += 1
            self.seen[seq] += 1

    def free(self, seq: int) -> None:
        """Forget a sequence; its pages are free again for calls that follow on the same stream."""
        _need(0 <= seq < self.max_seqs, f"sequence {seq} of a cache for {self.max_seqs}")
        self.free_pages += reversed(self.pages[seq])
        self.pages[seq], self.lengths[seq], self.seen[seq] = [], 0, 0
        self.table[seq].fill_(-1)  # (assigning a number to an element copies it from the host and waits)
        for t in (self.lens, self.positions, self.live):
            t[seq].fill_(0)
        if self.weights is not None:
            self.weights[:, seq].zero_()

    def evict(self, budget: int, recent: int = 0) -> list[int]:
        """Cut every sequence of more than ``budget`` slots to the ``recent`` last and the ones of highest accumulated
        weight (``paged_evict``, per layer and kv head); returns the sequences that were cut.  Slots that no decode step
        has attended weigh 0, and of equal weights the lower slots stay: right after a prompt, its beginning.  Needs free
        pages for the kept slots of one sequence at a time, or raises before the first is cut (a cut gives back at least
        as many as it takes)."""
        _need(self.weights is not None, "evict needs a cache with track_weights")
        _need(budget >= 1 and 0 <= recent <= budget, f"budget {budget} and recent {recent}: 0 <= recent <= budget, budget >= 1")
        cut = [seq for seq in range(self.max_seqs) if self.lengths[seq] > budget]
        need = -(-budget // self.page_size)
        for seq in cut:
            if need > len(self.free_pages):
                raise _lib.Int4B200Error(f"paged cache: eviction of sequence {seq} wants {need} pages, {len(self.free_pages)} free")
            fresh = [self.free_pages.pop() for _ in range(need)]
            new_table = _upload([fresh], self.table.device).to(torch.int32)
            row = slice(seq, seq + 1)
            for layer in range(self.k.shape[0]):
                w = self.weights[layer, row]
                paged_evict(w, self.lens[row], self.table[row], self.k[layer], self.v[layer], new_table, budget,
                            recent=recent, weights_out=w)
            self.free_pages += reversed(self.pages[seq])
            self.pages[seq], self.lengths[seq] = fresh, budget
            self.table[seq, need:].fill_(-1)
            self.table[row, :need] = new_table
            self.lens[seq].fill_(budget)
        return cut
