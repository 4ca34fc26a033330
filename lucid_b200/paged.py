"""Paged cache of raw keys and solved values, and the operators that read and move it.

  paged_decode_step       one new token per sequence: get_new_v_prime (modeling_lucid.py:576-598),
                          the attention over the cache and the new token (:505-549), the append
  paged_decode_attention  the attention alone, over the cached tokens
  paged_append            rows of new keys / solved values into the sequences' pages
  copy_pages              whole pages copied in every layer
  PagedCache, PagedBatch  the bookkeeping: sequences, forking, freeing, compacting

A pool is [P, Hkv, page_size, D] bf16 (any strides with a unit innermost one); the block
table [B, M] int32 names the pages of each sequence in order and ``lengths`` [B] int32 the
tokens cached so far; both live on the pool's device.  A negative length marks an unused
place of the batch: zeros come out and nothing is written.  Only the rows below a
sequence's length are ever read, so pages need no clearing; an infinity or NaN among
them can make its sequence's results NaN.  What only the device can see (a page outside the
pool, a length past the block table) is not followed but reported: the next call of this
package or ``check_status()`` raises LucidError.

These operators are inference only; their outputs carry no gradient.  They can be captured
into CUDA graphs; the workspace of a captured call belongs to its graph.  A sequence's
results do not depend on timing, but their last bits may depend on what else is in the
batch: the split of the cached tokens over the GPU, and so the order of the fp32 sums, follows
all its lengths.
"""
from __future__ import annotations

import array
import contextlib
import functools
import heapq

import torch

from . import _lib
from ._lib import LucidError

__all__ = ["paged_decode_step", "paged_decode_attention", "paged_append", "copy_pages", "PagedCache", "PagedBatch"]

_NO_GUARD = contextlib.nullcontext()
_BF16, _INT32 = torch.bfloat16, torch.int32


def _raw_stream(index: int) -> int:
    """current_stream(index).cuda_stream without building a Stream."""
    return torch._C._cuda_getCurrentRawStream(index)


def _on(index: int):
    """Context in which device ``index``, which holds a tensor, is the current one."""
    return _NO_GUARD if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def _capturing() -> bool:
    try:
        return torch.cuda.is_current_stream_capturing()
    except RuntimeError:             # no usable CUDA: a cache on the CPU keeps its books
        return False


@functools.lru_cache(maxsize=1024)
def _workspace_words(index: int, B: int, Hq: int, Hkv: int, D: int, step: int) -> int:
    """Decoding workspace on device ``index`` (the current one), in 4-byte words."""
    return _lib.load().lucid_paged_decode_workspace_bytes(B, Hq, Hkv, D, step) + 3 >> 2


def _rows(t: torch.Tensor, name: str, shape, device):
    """A bf16 CUDA operand of the given shape, copied if its rows are not 8-byte aligned:
    (tensor, address, strides)."""
    s, at = t.stride(), t.data_ptr()
    if t.dtype is not _BF16 or t.shape != shape or t.device != device:
        if not t.is_cuda:
            raise RuntimeError(f"{name}: LUCID B200 kernels need CUDA tensors (no CPU fallback)")
        if t.dtype != _BF16:
            raise TypeError(f"{name}: expected bfloat16, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
        raise ValueError(f"{name} is on {t.device}, the pool on {device}")
    if s[3] == 1 and not (s[0] | s[1] | s[2] | at >> 1) & 3:
        return t, at, s
    t = t.detach().clone(memory_format=torch.contiguous_format)  # contiguous() keeps an odd start
    return t, t.data_ptr(), t.stride()


def _pools(key_pages: torch.Tensor, x_pages: torch.Tensor, dims: int = 4):
    """The pools as they are, never copied: what the kernels cannot address is refused.
    Returns (device, its index, key address and strides, value address and strides)."""
    ks, xs = key_pages.stride(), x_pages.stride()
    kp, xp = key_pages.data_ptr(), x_pages.data_ptr()
    device = key_pages.device
    low = kp >> 1 | xp >> 1
    for s in ks[:-1]:
        low |= s
    for s in xs[:-1]:
        low |= s
    if (device.type != "cuda" or key_pages.dtype is not _BF16 or x_pages.dtype is not _BF16 or len(ks) != dims
            or x_pages.shape != key_pages.shape or x_pages.device != device or ks[-1] != 1 or xs[-1] != 1 or low & 3
            or 0 in ks or 0 in xs):
        _refuse_pools(key_pages, x_pages, dims)
    return device, device.index, kp, ks, xp, xs


def _refuse_pools(key_pages, x_pages, dims) -> None:
    """Says what is wrong with the pools, if anything (a dimension of one may have stride 0)."""
    for t, name in ((key_pages, "key_pages"), (x_pages, "x_pages")):
        if not t.is_cuda:
            raise RuntimeError(f"{name}: LUCID B200 kernels need CUDA tensors (no CPU fallback)")
        if t.dtype != _BF16:
            raise TypeError(f"{name}: expected bfloat16, got {t.dtype}")
        s = t.stride()
        if len(s) != dims:
            raise ValueError(f"{name}: expected a {dims}-D pool, got shape {tuple(t.shape)}")
        if s[-1] != 1 or t.data_ptr() % 8 or any(st % 4 or st == 0 and n > 1 for st, n in zip(s[:-1], t.shape[:-1])):
            raise ValueError(f"{name}: needs a unit innermost stride, the others nonzero multiples of 4 elements, "
                             f"and an 8-byte aligned base; got strides {s}")
    if x_pages.shape != key_pages.shape or x_pages.device != key_pages.device:
        raise ValueError(f"key_pages {tuple(key_pages.shape)} on {key_pages.device} and x_pages "
                         f"{tuple(x_pages.shape)} on {x_pages.device} must match")


def _index(t: torch.Tensor, name: str, shape, device) -> int:
    """Address of an int32 table or vector on the pool's device; None in ``shape`` is any size."""
    s = t.shape
    if t.dtype is not _INT32 or t.device != device or len(s) != len(shape) or s[0] != shape[0] or t.stride(-1) != 1 and s[-1] > 1:
        if t.dtype != _INT32:
            raise TypeError(f"{name}: expected int32, got {t.dtype}")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the pool on {device}")
        if len(s) != len(shape) or s[0] != shape[0]:
            raise ValueError(f"{name}: expected shape {shape}, got {tuple(s)}")
        raise ValueError(f"{name}: needs a unit innermost stride")
    return t.data_ptr()


def _one_token(query: torch.Tensor):
    s = query.shape
    if len(s) != 4 or s[2] != 1:
        raise ValueError(f"query: expected [B, Hq, 1, D] (one new token), got {tuple(s)}")
    return s[0], s[1]


def paged_decode_step(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
                      x_pages: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scale: float,
                      eps: float = 1e-5, append: bool = True):
    """One decoding step of LucidAttention.forward (modeling_lucid.py:467-481, then :505-549)
    for one new token per sequence, in one pass over the paged cache, for any number of
    query heads per kv head.  query [B,Hq,1,D], key / value [B,Hkv,1,D], D a multiple of 4
    up to 128.  ``lengths`` counts the tokens before the step.  With ``append`` the new key
    and its solved value are also written into row lengths[b] of sequence b, whose page the
    caller has assigned (and shares with no other sequence); ``lengths`` stays as it is.
    Returns (O [B,1,Hq,D], x_new [B,Hkv,1,D])."""
    lib = _lib._lib or _lib.load()
    _lib.STATUS.poll()
    dev, index, kp, ks, xp, xs = _pools(key_pages, x_pages)
    P, Hkv, ps, D = key_pages.shape
    B, Hq = _one_token(query)
    if Hq == 0:
        raise ValueError("query: a step needs at least one query head")
    query, qp, qs = _rows(query, "query", (B, Hq, 1, D), dev)
    key, kn, kns = _rows(key, "key", (B, Hkv, 1, D), dev)
    value, vn, vns = _rows(value, "value", (B, Hkv, 1, D), dev)
    table = _index(block_table, "block_table", (B, None), dev)
    lens = _index(lengths, "lengths", (B,), dev)
    x_new = key_pages.new_empty((B, Hkv, 1, D))
    o = key_pages.new_empty((B, 1, Hq, D))
    with _on(index):
        words = _workspace_words(index, B, Hq, Hkv, D, 1)
        ws = lengths.new_empty(words)
        rc = lib.lucid_paged_decode_step(
            B, Hq, Hkv, D, P, ps, block_table.shape[1], float(scale), float(eps), qp, qs[0], qs[1], kn, kns[0], kns[1],
            vn, vns[0], vns[1], kp, ks[0], ks[1], ks[2], xp, xs[0], xs[1], xs[2], table, block_table.stride(0), lens,
            x_new.data_ptr(), Hkv * D, D, o.data_ptr(), Hq * D, D, 1 if append else 0, _lib.STATUS.device_word(index),
            ws.data_ptr(), 4 * words, _raw_stream(index))
    _lib.check(rc, "lucid_paged_decode_step")
    _lib.STATUS.settle()
    return o, x_new


def paged_decode_attention(query: torch.Tensor, key_pages: torch.Tensor, x_pages: torch.Tensor,
                           block_table: torch.Tensor, lengths: torch.Tensor, scale: float) -> torch.Tensor:
    """softmax(s q K^T) X of one new query per sequence over its ``lengths`` cached tokens
    (eager_lucid_attention_forward during decoding, the new token's row already in the
    cache).  query [B,Hq,1,D]; a sequence without tokens gives zeros.  Returns O [B,1,Hq,D]."""
    lib = _lib._lib or _lib.load()
    _lib.STATUS.poll()
    dev, index, kp, ks, xp, xs = _pools(key_pages, x_pages)
    P, Hkv, ps, D = key_pages.shape
    B, Hq = _one_token(query)
    query, qp, qs = _rows(query, "query", (B, Hq, 1, D), dev)
    table = _index(block_table, "block_table", (B, None), dev)
    lens = _index(lengths, "lengths", (B,), dev)
    o = key_pages.new_empty((B, 1, Hq, D))
    with _on(index):
        words = _workspace_words(index, B, Hq, Hkv, D, 0)
        ws = lengths.new_empty(words)
        rc = lib.lucid_paged_decode_attn(
            B, Hq, Hkv, D, P, ps, block_table.shape[1], float(scale), qp, qs[0], qs[1], kp, ks[0], ks[1], ks[2], xp, xs[0],
            xs[1], xs[2], table, block_table.stride(0), lens, o.data_ptr(), Hq * D, D, _lib.STATUS.device_word(index),
            ws.data_ptr(), 4 * words, _raw_stream(index))
    _lib.check(rc, "lucid_paged_decode_attn")
    _lib.STATUS.settle()
    return o


def paged_append(key: torch.Tensor, x: torch.Tensor, key_pages: torch.Tensor, x_pages: torch.Tensor,
                 block_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None = None) -> None:
    """Writes rows i < counts[b] (at most N; None: all N) of key and x [B,Hkv,N,D] into the rows
    lengths[b] + i of sequence b's pages, in place; rows past the counts (a padded batch)
    are not touched, nor are ``lengths``.  The caller has assigned the pages, and no two
    sequences of the call write the same one."""
    lib = _lib._lib or _lib.load()
    _lib.STATUS.poll()
    dev, index, kp, ks, xp, xs = _pools(key_pages, x_pages)
    P, Hkv, ps, D = key_pages.shape
    if key.dim() != 4:
        raise ValueError(f"key: expected [B, Hkv, N, D], got {tuple(key.shape)}")
    B, _, N, _ = key.shape
    key, kr, krs = _rows(key, "key", (B, Hkv, N, D), dev)
    x, xr, xrs = _rows(x, "x", (B, Hkv, N, D), dev)
    table = _index(block_table, "block_table", (B, None), dev)
    lens = _index(lengths, "lengths", (B,), dev)
    with _on(index):
        rc = lib.lucid_paged_append(
            B, Hkv, N, D, P, ps, block_table.shape[1], kr, krs[0], krs[1], krs[2], xr, xrs[0], xrs[1], xrs[2],
            kp, ks[0], ks[1], ks[2], xp, xs[0], xs[1], xs[2], table, block_table.stride(0), lens,
            None if counts is None else _index(counts, "counts", (B,), dev), _lib.STATUS.device_word(index),
            _raw_stream(index))
    _lib.check(rc, "lucid_paged_append")
    _lib.STATUS.settle()


def _ids(v, name: str) -> array.array:
    """Page numbers as a C int array; sequences of ints or a CPU tensor."""
    if isinstance(v, torch.Tensor):
        if v.is_cuda or v.dim() != 1 or v.is_floating_point() or v.is_complex() or v.dtype == torch.bool:
            raise TypeError(f"{name}: expected a 1-D integer CPU tensor or a sequence of page numbers")
        v = v.tolist()
    try:
        return array.array("i", v)
    except (TypeError, OverflowError) as e:
        raise TypeError(f"{name}: expected page numbers ({e})") from None


def copy_pages(key_pages: torch.Tensor, x_pages: torch.Tensor, src, dst) -> None:
    """Page dst[i] becomes a copy of page src[i], in place, in both pools: [P,Hkv,ps,D], or
    [layers,P,Hkv,ps,D] for all layers at once.  src and dst are host sequences (or CPU
    tensors) of page numbers; each dst is named once and is no src, so the order of the
    copies is free.  A page's [Hkv,ps,D] block must be dense."""
    lib = _lib._lib or _lib.load()
    _lib.STATUS.poll()
    shape = key_pages.shape
    _, index, kp, ks, xp, xs = _pools(key_pages, x_pages, 5 if len(shape) == 5 else 4)
    layers, P = (shape[0], shape[1]) if len(shape) == 5 else (1, shape[0])
    src, dst = _ids(src, "src"), _ids(dst, "dst")
    if len(src) != len(dst):
        raise ValueError(f"src names {len(src)} pages, dst {len(dst)}")
    n = shape[-3] * shape[-2] * shape[-1]
    usual = (shape[-2] * shape[-1], shape[-1], 1)
    for s, name in ((ks, "key_pages"), (xs, "x_pages")):
        if s[-3:] != usual:               # any other dense order will do
            span = 1
            for st, size in sorted((st, size) for st, size in zip(s[-3:], shape[-3:]) if size > 1):
                if st != span:
                    raise ValueError(f"{name}: the pages' [Hkv, page_size, D] blocks must be dense, got strides {s}")
                span *= size
    if len(src) == 0 or layers == 0 or n == 0:
        return
    if n % 4:
        raise ValueError(f"a page of {n} elements is not a multiple of 8 bytes")
    with _on(index):
        rc = lib.lucid_copy_pages(layers, P, 2 * n, kp, 2 * ks[0] if len(shape) == 5 else 0, 2 * ks[-4],
                                  xp, 2 * xs[0] if len(shape) == 5 else 0, 2 * xs[-4],
                                  src.buffer_info()[0], dst.buffer_info()[0], len(src), _raw_stream(index))
    if rc == 1:
        raise ValueError(f"copy_pages: pages must lie in [0, {P}), each dst named once and none of them a src")
    _lib.check(rc, "lucid_copy_pages")


class _Sequence:
    __slots__ = ("pages", "length", "edits")

    def __init__(self, pages=(), length: int = 0):
        self.pages: list[int] = list(pages)
        self.length = length
        self.edits = 0          # grows with every change of ``pages``


class PagedCache:
    """Key / solved-value cache of every layer in pages of ``page_size`` tokens, shared by
    any number of sequences: ``key_pages`` / ``x_pages`` are [layers, P, Hkv, page_size, D]
    and page p holds the same tokens in every layer.  The page lists live on the host, so
    running out of pages is an exception before anything changes; copies are queued on
    the current stream.

        cache = PagedCache(layers, kv_heads, head_dim, num_pages=4096)
        batch = cache.batch(cache.new(8))
        logits = model(ids, past_key_values=batch, prompt_lengths=lens)     # prefill
        logits = model(next_ids, past_key_values=batch)                     # one token each
        other = cache.fork(batch.sequences[0]); cache.free(batch.sequences[1]); cache.compact()
    """

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, num_pages: int, page_size: int = 64,
                 device="cuda"):
        if min(num_layers, num_kv_heads, num_pages, page_size) < 1 or not 4 <= head_dim <= 128 or head_dim % 4:
            raise ValueError("PagedCache: sizes must be positive and head_dim a multiple of 4 up to 128")
        self.page_size = page_size
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.key_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.x_pages = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self._refs = [0] * num_pages
        self._free = list(range(num_pages))   # a heap: the lowest page first
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0
        self._version = 0                     # grows when page lists change under a batch
        self._steps = 0                       # and this one when a batch's sequences grow

    @classmethod
    def for_config(cls, config, num_pages: int, page_size: int = 64, device="cuda") -> "PagedCache":
        """A cache for a decoder configuration (decoder.lucid_config)."""
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        return cls(config.num_hidden_layers, config.num_key_value_heads, head_dim, num_pages, page_size, device)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def new(self, count: int = 1) -> list[int]:
        """``count`` empty sequences; a sequence is known by its number."""
        if count < 0:
            raise ValueError(f"new: a count of {count} sequences")
        made = list(range(self._next, self._next + count))
        self._next += count
        for i in made:
            self._sequences[i] = _Sequence()
        return made

    def _get(self, sequence: int) -> _Sequence:
        try:
            return self._sequences[sequence]
        except KeyError:
            raise LucidError(f"sequence {sequence} is not in the cache") from None

    def length(self, sequence: int) -> int:
        return self._get(sequence).length

    def pages(self, sequence: int) -> list[int]:
        """The pages of the sequence's tokens, in order."""
        s = self._get(sequence)
        return s.pages[:-(-s.length // self.page_size)]

    def _drop(self, pages) -> None:
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                heapq.heappush(self._free, p)

    def _take(self) -> int:
        p = heapq.heappop(self._free)
        self._refs[p] = 1
        return p

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens, sharing the pages; a shared page that one of
        them goes on to fill is copied first (``PagedBatch.reserve``)."""
        pages = self.pages(sequence)
        child, = self.new()
        self._sequences[child] = _Sequence(pages, self._sequences[sequence].length)
        for p in pages:
            self._refs[p] += 1
        self._version += 1
        return child

    def free(self, sequence: int) -> None:
        """Ends a sequence; pages that no other one shares become free."""
        self._drop(self._get(sequence).pages)
        del self._sequences[sequence]
        self._version += 1

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool (every page at or past the number
        in use goes to a free one before it) and returns how many moved."""
        if _capturing():
            raise LucidError("PagedCache.compact works on the host: call it outside the capture")
        used = len(self._refs) - len(self._free)
        src = [p for p in range(used, len(self._refs)) if self._refs[p]]
        dst = [p for p in range(used) if not self._refs[p]]
        if not src:
            return 0
        copy_pages(self.key_pages, self.x_pages, src, dst)
        to = dict(zip(src, dst))
        for s in self._sequences.values():
            s.pages = [to.get(p, p) for p in s.pages]
            s.edits += 1
        for a, b in to.items():
            self._refs[b], self._refs[a] = self._refs[a], 0
        self._free = list(range(used, len(self._refs)))
        self._version += 1
        return len(src)

    def batch(self, sequences) -> "PagedBatch":
        return PagedBatch(self, sequences)


class PagedBatch:
    """Sequences of a PagedCache that run together: the model's ``past_key_values``.

    One model step is ``reserve(counts)``, then ``append`` or ``step`` in every layer, then
    ``advance()``; LucidForCausalLM.forward does all three.  ``block_table``, ``lengths``
    and ``counts`` are the device tensors the operators read; they are written in place, so
    a captured ``append`` or ``step`` follows them.  Replay it where the eager call would
    be, after ``reserve`` (a replay checks nothing) and before ``advance`` on one stream, and
    keep the batch as long as the graph.  A batch whose table a graph reads does not outgrow
    it: ``reserve`` refuses."""

    def __init__(self, cache: PagedCache, sequences):
        self.cache = cache
        self.sequences = list(sequences)
        if not self.sequences or len(set(self.sequences)) != len(self.sequences):
            raise ValueError("a batch is one or more different sequences")
        for s in self.sequences:
            cache._get(s)
        self._counts: list[int] | None = None   # reserved and not advanced yet
        self._version = self._steps = -1
        self._table = torch.empty(0, 0, dtype=torch.int32)   # the block table on the host
        self._edits: list[int] = []                          # and the edits it shows
        self._host_lengths: list[int] = []
        self._host_counts: list[int] = []
        self.block_table = self.lengths = self.counts = None
        self._captured = False                               # a graph reads these three

    def __len__(self) -> int:
        return len(self.sequences)

    @property
    def host_lengths(self) -> list[int]:
        return [self.cache.length(s) for s in self.sequences]

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """The longest sequence's cached tokens."""
        return max(self.host_lengths)

    def reserve(self, counts) -> None:
        """Assigns the pages for ``counts`` more tokens of each sequence (one number for
        all, or one each) and copies shared pages that would be written.  Raises LucidError,
        with nothing changed, when the pool has too few free pages or the copy fails."""
        if _capturing():
            raise LucidError("PagedBatch.reserve works on the host: call it before the capture")
        c = self.cache
        seqs = [c._get(s) for s in self.sequences]
        counts = [counts] * len(seqs) if isinstance(counts, int) else [int(n) for n in counts]
        if len(counts) != len(seqs) or min(counts) < 0:
            raise ValueError(f"reserve: {len(seqs)} sequences need as many counts, none negative; got {counts}")
        ps, dropped, shared, need = c.page_size, {}, [], 0
        for s, n in zip(seqs, counts):
            if n and s.length % ps:
                p = s.pages[s.length // ps]
                if c._refs[p] - dropped.get(p, 0) > 1:
                    dropped[p] = dropped.get(p, 0) + 1
                    shared.append(s)
                    need += 1
            need += max(0, -(-(s.length + n) // ps) - len(s.pages))
        if self._captured and self.block_table.shape[1] < max(max(len(s.pages), -(-(s.length + n) // ps))
                                                              for s, n in zip(seqs, counts)):
            raise LucidError(f"a sequence outgrows the {self.block_table.shape[1]} pages of the block table that a captured "
                             "graph reads: make a new batch of the sequences and capture again")
        if need > len(c._free):
            raise LucidError(f"the paged cache is full: {need} pages needed, {len(c._free)} of {len(c._refs)} free")
        src, dst = [s.pages[s.length // ps] for s in shared], [c._take() for _ in shared]
        if src:
            try:
                copy_pages(c.key_pages, c.x_pages, src, dst)
            except BaseException:                # an earlier call's error may surface there
                c._drop(dst)
                raise
        for s, old, new in zip(shared, src, dst):
            c._refs[old] -= 1
            s.pages[s.length // ps] = new
            s.edits += 1
        for s, n in zip(seqs, counts):
            if len(s.pages) * ps < s.length + n:
                s.pages += [c._take() for _ in range(-(-(s.length + n) // ps) - len(s.pages))]
                s.edits += 1
        self._upload(seqs, counts)
        self._counts, self._version, self._steps = counts, c._version, c._steps

    @torch.inference_mode(False)   # a tensor made in inference mode could not be written outside it
    def _upload(self, seqs, counts) -> None:
        """Brings the device tensors up to date, touching those that changed."""
        edits = [s.edits for s in seqs]
        if edits != self._edits or self.block_table is None:
            width = max(1, max(len(s.pages) for s in seqs))
            if width > self._table.shape[1]:                 # with room to grow: a page at a time is usual
                table = torch.full((len(seqs), width + width // 2 + 8), -1, dtype=torch.int32)
                self.block_table = torch.empty_like(table, device=self.cache.key_pages.device)
                self._table, self._edits = table, []
            for i, s in enumerate(seqs):
                if not self._edits or self._edits[i] != edits[i]:
                    self._table[i, :len(s.pages)] = torch.tensor(s.pages, dtype=torch.int32)
            self.block_table.copy_(self._table)
            self._edits = edits
        lengths = [s.length for s in seqs]
        if lengths != self._host_lengths:
            self.lengths = self._fill(self.lengths, lengths)
            self._host_lengths = lengths
        if counts != self._host_counts:
            self.counts = self._fill(self.counts, counts)
            self._host_counts = counts

    def _fill(self, t: torch.Tensor | None, values) -> torch.Tensor:
        host = torch.tensor(values, dtype=torch.int32)
        return host.to(self.cache.key_pages.device, copy=True) if t is None else t.copy_(host)

    def _check(self) -> None:
        if self._counts is None:
            raise LucidError("reserve() the step's tokens first")
        if self._version != self.cache._version:
            raise LucidError("the cache's pages changed since reserve(): reserve again")
        if self._steps != self.cache._steps:         # some batch has advanced: one with a sequence of this one?
            if self.host_lengths != self._host_lengths:
                raise LucidError("a sequence has grown in another batch since reserve(): reserve again")
            self._steps = self.cache._steps
        if _capturing():
            self._captured = True

    def append(self, layer: int, key: torch.Tensor, x: torch.Tensor) -> None:
        """The reserved tokens' rows of one layer, key / x [B,Hkv,N,D] with N at least the
        largest count; rows past a sequence's count are padding."""
        self._check()
        if key.shape[2] < max(self._counts):
            raise ValueError(f"append: {max(self._counts)} tokens were reserved, {key.shape[2]} rows given")
        paged_append(key, x, self.cache.key_pages[layer], self.cache.x_pages[layer], self.block_table, self.lengths,
                     self.counts)

    def step(self, layer: int, query, key, value, scale: float, eps: float = 1e-5):
        """paged_decode_step of one layer, appending; one token of every sequence reserved."""
        self._check()
        if any(n != 1 for n in self._counts):
            raise ValueError("step: reserve one token of every sequence")
        return paged_decode_step(query, key, value, self.cache.key_pages[layer], self.cache.x_pages[layer],
                                 self.block_table, self.lengths, scale, eps)

    def advance(self) -> None:
        """Counts the reserved tokens as cached."""
        if _capturing():
            raise LucidError("PagedBatch.advance works on the host: call it after the capture")
        self._check()
        for s, n in zip(self.sequences, self._counts):
            self.cache._sequences[s].length += n
        self.lengths.add_(self.counts)
        self._host_lengths = [a + n for a, n in zip(self._host_lengths, self._counts)]
        self._counts = None
        self.cache._steps += 1
