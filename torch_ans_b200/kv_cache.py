"""A 4-bit key/value cache of one attention layer whose pages the entropy coder stores and loads.

A serving program keeps its keys and values as 4-bit codes in pages (``_C.kv4_append``), answers from them
(``_C.kv4_attend``: one token, drafted tokens or whole prompts for each sequence), and moves a sequence that
is not at work -- a shared prefix, a paused conversation -- out of the cache as a byte string: its codes are
symbols of the rANS coder (``_C.kv4_to_symbols``), one stream for each page, side and head, with one table of
16 frequencies for each side and head (or channel).  Loading it back gives the same codes, so the same answers.

The reference codes tensors of symbols and has no counterpart to this module; the coder underneath is the
reference's format (``rans64_push`` / ``rans64_pop`` and the container of ``merge_bytes``).

    cache = PagedKVCache4(num_pages=1024, kv_heads=8, head_dim=128)
    step = cache.reserve([7], [len(prompt)])                 # sequence 7 gets room for its prompt
    q = cache.append(step, k, v, q=q, rotation=rotation)     # keys and queries turned to their positions
    out = cache.attend(step, q)
    step = cache.reserve([7], [1])                           # ... then token by token
    data = cache.store(7)                                    # bytes; cache.free(7) makes its pages available
    cache.load(data, 9)                                      # sequence 9 goes on where 7 was
"""
from __future__ import annotations

import struct
import zlib
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from . import _C

__all__ = ["PagedKVCache4", "Step"]

_HEADER = struct.Struct("<4sIIIIII")  # magic, length, pages, kv_heads, page_size, head_dim, tables by channel
_MAGIC = b"KV4\x02"
_MAGIC_1 = b"KV4\x01"  # the same without the checksum at the end
_CRC = struct.Struct("<I")  # of all before it
_PRECISION = 16


def _frequencies(counts: torch.Tensor) -> torch.Tensor:
    """Tables of 16 frequencies, at least 1 each, that sum to 2^16, for counts (tables, 16) in 64 bits: what is left
    of the sum when all are rounded down goes to the most frequent symbol.  (rans_pmf_to_quantized_cdf takes a
    product in 32 bits, which a symbol of half the sum or more leaves.)"""
    spare = (1 << _PRECISION) - 16
    freqs = 1 + counts * spare // counts.sum(1, keepdim=True)
    return freqs.scatter_add(1, counts.argmax(1, keepdim=True), (1 << _PRECISION) - freqs.sum(1, keepdim=True))


def _cdfs(freqs: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.pad(freqs.cumsum(1), (1, 0)).to(torch.int32)


@dataclass
class Step:
    """What the tokens that a call adds need on the device: one entry for each token (slots, positions) or
    each sequence (pages, lengths with the new tokens, starts of its queries)."""
    slots: torch.Tensor
    positions: torch.Tensor
    pages: torch.Tensor
    lengths: torch.Tensor
    q_starts: torch.Tensor
    max_queries: int


class PagedKVCache4:
    """The cache of one layer: ``codes`` and ``params`` (the arrays of ``_C.kv4_*``) and the pages of each
    sequence.  Sequences are named by the caller; pages are given out and taken back on the host."""

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 16, device=None) -> None:
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, not {head_dim}")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16, not {page_size}")
        if num_pages < 1 or kv_heads < 1:
            raise ValueError("num_pages and kv_heads must be at least 1")
        self.device = torch.device(device) if device is not None else torch.device("cuda")
        self.kv_heads, self.head_dim, self.page_size = kv_heads, head_dim, page_size
        shape = (num_pages, 2, kv_heads, page_size)
        self.codes = torch.empty(*shape, head_dim // 2, dtype=torch.uint8, device=self.device)
        self.params = torch.empty(*shape, 2, dtype=torch.bfloat16, device=self.device)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: Dict[object, List[int]] = {}
        self._length: Dict[object, int] = {}

    def length(self, sequence) -> int:
        """Tokens of a sequence (0 for one that is not in the cache)."""
        return self._length.get(sequence, 0)

    def reserve(self, sequences: Sequence, counts: Sequence[int]) -> Step:
        """Room for ``counts[i]`` more tokens of ``sequences[i]`` (each named once); new names are new
        sequences.  Raises RuntimeError, and changes nothing, when the pages do not suffice."""
        if len(sequences) != len(counts) or len(set(sequences)) != len(sequences):
            raise ValueError("each sequence is named once, with one count")
        if any(n < 0 for n in counts):
            raise ValueError("counts must not be negative")
        p = self.page_size
        more = [-(-(self.length(s) + n) // p) - len(self._pages.get(s, ())) for s, n in zip(sequences, counts)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, and {sum(more)} are needed")
        slots, positions, starts = [], [], [0]
        for s, n, m in zip(sequences, counts, more):
            pages = self._pages.setdefault(s, [])
            pages.extend(self._free.pop() for _ in range(m))
            first = self.length(s)
            positions.extend(range(first, first + n))
            slots.extend(pages[t // p] * p + t % p for t in range(first, first + n))
            starts.append(starts[-1] + n)
            self._length[s] = first + n
        width = max((len(self._pages[s]) for s in sequences), default=0)
        table = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in sequences]
        i64 = torch.tensor([slots, positions], dtype=torch.int64).to(self.device, non_blocking=True)
        i32 = torch.tensor([self._length[s] for s in sequences] + starts + [x for row in table for x in row],
                           dtype=torch.int32).to(self.device, non_blocking=True)
        n = len(sequences)
        return Step(i64[0], i64[1], i32[2 * n + 1:].view(n, width), i32[:n], i32[n: 2 * n + 1], max(counts, default=0))

    def append(self, step: Step, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
               rotation: Optional[torch.Tensor] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
        """Store the step's keys and values (tokens, kv_heads, head_dim); with ``rotation`` (positions,
        rotary_dim: cosines, then sines) keys and queries are turned to their positions.  Returns the queries."""
        return _C.kv4_append(self.codes, self.params, k, v, step.slots, q=q,
                             positions=step.positions if rotation is not None else None, rotation=rotation,
                             interleaved=interleaved)

    def attend(self, step: Step, q: torch.Tensor, scale: Optional[float] = None, causal: bool = True) -> torch.Tensor:
        """The step's queries (tokens, heads, head_dim) over their sequences, the step's own tokens included."""
        return _C.kv4_attend(q, self.codes, self.params, step.pages, step.lengths, q_starts=step.q_starts,
                             max_queries=step.max_queries, scale=scale, causal=causal)

    def gather(self, sequence, dtype: torch.dtype = torch.bfloat16):
        """(keys, values) that a sequence's rows stand for, (tokens, kv_heads, head_dim) each."""
        pages = torch.tensor(self._pages[sequence], dtype=torch.int64, device=self.device)
        t = torch.arange(self._length[sequence], device=self.device)
        return _C.kv4_gather(self.codes, self.params, pages[t // self.page_size] * self.page_size + t % self.page_size,
                             dtype)

    def free(self, sequence) -> None:
        """Give a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(sequence)))
        del self._length[sequence]

    def store(self, sequence, by_channel: bool = False) -> bytes:
        """A sequence as bytes: a header, the tables' frequencies, the rows' parameters, and the codes as the
        container of one rANS stream for each page, side and head, and a checksum of all that.  Rows of the last page after the sequence's end
        are zeros: what was in that memory stays there."""
        pages = self._pages[sequence]
        ids = torch.tensor(pages, dtype=torch.int64, device=self.device)
        head = _HEADER.pack(_MAGIC, self._length[sequence], len(pages), self.kv_heads, self.page_size, self.head_dim,
                            int(by_channel))
        if not pages:
            return head + _CRC.pack(zlib.crc32(head))
        symbols, indexes = _C.kv4_to_symbols(self.codes, ids, by_channel=by_channel)
        params = self.params[ids]
        end = self._length[sequence] - (len(pages) - 1) * self.page_size
        symbols.view(len(pages), -1, self.page_size, self.head_dim)[-1, :, end:] = 0
        params[-1, :, :, end:] = 0
        tables = 2 * self.kv_heads * (self.head_dim if by_channel else 1)
        counts = torch.bincount((indexes * 16 + symbols).flatten(), minlength=tables * 16).view(tables, 16)
        freqs = _frequencies(counts)
        cdfs = _cdfs(freqs)
        stream = _C.rans64_init_stream(symbols.shape[0], device=str(self.device))
        _C.rans64_push(stream, symbols, indexes, cdfs, *self._sizes(tables), freq_precision=_PRECISION,
                       bypass_coding=False)
        freqs = freqs.cpu().to(torch.uint16)  # 16 symbols of at least 1: under 2^16 each
        params = params.view(torch.int16).cpu()
        data = b"".join([head, freqs.numpy().tobytes(), params.numpy().tobytes(), _C.stream_to_merged_bytes(stream, 4)])
        return data + _CRC.pack(zlib.crc32(data))

    def load(self, data: bytes, sequence) -> None:
        """Bring a stored sequence back under a new name.  Raises ValueError, and changes nothing, for bytes that are not
        a whole stored sequence of this layout."""
        if sequence in self._pages:
            raise ValueError(f"sequence {sequence!r} is in the cache")
        if len(data) < _HEADER.size:
            raise ValueError("not a stored sequence")
        magic, length, n, kv_heads, page_size, head_dim, by_channel = _HEADER.unpack_from(data)
        if magic not in (_MAGIC, _MAGIC_1):
            raise ValueError("not a stored sequence")
        body = len(data) - (_CRC.size if magic == _MAGIC else 0)
        if (kv_heads, page_size, head_dim) != (self.kv_heads, self.page_size, self.head_dim) or \
                n != -(-length // page_size) or by_channel > 1:
            raise ValueError("the stored sequence is of another cache layout")
        if n > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, and {n} are needed")
        if not n:
            self._whole(data, _HEADER.size, body)
        else:
            tables, rows = 2 * kv_heads * (head_dim if by_channel else 1), n * 2 * kv_heads
            at = _HEADER.size
            sizes = (tables * 16 * 2, rows * page_size * 2 * 2)
            if body < at + sum(sizes):
                raise ValueError("the stored sequence is cut short")
            end = at + sum(sizes)
            for _ in range(rows):  # the container's records: each as long as it says, the last ends the data
                end += 4 + struct.unpack_from("<I", data, end)[0] if end + 4 <= body else body + 1
            raw = torch.frombuffer(bytearray(data), dtype=torch.uint8)
            freqs = raw[at: at + sizes[0]].view(torch.uint16).to(torch.int32).view(tables, 16)
            cdfs = _cdfs(freqs)
            if not bool((cdfs[:, -1] == 1 << _PRECISION).all()) or not bool((freqs > 0).all()):
                raise ValueError("the stored sequence's tables are not valid")
            self._whole(data, end, body)
            params = raw[at + sizes[0]: at + sum(sizes)].view(torch.int16).view(n, 2, kv_heads, page_size, 2)
            stream = _C.merged_tensor_to_stream(raw[at + sum(sizes): end].clone(), 4, device=str(self.device))
            ids = torch.tensor(self._free[-n:][::-1], dtype=torch.int64, device=self.device)
            _, indexes = _C.kv4_to_symbols(self.codes, ids, by_channel=bool(by_channel))
            before = _C.device_status(self.device.index, reset=False)
            symbols = _C.rans64_pop(stream, indexes, cdfs.to(self.device), *self._sizes(tables),
                                    freq_precision=_PRECISION, bypass_coding=False)
            if _C.device_status(self.device.index, reset=before == 0) & ~before:
                raise ValueError("the stored sequence's streams are damaged")
            _C.kv4_from_symbols(symbols, self.codes, ids)
            self.params[ids] = params.to(self.device).view(torch.bfloat16)
        self._pages[sequence] = [self._free.pop() for _ in range(n)]
        self._length[sequence] = length

    @staticmethod
    def _whole(data: bytes, end: int, body: int) -> None:
        """What the parts add up to is what is there, and the checksum (where there is one) is right."""
        if end != body:
            raise ValueError("the stored sequence is cut short")
        if body < len(data) and zlib.crc32(memoryview(data)[:body]) != _CRC.unpack_from(data, body)[0]:
            raise ValueError("the stored sequence is damaged")

    def _sizes(self, tables: int):
        full = dict(dtype=torch.int32, device=self.device)
        return torch.full((tables,), 17, **full), torch.zeros(tables, **full)
