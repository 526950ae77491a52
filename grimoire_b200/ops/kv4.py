"""KV cache in 4 bits: the pages of one layer, the calls that write and read them, attention over them, the attention weight
that every cached token has drawn, and the cut of a cache to the tokens that drew the most (csrc/kernels/kv4.cu, kv4_attn.cu;
CPU tensors run the fp32 forms of ``ops.ref``).

A page record of 18 * D bytes holds 16 tokens of one kv head: 4-bit codes and one bf16 maximum per 32 elements, 4.5 bits an
element against 8.25 of the int8 pages at head_dim 128.  Like the int8 pages they are addressed through a block table
(int32 [slots][pages of a sequence], -1 where nothing is mapped).  A table entry outside the pool maps nothing: rows are not
written there and keys there do not exist.

Every call checks its arguments' types, shapes and devices on the host, works on the current stream of the tensors' device,
takes its scratch from the caching allocator (so calls on several streams and captured graphs never share any), and does not
synchronise.  Lengths, positions and tables are read on the device; values outside the table are ignored, never followed.
"""
from __future__ import annotations

import ctypes
import struct
from contextlib import nullcontext
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _native
from . import ref
from .core import PAGE, AttnGeom

HEAD_DIMS = (64, 128, 256)
MAX_GROUP = 16          # query heads of a kv head
MAX_PAGES = 1 << 20     # pages of a sequence


@dataclass(frozen=True)
class Kv4Layer:
    """4-bit K / V pages of one layer: ``data`` uint8 [P][Hkv][18 * D]; ``mass`` (optional) fp32 [P][Hkv][16], the attention
    weight drawn by every cached token."""

    data: torch.Tensor
    mass: Optional[torch.Tensor] = None

    def __post_init__(self):
        data, mass = self.data, self.mass
        if data.dim() != 3 or data.dtype != torch.uint8 or not data.is_contiguous() or data.shape[2] not in (1152, 2304, 4608):
            raise ValueError(f"4-bit KV pages: data must be a contiguous uint8 [pages][kv heads][18 * head_dim] with head_dim in {HEAD_DIMS}")
        if data.numel() == 0 or data.data_ptr() % 16:
            raise ValueError("4-bit KV pages: data must hold a page and start on a 16-byte boundary")
        if mass is not None and (mass.dtype != torch.float32 or not mass.is_contiguous() or mass.shape != (data.shape[0], data.shape[1], PAGE)
                                 or mass.device != data.device or mass.data_ptr() % 16):
            raise ValueError("4-bit KV pages: mass must be a contiguous fp32 [pages][kv heads][16] on the device of the data, on a 16-byte boundary")

    @staticmethod
    def alloc(pages: int, Hkv: int, D: int, device, mass: bool = False) -> "Kv4Layer":
        if D not in HEAD_DIMS:
            raise ValueError(f"4-bit KV pages need head_dim in {HEAD_DIMS}, got {D}")
        return Kv4Layer(torch.zeros(pages, Hkv, 18 * D, dtype=torch.uint8, device=device),
                        torch.zeros(pages, Hkv, PAGE, dtype=torch.float32, device=device) if mass else None)

    @property
    def D(self) -> int:
        return self.data.shape[2] // 18

    def copy_page(self, src: int, dst: int) -> None:
        self.data[dst].copy_(self.data[src])
        if self.mass is not None:
            self.mass[dst].copy_(self.mass[src])

    def bytes_per_token(self) -> int:
        Hkv, rec = self.data.shape[1], self.data.shape[2]
        return Hkv * rec // PAGE + (4 * Hkv if self.mass is not None else 0)


# The calls are short (a decode step makes some per layer): arguments travel as one record of 64-bit words, and tensors are
# checked with as few attribute reads as that takes.
_pack = {n: struct.Struct(f"{n}q").pack for n in (14, 15, 17, 19)}
_pack_attn = struct.Struct("21qd4q").pack
_lib = None
_INT, _BF16 = torch.int32, torch.bfloat16
_OBSERVE = {None: 0, "set": 1, "add": 2}
_NEEDS_SCRATCH = -3                # of grm_kv4_attn: nothing was launched, the keys are cut between CTAs


def _cuda():
    """The kernel library with the argument types of this module's entry points declared."""
    global _lib
    if _lib is None:
        lib = _native.cuda()
        for fn in (lib.grm_kv4_append, lib.grm_kv4_gather, lib.grm_kv4_select, lib.grm_kv4_compact, lib.grm_kv4_attn):
            fn.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
        lib.grm_kv4_attn_scratch.argtypes = [ctypes.c_int] * 8
        lib.grm_kv4_attn_scratch.restype = ctypes.c_long
        _lib = lib
    return _lib


def _check_table(table: torch.Tensor, dev: int, what: str):
    """(pointer, slots, pages of a slot, stride) of a block table."""
    if table.dtype is not _INT or table.dim() != 2 or table.get_device() != dev:
        raise ValueError(f"{what}: block_table must be int32 [slots][pages] on the cache's device")
    slots, width = table.shape
    stride = table.stride()
    if not slots or not width or (stride[1] != 1 and width > 1):
        raise ValueError(f"{what}: block_table must be non-empty with contiguous rows")
    if width > MAX_PAGES:
        raise ValueError(f"{what}: at most {MAX_PAGES} pages a sequence are served")
    return table.data_ptr(), slots, width, stride[0]


def _check_ints(t: Optional[torch.Tensor], n: int, dev: int, what: str) -> int:
    if t is None:
        return 0
    if t.dtype is not _INT or t.dim() != 1 or t.shape[0] != n or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what}: rows, positions, slots and lengths must be contiguous int32 vectors on the cache's device, an entry per row or sequence")
    return t.data_ptr()


def _check_rows(t: torch.Tensor, M: int, W: int, dev: int, name: str, what: str):
    """(pointer, row stride) of bf16 rows."""
    if t.dtype is not _BF16 or t.dim() != 2 or t.shape[0] != M or t.shape[1] != W or t.get_device() != dev:
        raise ValueError(f"{what}: {name} must be bf16 [{M}][{W}] on the cache's device")
    stride = t.stride()
    if stride[1] != 1:
        raise ValueError(f"{what}: the rows of {name} must be contiguous")
    return t.data_ptr(), stride[0]


def _apart(t: torch.Tensor) -> bool:
    """Whether no two rows of ``t`` (the last dimension, contiguous) share memory: what a call writes must have places of its own."""
    extent = t.shape[-1]
    for stride, n in sorted((st, n) for st, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        if stride < extent:
            return False
        extent += stride * (n - 1)
    return True


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _on(dev: int):
    """Makes ``dev`` the current device, where it is not already."""
    return nullcontext() if torch._C._cuda_getDevice() == dev else torch.cuda.device(dev)


def _launch(fn, words: bytes, dev: int, what: str) -> None:
    with _on(dev):
        _native.check(fn(words, _native.raw_stream(dev)), what)


# ---------------------------------------------------------------------------------------------
# write and read back
# ---------------------------------------------------------------------------------------------
def kv4_append(kv: Kv4Layer, k: torch.Tensor, v: torch.Tensor, row_pos: torch.Tensor, row_seq: torch.Tensor, block_table: torch.Tensor) -> None:
    """Quantise row m of ``k`` / ``v`` (bf16 [M][Hkv * D], after norm and RoPE) into position ``row_pos[m]`` of sequence
    slot ``row_seq[m]``; its mass starts at zero.  Rows with a negative position or slot, or whose page is not mapped, are
    skipped.  A position may come once per call.

    Per group of 32 elements ``code = round(7 x / max|x|)``, ties to even, exactly as in 64-bit arithmetic.  A group with an
    infinity or a NaN reads back as NaN."""
    data = kv.data
    P, Hkv, rec = data.shape
    D, M, dev, what = rec // 18, k.shape[0], data.get_device(), "kv4_append"
    table = _check_table(block_table, dev, what)
    kp, ks = _check_rows(k, M, Hkv * D, dev, "k", what)
    vp, vs = _check_rows(v, M, Hkv * D, dev, "v", what)
    pos, seq = _check_ints(row_pos, M, dev, what), _check_ints(row_seq, M, dev, what)
    if M == 0:
        return
    if dev < 0:
        codes, amax = ref.kv4_views(kv.data)
        for m in range(M):
            page, slot, ok = ref.kv4_place(block_table, int(row_seq[m]), row_pos[m: m + 1], kv.data.shape[0])
            if bool(ok):
                for which, x in ((0, k), (1, v)):
                    c, a = ref.quant_kv4(x[m].reshape(Hkv, D))
                    codes[page[0], :, which, slot[0]] = c[:, 0::2] | (c[:, 1::2] << 4)
                    amax[page[0], :, slot[0], which] = a
                if kv.mass is not None:
                    kv.mass[page[0], :, slot[0]] = 0
        return
    words = _pack[17](data.data_ptr(), _ptr(kv.mass), *table, P, kp, vp, ks, vs, pos, seq, M, Hkv, D, (kp | vp | 2 * ks | 2 * vs) % 8 == 0)
    _launch(_cuda().grm_kv4_append, words, dev, what)


def kv4_gather(kv: Kv4Layer, block_table: torch.Tensor, slots: Optional[torch.Tensor], lengths: Optional[torch.Tensor], out_k: torch.Tensor,
               out_v: torch.Tensor) -> None:
    """Dequantise the first ``min(lengths[i], T)`` cached tokens of sequence slot ``slots[i]`` into ``out_k[i]`` / ``out_v[i]``
    (bf16 [S][T][Hkv * D], rounded once).  ``slots`` None: sequence i is row i of the table; ``lengths`` None: all T tokens.
    Rows past a sequence's length, and those of pages that are not mapped, stay as they are."""
    data = kv.data
    P, Hkv, rec = data.shape
    D, dev, what = rec // 18, data.get_device(), "kv4_gather"
    table = _check_table(block_table, dev, what)
    for t in (out_k, out_v):
        if t.dtype is not _BF16 or t.dim() != 3 or t.shape[2] != Hkv * D or t.shape[:2] != out_k.shape[:2] or t.get_device() != dev or t.stride(2) != 1:
            raise ValueError("kv4_gather: out_k / out_v must be bf16 [sequences][tokens][kv heads * head_dim] with contiguous rows on the cache's device")
        if not (t.is_contiguous() or _apart(t)):
            raise ValueError("kv4_gather: rows of out_k / out_v must not share memory")
    S, T = out_k.shape[:2]
    seq, length = _check_ints(slots, S, dev, what), _check_ints(lengths, S, dev, what)
    if slots is None and S > table[1]:
        raise ValueError("kv4_gather: more sequences than the table has rows")
    if S > 65535:
        raise ValueError("kv4_gather: at most 65535 sequences")
    if S == 0 or T == 0:
        return
    if dev < 0:
        for i in range(S):
            n = max(0, T if lengths is None else min(T, int(lengths[i])))
            t = torch.arange(n)
            page, slot, ok = ref.kv4_place(block_table, i if slots is None else int(slots[i]), t, P)
            for out, x in zip((out_k, out_v), ref.kv4_rows(kv.data, page, slot)):
                out[i, :n][ok] = x[ok].reshape(-1, Hkv * D).to(torch.bfloat16)
        return
    kp, vp = out_k.data_ptr(), out_v.data_ptr()
    (kb, ks, _), (vb, vs, _) = out_k.stride(), out_v.stride()
    words = _pack[19](data.data_ptr(), *table, P, seq, length, kp, vp, ks, vs, kb, vb, S, T, Hkv, D, (kp | vp | 2 * (ks | vs | kb | vb)) % 16 == 0)
    _launch(_cuda().grm_kv4_gather, words, dev, what)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def length_bucket(n: int) -> int:
    """The longest length of a step, rounded up to a power of two: the host's bound that a captured step is keyed by."""
    return max(PAGE, 1 << (max(1, n) - 1).bit_length())


def kv4_attn(q: torch.Tensor, row_seq: torch.Tensor, row_pos: torch.Tensor, block_table: torch.Tensor, kv: Kv4Layer, geom: AttnGeom,
             out: torch.Tensor, max_len: int, gate: Optional[torch.Tensor] = None, block: int = 1, observe: Optional[str] = None, alone: bool = False) -> torch.Tensor:
    """Attention of M rows over the 4-bit pages: row m (bf16 [Hq * D], after norm and RoPE) of sequence slot ``row_seq[m]`` sees
    the cached positions 0 .. ``row_pos[m]``, the last ``geom.window`` of them with a window, and leaves its output (bf16,
    times sigmoid(``gate[m]``) with a gate) in ``out[m]`` (which must not overlap ``q``).  A row that sees no key (a negative position, no mapped page)
    gives zeros.

    Softmax weights, and codes times their maxima, are fp16 operands (11 bits) of products that are summed in fp32.  Hence: within
    a block, values below 2^-24 of the largest one that any of its rows sees are rounded to fewer bits (2^-36 of that one at
    worst); so are, for blocks of many rows and for the observed weight, keys below 2^-24 of the largest one of their page, whether
    a row sees that one or not.  Keys are served up to a magnitude of 2^64 (scores are held without the query's power of two and
    would overflow from 2^100 on).

    ``max_len`` is the longest row's ``row_pos + 1`` as the host knows it: it sets how the keys are split, and
    bounds the tokens that ``observe`` covers.

    ``block`` > 1: every ``block`` consecutive rows belong to one sequence (the last rows of a prompt, a verify block).
    ``alone``: cut every block's keys as a call of that block alone would (of the same ``max_len``), so that a row's output does
    not depend on the other rows of the call, to the bit.
    ``observe``: "set" or "add" the softmax weight that every token drew from the rows of its sequence in this call, summed
    over the rows and the query heads of a kv head, to ``kv.mass``; "set" covers all tokens up to the block's last position.  No page
    may belong to two of the call's sequences then: their sums would race.
    """
    data = kv.data
    P, heads, rec = data.shape
    M, Hq, D, Hkv, dev, what = q.shape[0], geom.Hq, geom.D, geom.Hkv, data.get_device(), "kv4_attn"
    table = _check_table(block_table, dev, what)
    if rec != 18 * D or heads != Hkv:
        raise ValueError(f"kv4_attn: the cache holds {heads} kv heads of {rec // 18}, the geometry says {Hkv} of {D}")
    if Hq % Hkv or not 1 <= Hq // Hkv <= MAX_GROUP:
        raise ValueError(f"kv4_attn: {Hq} query heads over {Hkv} kv heads: 1 to {MAX_GROUP} query heads a kv head are served")
    qp, qs = _check_rows(q, M, Hq * D, dev, "q", what)
    op, os_ = _check_rows(out, M, Hq * D, dev, "out", what)
    if os_ < Hq * D and M > 1:
        raise ValueError("kv4_attn: rows of out must not share memory")
    gp, gs = (0, 0) if gate is None else _check_rows(gate, M, Hq * D, dev, "gate", what)
    seq, pos = _check_ints(row_seq, M, dev, what), _check_ints(row_pos, M, dev, what)
    if block < 1 or M % block or M > 65535:
        raise ValueError(f"kv4_attn: {M} rows in blocks of {block}: a whole number of blocks and at most 65535 rows are served")
    mode = _OBSERVE.get(observe, -1)
    if mode < 0:
        raise ValueError(f"kv4_attn: observe must be None, 'set' or 'add', got {observe!r}")
    if mode and kv.mass is None:
        raise ValueError("kv4_attn: observe needs a cache with mass")
    if not 1 <= max_len <= MAX_PAGES * PAGE:
        raise ValueError(f"kv4_attn: max_len must lie in 1 .. {MAX_PAGES * PAGE}")
    if M == 0:
        return out
    if dev < 0:
        o, weights = ref.kv4_attention(q, row_seq, row_pos, block_table, kv.data, Hq, geom.scale, geom.window)
        if gate is not None:
            o = o * torch.sigmoid(gate.float())
        out.copy_(o.to(out.dtype))
        if observe is not None:
            for slot in dict.fromkeys(row_seq[::block].tolist()):
                rows = [m for m in range(M) if int(row_seq[m // block * block]) == slot]
                n = max(weights[m].shape[1] for m in rows)
                n = min(n, (max_len + PAGE - 1) // PAGE * PAGE)
                w = torch.zeros(Hkv, n)
                for m in rows:
                    x = weights[m].reshape(Hkv, Hq // Hkv, -1).sum(1)[:, :n]
                    w[:, : x.shape[1]] += x
                page, place, ok = ref.kv4_place(block_table, int(slot), torch.arange(n), kv.data.shape[0])
                old = kv.mass[page[ok], :, place[ok]] if observe == "add" else 0
                kv.mass[page[ok], :, place[ok]] = old + w[:, ok].t()
        return out
    lib = _cuda()
    head = (data.data_ptr(), _ptr(kv.mass), *table, P, qp, qs, seq, pos, gp, gs, op, os_)
    tail = (M, Hq, Hkv, D, geom.window, geom.scale, block, mode, max_len, alone)
    with _on(dev):
        stream = _native.raw_stream(dev)
        code = lib.grm_kv4_attn(_pack_attn(*head, 0, *tail), stream)
        if code == _NEEDS_SCRATCH:
            floats = lib.grm_kv4_attn_scratch(M, Hq, Hkv, D, block, max_len, mode, alone)
            scratch = torch.empty(floats, dtype=torch.float32, device=data.device)
            code = lib.grm_kv4_attn(_pack_attn(*head, scratch.data_ptr(), *tail), stream)
        _native.check(code, what)
    return out


# ---------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------
def kv4_select(kv: Kv4Layer, slots: Optional[torch.Tensor], lengths: torch.Tensor, block_table: torch.Tensor, keep: int, recent: int,
               sink: int = 0) -> torch.Tensor:
    """Which tokens stay when sequence ``slots[i]`` of ``lengths[i]`` cached tokens is cut to ``keep``: the first ``sink``, the
    last ``recent`` and, per kv head, those of the rest with the most mass (ties to the earlier token; NaN and tokens without
    a page come last).  Returns int32 [S][Hkv][keep], positions in ascending order, -1 behind the last one of a sequence
    that is not longer than ``keep``."""
    P, Hkv, _ = kv.data.shape
    S, dev, what = lengths.numel(), kv.data.get_device(), "kv4_select"
    table = _check_table(block_table, dev, what)
    seq, length = _check_ints(slots, S, dev, what), _check_ints(lengths, S, dev, what)
    if kv.mass is None:
        raise ValueError("kv4_select needs a cache with mass")
    if keep < 1 or recent < 0 or sink < 0 or recent + sink > keep:
        raise ValueError(f"kv4_select: keep {keep} >= 1, recent {recent} and sink {sink} >= 0 and recent + sink <= keep are wanted")
    if slots is None and S > table[1]:
        raise ValueError("kv4_select: more sequences than the table has rows")
    if S > 65535:
        raise ValueError("kv4_select: at most 65535 sequences")
    idx = torch.empty(S, Hkv, keep, dtype=torch.int32, device=kv.data.device)
    if S == 0:
        return idx
    if dev < 0:
        idx.fill_(-1)
        for i in range(S):
            n = max(0, min(int(lengths[i]), block_table.shape[1] * PAGE))
            t = torch.arange(n)
            page, place, ok = ref.kv4_place(block_table, i if slots is None else int(slots[i]), t, kv.data.shape[0])
            must = (t < sink) | (t >= n - recent)
            for h in range(Hkv):
                m = kv.mass[page, h, place]
                last = ~ok | torch.isnan(m)                                   # three keys, the least significant first: a stable sort each
                order = torch.sort(m.masked_fill(last, 0), descending=True, stable=True).indices
                order = order[torch.sort(last[order].int(), stable=True).indices]
                order = order[torch.sort((~must[order]).int(), stable=True).indices]
                got = order[:keep].sort().values
                idx[i, h, : got.numel()] = got.to(torch.int32)
        return idx
    words = _pack[14](kv.mass.data_ptr(), *table, P, seq, length, idx.data_ptr(), S, Hkv, keep, recent, sink)
    _launch(_cuda().grm_kv4_select, words, dev, what)
    return idx


def kv4_compact(kv: Kv4Layer, slots: Optional[torch.Tensor], idx: torch.Tensor, block_table: torch.Tensor, dst_table: torch.Tensor) -> None:
    """Copy token ``idx[i][h][j]`` of sequence ``slots[i]`` (kv head h, codes, maxima and mass as they are) to place j of the
    pages ``dst_table[i]`` (int32 [S][>= ceil(keep / 16)]).  The destination pages must not be among the sources, nor come twice:
    pages that other sequences share stay intact, and the caller swaps the tables afterwards.  Places whose ``idx`` is -1, or whose token
    has no page (``kv4_select`` takes such a token only where too few others are left), stay as they are."""
    data = kv.data
    P, Hkv, rec = data.shape
    dev, what = data.get_device(), "kv4_compact"
    table = _check_table(block_table, dev, what)
    if idx.dtype is not _INT or idx.dim() != 3 or not idx.is_contiguous() or idx.shape[1] != Hkv or idx.get_device() != dev:
        raise ValueError("kv4_compact: idx must be a contiguous int32 [sequences][kv heads][keep] on the cache's device")
    S, _, keep = idx.shape
    if dst_table.dtype is not _INT or dst_table.dim() != 2 or dst_table.shape[0] != S or dst_table.shape[1] * PAGE < keep or \
            (dst_table.stride(1) != 1 and dst_table.shape[1] > 1) or dst_table.get_device() != dev:
        raise ValueError("kv4_compact: dst_table must be int32 [sequences][>= keep / 16 pages] with contiguous rows on the cache's device")
    seq = _check_ints(slots, S, dev, what)
    if slots is None and S > table[1]:
        raise ValueError("kv4_compact: more sequences than the table has rows")
    if S > 65535:
        raise ValueError("kv4_compact: at most 65535 sequences")
    if S == 0 or keep == 0:
        return
    if dev < 0:
        codes, amax = ref.kv4_views(kv.data)
        P = kv.data.shape[0]
        for i in range(S):
            to, place, into = ref.kv4_place(dst_table, i, torch.arange(keep), P)
            for h in range(Hkv):
                page, at, ok = ref.kv4_place(block_table, i if slots is None else int(slots[i]), idx[i, h], P)
                ok = ok & into
                a, b, c, d = page[ok], at[ok], to[ok], place[ok]
                codes[c, h, :, d], amax[c, h, d] = codes[a, h, :, b], amax[a, h, b]
                if kv.mass is not None:
                    kv.mass[c, h, d] = kv.mass[a, h, b]
        return
    words = _pack[15](data.data_ptr(), _ptr(kv.mass), *table, P, seq, idx.data_ptr(), dst_table.data_ptr(), dst_table.stride(0), S, Hkv, rec // 18, keep)
    _launch(_cuda().grm_kv4_compact, words, dev, what)
