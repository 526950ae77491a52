"""Blocks of many rows over long 4-bit caches: tiles of 128 (row, head) pairs whose CTAs walk through 30 and more blocks of 64
tokens, against the definition in 64 bits and against themselves."""
import math

import pytest
import torch

from grimoire_b200.ops import kv4, ref
from grimoire_b200.ops.core import AttnGeom

from .test_kv4_ops import Cache, close, scores_in_range

PAGE = 16


class LongCache:
    """Sequences of ``lens`` tokens, each on pages of its own, filled on the device.  Keys carry a component along a fixed pattern of
    signs that grows from 0 to 3 over the sequence: rows with a share of it in their query see maxima that rise to the end."""

    def __init__(self, lens, Hkv, D, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        per = [(n + PAGE - 1) // PAGE for n in lens]
        order = torch.randperm(sum(per), generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), max(per)), -1, dtype=torch.int32, device="cuda")
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at: at + n]
            at += n
        self.lens, self.Hkv, self.D = lens, Hkv, D
        self.sign = torch.randint(0, 2, (D,), generator=g, device="cuda").float() * 2 - 1
        self.kv = kv4.Kv4Layer.alloc(sum(per), Hkv, D, "cuda", mass=True)
        for s, n in enumerate(lens):
            pos = torch.arange(n, dtype=torch.int32, device="cuda")
            k, v = (torch.randn(n, Hkv, D, generator=g, device="cuda") for _ in range(2))
            k += (3 * pos / n)[:, None, None] * self.sign
            kv4.kv4_append(self.kv, k.bfloat16().flatten(1), v.bfloat16().flatten(1), pos, torch.full_like(pos, s), self.table)

    def values(self, s):
        """K, V of sequence ``s`` in 64 bits: [Hkv][n][D]."""
        codes, amax = ref.kv4_views(self.kv.data[self.table[s, : (self.lens[s] + PAGE - 1) // PAGE].long()])
        q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).double() - 8                       # [pages][Hkv][K, V][16][D]
        x = (q.unflatten(-1, (8, self.D // 32, 4)) * amax.transpose(2, 3).double()[..., None, :, None] / 7).flatten(-3)
        return (x[:, :, i].transpose(0, 1).flatten(1, 2)[:, : self.lens[s]] for i in (0, 1))

    def mass_of(self, s):
        t = torch.arange(self.lens[s], device="cuda")
        return self.kv.mass[self.table[s, t // PAGE].long(), :, t % PAGE].t()


def deep_case(D, G, block, seqs, seed):
    """(cache, query rows [seqs * block][Hkv * G * D], positions) with late maxima for every other 32 pairs of a block."""
    Hkv = 4
    c = LongCache([2000 - 2 * (s % 37) for s in range(seqs)], Hkv, D, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    pair = torch.arange(block * G, device="cuda").reshape(block, 1, G, 1)
    late = (pair // 32 % 2 == 1).float() * (20 / (3 * math.sqrt(D)))             # scores that rise by 20 (29 binades)
    q = torch.randn(seqs, block, Hkv, G, D, generator=g, device="cuda") + late * c.sign
    pos = torch.tensor([n - block + r for n in c.lens for r in range(block)], dtype=torch.int32, device="cuda")
    return c, q.bfloat16().reshape(seqs * block, -1), pos


def against_definition(c, q, pos, out, G, block, scale):
    D, Hkv = c.D, c.Hkv
    for s, n in enumerate(c.lens):
        k, v = c.values(s)
        rows = slice(s * block, (s + 1) * block)
        qq = q[rows].double().reshape(block, Hkv, G, D)
        size = float(torch.einsum("rhgd,htd->rhgt", qq.abs(), k.abs()).max()) * abs(scale)
        scores_in_range(D, size)
        w = torch.einsum("rhgd,htd->rhgt", qq, k) * scale
        hidden = torch.arange(n, device="cuda") > pos[rows, None]
        w = torch.softmax(w.masked_fill(hidden[:, None, None], -math.inf), dim=-1)
        o, a = (torch.einsum("rhgt,htd->rhgd", w, x).reshape(block, -1).cpu() for x in (v, v.abs()))
        close(out[rows].cpu(), o, a)
        # A weight: twice the error of a score and of the maximum, as for short blocks, and 2^-19.  The sum over a row's tokens: a thread
        # adds 32 + 2 numbers a block of 64 tokens and one number a block in turn (2^-24 each), and scales the sum once a block at worst, by an
        # exponential of 2^-22 + 2^-24; the row's parts, a few, add 2^-24 each.  The sum over a token's pairs: 2^-24 each.
        blocks = (n + 63) // 64
        eps = 2 * (D + 16) * 2 ** -24 * size + 2 ** -19 + (34 + blocks + 8) * 2 ** -24 + blocks * (2 ** -22 + 2 ** -24) + block * G * 2 ** -24
        want = w.sum((0, 2))
        assert bool(((c.mass_of(s).double() - want).abs() <= eps * want + 1e-35).all())


@pytest.mark.gpu
@pytest.mark.parametrize("D,seqs", [(64, 38), (128, 38), (256, 19)])
@pytest.mark.parametrize("G,block", [(5, 8), (5, 16), (8, 16)])
def test_deep_tiles_are_the_definition_and_repeat_to_the_bit(D, seqs, G, block):
    """As many units as fill the GPU, so that a CTA walks through a whole sequence (31 blocks and more): every call gives the same bits,
    with warps that rescale at nearly every block beside warps that hardly ever do."""
    c, q, pos = deep_case(D, G, block, seqs, seed=D + G + block)
    geom = AttnGeom(c.Hkv * G, c.Hkv, D, D, 1 / math.sqrt(D))
    seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(block)
    out = torch.empty_like(q)
    kv4.kv4_attn(q, seq, pos, c.table, c.kv, geom, out, max(c.lens), block=block, observe="set")
    against_definition(c, q, pos, out, G, block, geom.scale)
    first, mass = out.clone(), c.kv.mass.clone()
    for _ in range(200):
        out.fill_(9)
        kv4.kv4_attn(q, seq, pos, c.table, c.kv, geom, out, max(c.lens), block=block, observe="set")
        assert torch.equal(out, first) and torch.equal(c.kv.mass, mass)


def call(c, rows, q, pos, G, max_len, block, **kw):
    """Outputs of blocks of sequences ``rows`` (a sequence per block)."""
    seq = torch.tensor(rows, dtype=torch.int32, device="cuda").repeat_interleave(block)
    out = torch.empty_like(q)
    kv4.kv4_attn(q, seq, torch.tensor(pos, dtype=torch.int32, device="cuda"), c.table, c.kv, AttnGeom(c.Hkv * G, c.Hkv, c.D, c.D, 0.1), out, max_len,
                 block=block, **kw)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hkv,G,block,max_len", [(128, 8, 5, 16, 4096), (128, 8, 5, 16, 8192), (64, 4, 8, 5, 16384), (256, 4, 6, 7, 12000), (128, 8, 5, 1, 4096)])
def test_alone_means_the_bits_of_a_call_of_one_block(D, Hkv, G, block, max_len):
    """Below and above the number of pairs and keys from which one block, or only several of them, would run in tiles."""
    c = LongCache([3000, 2100, 2900], Hkv, D, seed=D + block)
    q = torch.randn(3 * block, Hkv * G * D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(block)).bfloat16()
    pos = [n - block + r for n in c.lens for r in range(block)]
    together = call(c, [0, 1, 2], q, pos, G, max_len, block, alone=True)
    for s in range(3):
        rows = slice(s * block, (s + 1) * block)
        for kw in (dict(), dict(alone=True)):
            assert torch.equal(call(c, [s], q[rows], pos[rows], G, max_len, block, **kw), together[rows])


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hkv,G", [(128, 8, 5), (64, 16, 2), (256, 4, 6)])
@pytest.mark.parametrize("max_len", [1 << 16, 1 << 17, 1 << 18, 1 << 20])
def test_rows_of_a_verify_block_equal_single_steps_at_announced_lengths(D, Hkv, G, max_len):
    """One row by itself, and the same row among others with alone=True, below and above the lengths from which a batch's pages are dealt
    out over all CTAs."""
    c = LongCache([2500], Hkv, D, seed=G)
    q = torch.randn(5, Hkv * G * D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(G)).bfloat16()
    pos = list(range(2495, 2500))
    block = call(c, [0] * 5, q, pos, G, max_len, 1, alone=True)
    for i in range(5):
        assert torch.equal(call(c, [0], q[i: i + 1], pos[i: i + 1], G, max_len, 1), block[i: i + 1])


# ---------------------------------------------------------------------------------------------
# what a call writes
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_outputs_whose_rows_share_memory_are_refused(device):
    D, Hkv = 64, 2
    W = Hkv * D
    kv = kv4.Kv4Layer.alloc(4, Hkv, D, device)
    table = torch.zeros(2, 4, dtype=torch.int32, device=device)
    two = torch.tensor([0, 1], dtype=torch.int32, device=device)
    buf = torch.zeros(64 * W, dtype=torch.bfloat16, device=device)
    q = buf[: 2 * W].view(2, W)
    geom = AttnGeom(Hkv, Hkv, D, D, 0.1)
    attn = lambda out: kv4.kv4_attn(q, two * 0, two, table, kv, geom, out, 2)
    gather = lambda k, v: kv4.kv4_gather(kv, table, None, None, k, v)
    at = lambda s, t: buf.as_strided((2, 3, W), (s, t, 1), 8 * W)
    for out in (buf[:W].expand(2, W), buf.as_strided((2, W), (W - 8, 1))):
        with pytest.raises(ValueError):
            attn(out)
    ok = at(3 * W, W)
    for bad in (at(0, W), at(3 * W, 0), at(2 * W, W), at(W, W), at(W, 2 * W - 8)):
        for k, v in ((bad, ok), (ok, bad)):
            with pytest.raises(ValueError):
                gather(k, v)
    attn(buf.as_strided((2, W), (W + 2, 1), 4 * W))
    attn(buf[4 * W:].as_strided((2, W), (W, 1)))
    gather(ok, at(W, 2 * W))                                           # sequences inside, tokens outside
    kv4.kv4_attn(q[:1], two[:1], two[:1], table, kv, geom, buf[4 * W: 5 * W].expand(1, W), 2)


# ---------------------------------------------------------------------------------------------
# the documented range of keys
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("amp", [2.0 ** -64, 2.0 ** 62])
@pytest.mark.parametrize("block,max_len", [(1, 333), (12, 333), (12, 1 << 20)])
def test_keys_at_the_ends_of_their_range(device, amp, block, max_len):
    """Single rows, short blocks and tiles; queries carry the inverse factor, so that scores are of order one."""
    D, Hkv, G, n = 128, 2, 4, 333
    c = Cache([n], Hkv, D, device, seed=31, amp=amp)                                  # (normal values: up to four times amp)
    q = (torch.randn(block, Hkv * G * D, generator=torch.Generator().manual_seed(3)) / amp).bfloat16()
    pos = list(range(n - block, n))
    want, size, w, top = c.expect([0] * block, pos, q, G, 0.1)
    scores_in_range(D, top)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    out = torch.zeros(block, Hkv * G * D, dtype=torch.bfloat16, device=device)
    kv4.kv4_attn(q.to(device), i32([int(c.slots[0])] * block), i32(pos), c.table, c.kv, AttnGeom(Hkv * G, Hkv, D, D, 0.1), out, max_len, block=block,
                 observe="set")
    close(out.cpu(), want, size)
    total = sum(torch.nn.functional.pad(x, (0, n - x.shape[1])) for x in w)
    eps = 2 * (D + 16) * 2 ** -24 * top + 2 ** -19 + 64 * 2 ** -24                    # as in tiles above; few blocks and parts
    assert bool(((c.mass_of(0).double() - total).abs() <= eps * total + 1e-35).all())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_places_of_kept_tokens_without_a_page_stay(device):
    """Selection puts tokens of an unmapped page last; where they are kept all the same, their places are not written."""
    c = Cache([64], 2, 64, device, seed=8, spare=6)
    slot = int(c.slots[0])
    c.kv.mass.copy_(torch.rand(c.kv.mass.shape, generator=torch.Generator().manual_seed(3)) + 1)
    c.table[slot, 1] = -1                                              # tokens 16 .. 31
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    idx = kv4.kv4_select(c.kv, i32(slot), i32(64), c.table, 50, 0, 0)
    want = list(range(18)) + list(range(32, 64))                       # the 48 that exist, and the two earliest of the others
    assert idx[0].tolist() == [want, want]
    fresh = c.fresh[:4][None].contiguous()
    c.kv.data[fresh[0].long()] = 0x5a
    c.kv.mass[fresh[0].long()] = 7
    kv4.kv4_compact(c.kv, i32(slot), idx, c.table, fresh)
    mass = c.kv.mass[fresh[0].long()].transpose(1, 2).reshape(64, 2).cpu()
    assert bool((mass[[16, 17] + list(range(50, 64))] == 7).all()) and bool((mass[:16] < 2).all()) and bool((mass[18:50] < 2).all())
    codes, _ = ref.kv4_views(c.kv.data[fresh[0].long()].cpu())
    assert bool((codes[1, :, :, :2] == 0x5a).all()) and bool((codes[3, :, :, 2:] == 0x5a).all())


@pytest.mark.gpu
def test_deep_tiles_on_two_streams_at_once_captured_and_not():
    """Tiles of two head dimensions share the multiprocessors (and their TMEM): replayed on one stream, called on another, the bits stay."""
    jobs = []
    for D, seqs in ((128, 38), (256, 19)):
        c, q, pos = deep_case(D, 8, 8, seqs, seed=D)
        seq = torch.arange(seqs, dtype=torch.int32, device="cuda").repeat_interleave(8)
        out = torch.empty_like(q)

        def run(c=c, q=q, pos=pos, seq=seq, out=out, D=D):
            kv4.kv4_attn(q, seq, pos, c.table, c.kv, AttnGeom(c.Hkv * 8, c.Hkv, D, D, 1 / math.sqrt(D)), out, max(c.lens), block=8, observe="set")

        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        jobs.append((run, g, out, c, out.clone(), c.kv.mass.clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(40):
        for j, (run, g, out, c, _, _) in enumerate(jobs):
            with torch.cuda.stream(streams[j]):
                g.replay() if (i + j) % 2 else run()
    torch.cuda.synchronize()
    for _, _, out, c, want, mass in jobs:
        assert torch.equal(out, want) and torch.equal(c.kv.mass, mass)
