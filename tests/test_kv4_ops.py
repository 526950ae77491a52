"""The 4-bit KV cache against its definition in 64 bits: writing, reading back, attention, observed weight, selection and
moving of tokens.  Every test runs on CPU tensors (the fp32 forms) and, marked gpu, on the kernels.

Tolerances.  The page format is exact: codes, maxima, read-back rows, selected positions and moved records are compared bit
for bit.  An attention output is a bf16 (half a step: 2^-8 of the value) of a sum whose weights are rounded to at most two
factors of fp16 precision (2^-11 each, of sum p |v|).  A score is a sum of D products in fp32 over at least two partial sums:
its error is at most (D / 2) 2^-24 * scale * sum |q k|, a normalised weight moves by at most twice that, and the 2^-10 that
remain of the 2^-9 granted on sum p |v| cover it as long as D * 2^-24 * scale * sum |q k| < 2^-10, which every test's inputs
keep.  An observed weight is a sum of exp2 of such scores: relative error at most 2 (D + 16) 2^-24 * max(scale * sum |q k|)
for the scores (log2 e and the maximum's own error included) plus 2^-19 for exponentials, reciprocal and the sums over rows.
"""
import math

import pytest
import torch

from grimoire_b200.ops import kv4
from grimoire_b200.ops.core import AttnGeom

PAGE = 16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ---------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------------------------
def quantised(x):
    """[..., D] -> the values that its 4-bit form stands for, in 64 bits."""
    x = x.double().cpu()
    D = x.shape[-1]
    out = torch.empty_like(x)
    for j in range(D // 32):
        at = [d for d in range(D) if (d // 4) % (D // 32) == j]
        top = x[..., at].abs().amax(-1, keepdim=True)
        q = torch.round(7 * x[..., at] / torch.where(top > 0, top, torch.ones_like(top)))
        out[..., at] = q * top / 7
    return out


def attend64(q, k, v, pos, scale, window):
    """One row of one kv head: q [G][D], k / v [T][D] -> (out [G][D], sum p |v| [G][D], weights [G][T], scale * max sum |q k|)."""
    T = k.shape[0]
    t = torch.arange(T)
    seen = t <= pos
    if window:
        seen &= t > pos - window
    w = torch.zeros(q.shape[0], T, dtype=torch.float64)
    if not bool(seen.any()):
        z = torch.zeros(q.shape[0], k.shape[1], dtype=torch.float64)
        return z, z, w, 0.0
    s = scale * (q.double() @ k[seen].t())
    w[:, seen] = torch.softmax(s, dim=-1)
    size = float(scale * (q.double().abs() @ k[seen].abs().t()).max())
    return w @ v, w @ v.abs(), w, size


class Cache:
    """A filled cache with its values in 64 bits."""

    def __init__(self, lens, Hkv, D, device, seed=0, spare=4, mass=True, amp=1.0):
        g = torch.Generator().manual_seed(seed)
        per = [(n + PAGE - 1) // PAGE for n in lens]
        P = sum(per) + spare
        order = torch.randperm(P, generator=g).to(torch.int32)
        self.slots = torch.randperm(len(lens) + 1, generator=g)[: len(lens)].to(torch.int32)
        table = torch.full((len(lens) + 1, max(per + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in zip(self.slots.tolist(), per):
            table[s, :n] = order[at: at + n]
            at += n
        self.fresh = order[at:].to(device)
        self.table = table.to(device)
        self.lens, self.Hkv, self.D, self.device = list(lens), Hkv, D, device
        self.kv = kv4.Kv4Layer.alloc(P, Hkv, D, device, mass=mass)
        # what an earlier owner of the pages left: every byte pattern, NaN maxima among them
        self.kv.data.copy_(torch.randint(0, 256, self.kv.data.shape, generator=g, dtype=torch.uint8))
        self.kx = [(amp * torch.randn(n, Hkv * D, generator=g)).bfloat16() for n in lens]
        self.vx = [(amp * torch.randn(n, Hkv * D, generator=g)).bfloat16() for n in lens]
        total = sum(lens)
        if total:
            pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).to(device)
            seq = torch.cat([torch.full((n,), int(s)) for n, s in zip(lens, self.slots)]).to(torch.int32).to(device)
            kv4.kv4_append(self.kv, torch.cat(self.kx).to(device), torch.cat(self.vx).to(device), pos, seq, self.table)
        self.k = [quantised(x.reshape(-1, Hkv, D)) for x in self.kx]
        self.v = [quantised(x.reshape(-1, Hkv, D)) for x in self.vx]

    def attend(self, seqs, pos, q, G, scale, window=0, gate=None, **kw):
        geom = AttnGeom(self.Hkv * G, self.Hkv, self.D, self.D, scale, window=window)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.device)
        out = torch.full((len(seqs), self.Hkv * G * self.D), 9.0, dtype=torch.bfloat16, device=self.device)
        kv4.kv4_attn(q.to(self.device), i32([int(self.slots[s]) for s in seqs]), i32(list(pos)), self.table, self.kv, geom, out,
                     max(max(pos) + 1, 1), gate=None if gate is None else gate.to(self.device), **kw)
        return out.cpu()

    def expect(self, seqs, pos, q, G, scale, window=0):
        """(out, sum p |v|) [M][Hkv * G * D], weights per row [Hkv][T] (summed over G), size of the scores."""
        outs, sizes, weights, top = [], [], [], 0.0
        for m, (s, p) in enumerate(zip(seqs, pos)):
            o, a, w = [], [], []
            for h in range(self.Hkv):
                r = attend64(q[m].reshape(self.Hkv, G, self.D)[h], self.k[s][:, h], self.v[s][:, h], p, scale, window)
                o.append(r[0]); a.append(r[1]); w.append(r[2].sum(0)); top = max(top, r[3])
            outs.append(torch.cat(o).flatten()); sizes.append(torch.cat(a).flatten()); weights.append(torch.stack(w))
        return torch.stack(outs), torch.stack(sizes), weights, top

    def mass_of(self, s):
        t = torch.arange(self.lens[s])
        page = self.table.cpu()[int(self.slots[s]), t // PAGE].long()
        return self.kv.mass.cpu()[page, :, t % PAGE].t()                      # [Hkv][T]


def close(out, ref, size):
    tol = 2 ** -8 * ref.abs() + 2 ** -9 * size + 1e-30
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"largest excess {float((err - tol).max()):.3g}, error {float(err.max()):.3g}"


def scores_in_range(D, size):
    assert D * 2 ** -24 * size < 2 ** -10


# ---------------------------------------------------------------------------------------------
# write and read back
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,Hkv", [(64, 1), (64, 3), (128, 2), (128, 8), (256, 1), (256, 4)])
def test_append_then_gather_is_the_definition(device, D, Hkv):
    lens = [1, 16, 37]
    c = Cache(lens, Hkv, D, device, seed=D + Hkv)
    T = 40
    ok = torch.full((3, T, Hkv * D), 5.0, dtype=torch.bfloat16, device=device)
    ov = ok.clone()
    kv4.kv4_gather(c.kv, c.table, c.slots.to(device), torch.tensor(lens, dtype=torch.int32, device=device), ok, ov)
    for i, n in enumerate(lens):
        assert torch.equal(ok[i, :n].cpu(), c.k[i].reshape(n, -1).bfloat16())
        assert torch.equal(ov[i, :n].cpu(), c.v[i].reshape(n, -1).bfloat16())
        assert bool((ok[i, n:] == 5).all()) and bool((ov[i, n:] == 5).all())          # rows behind the sequence stay


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_codes_at_ties_zero_groups_and_extremes(device, D):
    x = torch.randn(12, D, generator=torch.Generator().manual_seed(3)).bfloat16()
    half = torch.tensor([1.0, 0.5, 0.21484375, -0.5, -1.0, 0.0, 3.5 / 7, 1.5])[torch.arange(D) % 8]
    x[0] = half.bfloat16()                     # halves of the maximum: ties of the rounding
    x[1] = 0
    x[2] = 3.3e38
    x[2, ::2] = -1e-38
    x[3] = torch.where(torch.arange(D) % 3 == 0, 1e-40, -3e-39).bfloat16()            # subnormal
    x[4, 8:] = 0
    x[5] = 2.0 ** -120
    k, v = x[:, None].expand(12, 2, D).reshape(12, 2 * D).contiguous(), (-x)[:, None].expand(12, 2, D).reshape(12, 2 * D).contiguous()
    kv = kv4.Kv4Layer.alloc(2, 2, D, device)
    table = torch.tensor([[1]], dtype=torch.int32, device=device)
    pos = torch.arange(12, dtype=torch.int32, device=device)
    kv4.kv4_append(kv, k.to(device), v.to(device), pos, torch.zeros_like(pos), table)
    ok, ov = (torch.zeros(1, 12, 2 * D, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv4.kv4_gather(kv, table, None, None, ok, ov)
    ref = quantised(k.reshape(12, 2, D)).reshape(12, -1)
    rows = [0, 1, 2, 4, 5] + list(range(6, 12))
    assert torch.equal(ok[0].cpu()[rows], ref[rows].bfloat16()) and torch.equal(ov[0].cpu()[rows], (-ref[rows]).bfloat16())
    # a subnormal result may be rounded once more on the way through fp32: one step of the subnormal grid
    assert float((ok[0].cpu()[3].double() - ref[3]).abs().max()) <= 2.0 ** -133


@pytest.mark.parametrize("device", DEVICES)
def test_group_with_nan_or_infinity_reads_back_as_nan(device):
    D = 128
    x = torch.randn(3, D).bfloat16()
    x[0, 5], x[1, 70], x[2, 127] = math.nan, math.inf, -math.inf
    kv = kv4.Kv4Layer.alloc(1, 1, D, device)
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    pos = torch.arange(3, dtype=torch.int32, device=device)
    kv4.kv4_append(kv, x.to(device), x.to(device), pos, torch.zeros_like(pos), table)
    ok, ov = (torch.zeros(1, 3, D, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv4.kv4_gather(kv, table, None, None, ok, ov)
    group = (torch.arange(D) // 4) % (D // 32)
    for row, d in ((0, 5), (1, 70), (2, 127)):
        bad = group == group[d]
        for o in (ok, ov):
            assert bool(torch.isnan(o[0, row].cpu()[bad]).all()) and bool(torch.isfinite(o[0, row].cpu()[~bad]).all())


@pytest.mark.parametrize("device", DEVICES)
def test_append_takes_strided_rows_and_skips_what_is_not_mapped(device):
    D, Hkv = 64, 2
    g = torch.Generator().manual_seed(1)
    big = torch.randn(6, 3 * Hkv * D + 3, generator=g).bfloat16().to(device)
    k, v = big[:, 1: 1 + Hkv * D], big[:, 1 + Hkv * D: 1 + 2 * Hkv * D]                # rows that start on 2-byte boundaries
    kv = kv4.Kv4Layer.alloc(3, Hkv, D, device, mass=True)
    kv.mass.fill_(7)
    before = kv.data.clone()
    table = torch.tensor([[2, -1], [99, 0]], dtype=torch.int32, device=device)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    #      written, unmapped, outside the table, bad page, written, bad slot / position
    kv4.kv4_append(kv, k, v, i32([3, 17, 40, 3, 31, -1]), i32([0, 0, 0, 1, 1, 0]), table)
    kv4.kv4_append(kv, k[:2], v[:2], i32([0, 0]), i32([-1, 2]), table)
    assert torch.equal(kv.data[1], before[1])
    ok, ov = (torch.zeros(2, 32, Hkv * D, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv4.kv4_gather(kv, table, None, None, ok, ov)
    ref = quantised(k.cpu().reshape(6, Hkv, D)).reshape(6, -1).bfloat16()
    assert torch.equal(ok[0, 3].cpu(), ref[0]) and torch.equal(ok[1, 31].cpu(), ref[4])
    assert bool((ok[0, 16:] == 0).all()) and bool((ok[1, :16] == 0).all())             # pages that are not mapped: rows stay
    m = kv.mass.cpu()
    assert bool((m[2, :, 3] == 0).all()) and bool((m[0, :, 15] == 0).all()) and int((m == 0).sum()) == 2 * Hkv


@pytest.mark.parametrize("device", DEVICES)
def test_gather_into_strided_rows(device):
    c = Cache([21], 2, 64, device, seed=5)
    big = torch.zeros(2, 21, 2 * 128 + 1, dtype=torch.bfloat16, device=device)
    kv4.kv4_gather(c.kv, c.table, c.slots.to(device), None, big[:1, :, 1:129], big[1:, :, 129:257])
    assert torch.equal(big[0, :, 1:129].cpu(), c.k[0].reshape(21, -1).bfloat16())
    assert torch.equal(big[1, :, 129:].cpu(), c.v[0].reshape(21, -1).bfloat16())
    assert bool((big[0, :, 0] == 0).all()) and bool((big[0, :, 129:] == 0).all())


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 9, 16])
def test_attention_head_layouts(device, D, G):
    lens, Hkv = [1, 16, 17, 95, 301], 2
    c = Cache(lens, Hkv, D, device, seed=G + D)
    q = (1.5 * torch.randn(5, Hkv * G * D, generator=torch.Generator().manual_seed(G))).bfloat16()
    seqs, pos, scale = [3, 0, 4, 1, 2], [94, 0, 300, 15, 16], 1 / math.sqrt(D)
    ref, size, _, top = c.expect(seqs, pos, q, G, scale)
    scores_in_range(D, top)
    close(c.attend(seqs, pos, q, G, scale), ref, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 2, 15, 31, 33, 127, 128, 129, 1000, 2049])
def test_attention_lengths(device, n):
    c = Cache([n], 1, 128, device, seed=n)
    q = (2 * torch.randn(1, 4 * 128, generator=torch.Generator().manual_seed(n))).bfloat16()
    ref, size, _, top = c.expect([0], [n - 1], q, 4, 0.1)
    scores_in_range(128, top)
    close(c.attend([0], [n - 1], q, 4, 0.1), ref, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window", [1, 5, 16, 17, 100, 5000])
@pytest.mark.parametrize("D", [64, 256])
def test_attention_window(device, window, D):
    lens = [200, 33, 8]
    c = Cache(lens, 2, D, device, seed=window)
    q = torch.randn(3, 2 * 3 * D, generator=torch.Generator().manual_seed(0)).bfloat16()
    pos = [199, 20, 7]
    ref, size, _, top = c.expect([0, 1, 2], pos, q, 3, 0.2, window)
    scores_in_range(D, top)
    close(c.attend([0, 1, 2], pos, q, 3, 0.2, window), ref, size)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_gate_strides_and_empty_rows(device):
    """Rows of a padded batch (negative position, no slot, nothing mapped) give zeros; rows may be slices of wider tensors."""
    D, Hkv, G = 128, 2, 5
    c = Cache([70, 130], Hkv, D, device, seed=2)
    w = Hkv * G * D
    g = torch.Generator().manual_seed(4)
    big = torch.randn(5, 2 * w + 5, generator=g).bfloat16()
    q, gate = big[:, 1: 1 + w], big[:, 1 + w: 1 + 2 * w]
    out = torch.full((5, w + 3), 3.0, dtype=torch.bfloat16, device=device)
    seq = torch.tensor([int(c.slots[0]), int(c.slots[1]), -1, int(c.slots[0]), 77], dtype=torch.int32, device=device)
    pos = torch.tensor([69, 100, 50, -1, 4], dtype=torch.int32, device=device)
    geom = AttnGeom(Hkv * G, Hkv, D, D, 0.1)
    big = big.to(device)
    kv4.kv4_attn(big[:, 1: 1 + w], seq, pos, c.table, c.kv, geom, out[:, 2: 2 + w], 101, gate=big[:, 1 + w: 1 + 2 * w])
    ref, size, _, top = c.expect([0, 1], [69, 100], q[:2], G, 0.1)
    scores_in_range(D, top)
    sg = torch.sigmoid(gate[:2].double())
    close(out[:2, 2: 2 + w].cpu(), ref * sg, size * sg)
    assert bool((out[2:, 2: 2 + w] == 0).all())
    assert bool((out[:, :2] == 3).all()) and bool((out[:, 2 + w:] == 3).all())


@pytest.mark.parametrize("device", DEVICES)
def test_attention_ignores_unmapped_pages_and_positions_behind_the_table(device):
    D, G = 64, 2
    c = Cache([64], 1, D, device, seed=9)
    table = c.table.clone()
    slot = int(c.slots[0])
    table[slot, 1], table[slot, 2] = -5, 10 ** 6
    c.table = table
    q = torch.randn(1, G * D, generator=torch.Generator().manual_seed(1)).bfloat16()
    out = c.attend([0], [1000], q, G, 0.3)                                            # 5 table entries: 80 positions
    seen = torch.tensor(list(range(16)) + list(range(48, 64)))
    o, a, _, top = attend64(q.reshape(G, D), c.k[0][seen, 0], c.v[0][seen, 0], 99, 0.3, 0)
    scores_in_range(D, top)
    close(out, o.flatten()[None], a.flatten()[None])


@pytest.mark.parametrize("device", DEVICES)
def test_attention_of_nan_stays_in_its_rows_and_channels(device):
    """NaN in a key that a row sees makes the row NaN; NaN in a value makes its 32 channels NaN; hidden ones change nothing."""
    D, n = 128, 40
    c = Cache([n, n, n], 1, D, device, seed=6)
    q = torch.randn(3, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    for s, which in ((0, "k"), (1, "v"), (2, "both")):
        k, v = c.kx[s][30:31].clone(), c.vx[s][30:31].clone()
        if which != "v":
            k[0, 3] = math.nan
        if which != "k":
            v[0, 3] = math.inf
        kv4.kv4_append(c.kv, k.to(device), v.to(device), i32([30]), i32([int(c.slots[s])]), c.table)
    seen = c.attend([0, 1, 2], [n - 1] * 3, q, 1, 0.1)
    bad = (torch.arange(D) // 4) % 4 == 0
    assert bool(torch.isnan(seen[0]).all())
    assert bool(torch.isnan(seen[1][bad]).all())
    ref, size, _, _ = c.expect([0, 1, 2], [n - 1] * 3, q, 1, 0.1)
    close(seen[1:2][:, ~bad], ref[1:2][:, ~bad], size[1:2][:, ~bad])
    ref, size, _, _ = c.expect([0, 1, 2], [29] * 3, q, 1, 0.1)
    close(c.attend([0, 1, 2], [29] * 3, q, 1, 0.1), ref, size)
    qn = q.clone()
    qn[0, 0] = math.nan
    assert bool(torch.isnan(c.attend([0], [29], qn[:1], 1, 0.1)).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("amp", [2.0 ** -60, 1e-4, 300.0, 2.0 ** 50])
def test_attention_over_small_and_large_values(device, amp):
    """Values far outside the range of fp16 (the scores stay of order one: the query carries the inverse factor)."""
    D, G, n = 128, 3, 150
    c = Cache([n], 1, D, device, seed=8, amp=amp)
    q = (torch.randn(1, G * D, generator=torch.Generator().manual_seed(3)) / amp).bfloat16()
    ref, size, _, top = c.expect([0], [n - 1], q, G, 0.1)
    scores_in_range(D, top)
    close(c.attend([0], [n - 1], q, G, 0.1), ref, size)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_with_one_token_of_far_larger_values(device):
    """A late token with values 2^30 times the others', and little weight: the running scale of the values follows it."""
    D, n = 64, 400
    c = Cache([n], 1, D, device, seed=12)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    big = (c.vx[0][210:211].float() * 2.0 ** 30).bfloat16()
    kv4.kv4_append(c.kv, c.kx[0][210:211].to(device), big.to(device), i32([210]), i32([int(c.slots[0])]), c.table)
    c.v[0][210] = quantised(big.reshape(1, 1, D))[0]
    q = torch.randn(1, 2 * D, generator=torch.Generator().manual_seed(5)).bfloat16()
    for pos in (209, 399):
        ref, size, _, top = c.expect([0], [pos], q, 2, 0.1)
        scores_in_range(D, top)
        close(c.attend([0], [pos], q, 2, 0.1), ref, size)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hkv,G,block,window", [(128, 8, 5, 1, 0), (64, 8, 12, 1, 0), (256, 4, 6, 1, 0), (128, 8, 4, 3, 0), (64, 16, 1, 1, 3000)])
def test_attention_of_a_large_ragged_batch(D, Hkv, G, block, window):
    """Enough pages for every SM: the keys are dealt out over the whole batch, whatever the rows' lengths; some rows see nothing."""
    lens = [5000, 33, 4811, 2600, 16, 4999, 3333, 1, 4096, 4990]
    c = Cache(lens, Hkv, D, "cuda", seed=D)
    seqs = [s for s in range(10) for _ in range(block)]
    pos = [max(0, lens[s] - block + r) for s in range(10) for r in range(block)]
    for m in (3 * block, 10 * block - 1):
        pos[m] = -1
    q = torch.randn(len(seqs), Hkv * G * D, generator=torch.Generator().manual_seed(G)).bfloat16()
    scale = 1 / math.sqrt(D)
    out = c.attend(seqs, pos, q, G, scale, window, block=block, observe="set")
    ref, size, w, top = c.expect(seqs, pos, q, G, scale, window)
    scores_in_range(D, top)
    close(out, ref, size)
    eps = 2 * (D + 16) * 2 ** -24 * top + 2 ** -19
    for s in range(10):
        rows = range(s * block, (s + 1) * block)
        want, seen = sum(w[r] for r in rows), max(pos[r] for r in rows) + 1
        got = c.mass_of(s).double()
        assert bool(((got - want)[:, :seen].abs() <= eps * want[:, :seen] + 1e-35).all())


# ---------------------------------------------------------------------------------------------
# observed weight
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,G,block,window", [(64, 1, 1, 0), (128, 5, 16, 0), (128, 8, 3, 40), (256, 2, 7, 0), (64, 16, 2, 9)])
def test_observed_weight_set_then_add(device, D, G, block, window):
    lens, Hkv = [37, 150, 16], 2
    c = Cache(lens, Hkv, D, device, seed=block)
    c.kv.mass.fill_(11.0)
    scale = 1 / math.sqrt(D)
    g = torch.Generator().manual_seed(D)
    seqs = [s for s in (0, 1, 2) for _ in range(block)]
    pos = [lens[s] - block + r for s in (0, 1, 2) for r in range(block)]
    q = torch.randn(len(seqs), Hkv * G * D, generator=g).bfloat16()
    out = c.attend(seqs, pos, q, G, scale, window, block=block, observe="set")
    ref, size, w0, top = c.expect(seqs, pos, q, G, scale, window)
    scores_in_range(D, top)
    close(out, ref, size)
    q1 = torch.randn(3, Hkv * G * D, generator=g).bfloat16()
    pos1 = [n - 1 for n in lens]
    out1 = c.attend([0, 1, 2], pos1, q1, G, scale, window, observe="add")
    ref1, size1, w1, top1 = c.expect([0, 1, 2], pos1, q1, G, scale, window)
    close(out1, ref1, size1)
    eps = 2 * (D + 16) * 2 ** -24 * max(top, top1) + 2 ** -19
    for s in (0, 1, 2):
        want = torch.stack(w0[s * block: (s + 1) * block]).sum(0) + w1[s]
        got = c.mass_of(s).double()
        assert bool(((got - want).abs() <= eps * want + 1e-35).all()), float(((got - want).abs() / want.clamp_min(1e-30)).max())
    live = torch.zeros(c.kv.mass.shape[0], PAGE, dtype=torch.bool)
    for s, n in enumerate(lens):
        t = torch.arange(n)
        live[c.table.cpu()[int(c.slots[s]), t // PAGE].long(), t % PAGE] = True
    assert bool((c.kv.mass.cpu().transpose(1, 2)[~live] == 11.0).all())               # nothing behind the last tokens, no other page


@pytest.mark.parametrize("device", DEVICES)
def test_observed_weight_of_two_blocks_of_one_sequence(device):
    D, G = 64, 2
    c = Cache([90, 20], 1, D, device, seed=3)
    seqs, pos = [0, 0, 1, 1, 0, 0], [80, 81, 10, 11, 88, 89]
    q = torch.randn(6, G * D, generator=torch.Generator().manual_seed(7)).bfloat16()
    c.attend(seqs, pos, q, G, 0.2, block=2, observe="set")
    _, _, w, top = c.expect(seqs, pos, q, G, 0.2)
    eps = 2 * (D + 16) * 2 ** -24 * top + 2 ** -19
    for s, rows in ((0, [0, 1, 4, 5]), (1, [2, 3])):
        want = sum(w[r] for r in rows)
        seen = max(pos[r] for r in rows) + 1
        got = c.mass_of(s).double()
        assert bool(((got - want)[:, :seen].abs() <= eps * want[:, :seen] + 1e-35).all())


# ---------------------------------------------------------------------------------------------
# selection and moving
# ---------------------------------------------------------------------------------------------
def expected_kept(m, n, keep, recent, sink):
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    must = [t for t in range(n) if t < sink or t >= n - recent]
    rest = sorted((t for t in range(n) if sink <= t < n - recent), key=lambda t: (math.isnan(m[t]), -m[t] if not math.isnan(m[t]) else 0, t))
    return sorted(must + rest[: keep - len(must)])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["normal", "ties", "zero", "special"])
@pytest.mark.parametrize("keep,recent,sink", [(1, 0, 0), (1, 1, 0), (7, 3, 4), (40, 8, 2), (100, 0, 0), (64, 60, 4), (2000, 16, 4)])
def test_selection(device, kind, keep, recent, sink):
    lens, Hkv = [300, 1, 101, 1537], 2
    c = Cache(lens, Hkv, 64, device, seed=keep)
    g = torch.Generator().manual_seed(keep)
    m = torch.rand(c.kv.mass.shape, generator=g)
    if kind == "ties":
        m = torch.randint(0, 3, m.shape, generator=g).float()
    elif kind == "zero":
        m.zero_()
    elif kind == "special":
        pick = torch.randint(0, 8, m.shape, generator=g)
        for i, x in enumerate([math.nan, math.inf, -0.0, 0.0, -1.5, 1e-42, -math.inf]):
            m[pick == i] = x
    c.kv.mass.copy_(m)
    idx = kv4.kv4_select(c.kv, c.slots.to(device), torch.tensor(lens, dtype=torch.int32, device=device), c.table, keep, recent, sink)
    for s, n in enumerate(lens):
        mass = c.mass_of(s)
        for h in range(Hkv):
            assert idx[s, h].tolist() == expected_kept(mass[h].tolist(), n, keep, recent, sink)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,keep", [(64, 1), (128, 33), (256, 48), (128, 200)])
def test_compaction_moves_records_and_mass_and_leaves_the_rest(device, D, keep):
    lens, Hkv = [120, 150], 2
    need = (keep + PAGE - 1) // PAGE
    c = Cache(lens, Hkv, D, device, seed=D, spare=2 * need + 2)
    c.kv.mass.copy_(torch.rand(c.kv.mass.shape, generator=torch.Generator().manual_seed(1)))
    fresh = c.fresh[: 2 * need].reshape(2, need)
    before, mass0 = c.kv.data.clone(), c.kv.mass.clone()
    idx = kv4.kv4_select(c.kv, c.slots.to(device), torch.tensor(lens, dtype=torch.int32, device=device), c.table, keep, 0, 0)
    kv4.kv4_compact(c.kv, c.slots.to(device), idx, c.table, fresh)
    ok, ov = (torch.zeros(2, keep, Hkv * D, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv4.kv4_gather(c.kv, fresh, None, torch.tensor(lens, dtype=torch.int32, device=device), ok, ov)
    for s, n in enumerate(lens):
        old = c.mass_of(s)
        for h in range(Hkv):
            at = [t for t in idx[s, h].tolist() if t >= 0]
            assert len(at) == min(keep, n)
            assert torch.equal(ok[s, : len(at), h * D: (h + 1) * D].cpu(), c.k[s][at, h].bfloat16())
            assert torch.equal(ov[s, : len(at), h * D: (h + 1) * D].cpu(), c.v[s][at, h].bfloat16())
            j = torch.arange(len(at))
            assert torch.equal(c.kv.mass.cpu()[fresh.cpu()[s, j // PAGE].long(), h, j % PAGE], old[h, at])
    others = torch.ones(before.shape[0], dtype=torch.bool)
    others[fresh.flatten().long().cpu()] = False
    assert torch.equal(c.kv.data.cpu()[others], before.cpu()[others]) and torch.equal(c.kv.mass.cpu()[others], mass0.cpu()[others])
    if keep % PAGE:                                                                   # the places behind the last kept token
        tail, t0 = fresh[0, need - 1], keep % PAGE
        assert torch.equal(c.kv.mass[tail, :, t0:], mass0[tail, :, t0:])


@pytest.mark.parametrize("device", DEVICES)
def test_a_conversation_that_is_written_read_weighed_and_cut(device):
    """Prompt, observed last rows, decode steps that add to the mass, a cut, and decode steps over what is left."""
    D, Hkv, G, n, keep = 128, 2, 4, 90, 48
    c = Cache([n], Hkv, D, device, seed=21, spare=20)
    slot = int(c.slots[0])
    g = torch.Generator().manual_seed(22)
    scale = 1 / math.sqrt(D)
    q = torch.randn(8, Hkv * G * D, generator=g).bfloat16()
    c.attend([0] * 8, list(range(n - 8, n)), q, G, scale, block=8, observe="set")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    free = c.fresh.tolist()
    c.table = torch.cat((c.table, torch.full((c.table.shape[0], 4), -1, dtype=torch.int32, device=device)), dim=1)
    c.table[slot, (n + PAGE - 1) // PAGE] = free.pop()

    def step(t):
        kx, vx = (torch.randn(1, Hkv * D, generator=g).bfloat16() for _ in range(2))
        kv4.kv4_append(c.kv, kx.to(device), vx.to(device), i32([t]), i32([slot]), c.table)
        c.k[0] = torch.cat((c.k[0], quantised(kx.reshape(1, Hkv, D))))
        c.v[0] = torch.cat((c.v[0], quantised(vx.reshape(1, Hkv, D))))
        q1 = torch.randn(1, Hkv * G * D, generator=g).bfloat16()
        out = c.attend([0], [t], q1, G, scale, observe="add")
        ref, size, _, _ = c.expect([0], [t], q1, G, scale)
        close(out, ref, size)

    for t in range(n, n + 9):
        step(t)
    c.lens = [n + 9]
    fresh = torch.tensor([[free.pop() for _ in range(keep // PAGE)]], dtype=torch.int32, device=device)
    mass = c.mass_of(0)
    idx = kv4.kv4_select(c.kv, i32([slot]), i32([n + 9]), c.table, keep, 8, 4)
    for h in range(Hkv):
        assert idx[0, h].tolist() == expected_kept(mass[h].tolist(), n + 9, keep, 8, 4)
    kv4.kv4_compact(c.kv, i32([slot]), idx, c.table, fresh)
    c.table[slot] = -1
    c.table[slot, : keep // PAGE] = fresh[0]
    c.table[slot, keep // PAGE] = free.pop()
    for x in (c.k, c.v):
        x[0] = torch.stack([x[0][idx[0, h].long().cpu(), h] for h in range(Hkv)], dim=1)
    c.lens = [keep]
    assert torch.equal(c.mass_of(0), torch.stack([mass[h, idx[0, h].long().cpu()] for h in range(Hkv)]))
    for t in range(keep, keep + 5):
        step(t)


# ---------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    D, Hkv = 64, 2
    kv = kv4.Kv4Layer.alloc(4, Hkv, D, device, mass=True)
    bare = kv4.Kv4Layer.alloc(4, Hkv, D, device)
    table = torch.zeros(1, 4, dtype=torch.int32, device=device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    x = torch.zeros(2, Hkv * D, dtype=torch.bfloat16, device=device)
    q = torch.zeros(2, 4 * D, dtype=torch.bfloat16, device=device)
    geom = AttnGeom(4, Hkv, D, D, 0.1)
    attn = lambda **k: kv4.kv4_attn(**{**dict(q=q, row_seq=i32(0, 0), row_pos=i32(0, 1), block_table=table, kv=kv, geom=geom, out=q.clone(), max_len=2), **k})
    attn()
    bad = [
        lambda: kv4.Kv4Layer.alloc(4, Hkv, 96, device),
        lambda: kv4.kv4_append(kv, x.float(), x, i32(0, 1), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x[:, :-1], x, i32(0, 1), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x, x[:1], i32(0, 1), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x, x, i32(0), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x, x, i32(0, 1).long(), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x, x, i32(0, 1), i32(0, 0), table.long()),
        lambda: kv4.kv4_append(kv, x, x, i32(0, 1), i32(0, 0), table[:, ::2]),
        lambda: kv4.kv4_append(kv4.Kv4Layer(kv.data[:, :1]), x, x, i32(0, 1), i32(0, 0), table),
        lambda: kv4.kv4_append(kv4.Kv4Layer(kv.data, kv.mass[:2]), x, x, i32(0, 1), i32(0, 0), table),
        lambda: kv4.kv4_append(kv, x.t().contiguous().t(), x, i32(0, 1), i32(0, 0), table),
        lambda: kv4.Kv4Layer(kv.data, torch.zeros(4 * Hkv * PAGE + 1, device=device)[1:].view(4, Hkv, PAGE)),
        lambda: kv4.Kv4Layer(torch.zeros(18 * D + 8, dtype=torch.uint8, device=device)[8:].view(1, 1, 18 * D)),
        lambda: kv4.kv4_gather(kv, table, None, None, x[None].float(), x[None]),
        lambda: kv4.kv4_gather(kv, table, None, None, x, x),
        lambda: kv4.kv4_gather(kv, table, None, None, x[None].expand(2, 2, Hkv * D), x[None].expand(2, 2, Hkv * D)),
        lambda: kv4.kv4_gather(kv, table, i32(0, 0), None, x[None], x[None]),
        lambda: attn(q=q.float()), lambda: attn(out=q[:1]), lambda: attn(gate=q[:, :-1]), lambda: attn(row_pos=i32(0)),
        lambda: attn(geom=AttnGeom(4, 4, D, D, 0.1)), lambda: attn(geom=AttnGeom(4, Hkv, 128, D, 0.1)), lambda: attn(geom=AttnGeom(5, Hkv, D, D, 0.1)),
        lambda: attn(geom=AttnGeom(34, Hkv, D, D, 0.1)), lambda: attn(block=0), lambda: attn(block=3), lambda: attn(observe="sum"),
        lambda: attn(observe="add", kv=bare), lambda: attn(max_len=0),
        lambda: kv4.kv4_select(bare, None, i32(3), table, 2, 0), lambda: kv4.kv4_select(kv, None, i32(3), table, 0, 0),
        lambda: kv4.kv4_select(kv, None, i32(3), table, 4, 3, 2), lambda: kv4.kv4_select(kv, None, i32(3), table, 4, -1),
        lambda: kv4.kv4_select(kv, None, i32(3, 3), table, 4, 0), lambda: kv4.kv4_select(kv, i32(0, 0), i32(3), table, 4, 0),
        lambda: kv4.kv4_compact(kv, None, torch.zeros(1, Hkv, 17, dtype=torch.int32, device=device), table, table[:, :1]),
        lambda: kv4.kv4_compact(kv, None, torch.zeros(1, Hkv, 8, dtype=torch.int64, device=device), table, table),
        lambda: kv4.kv4_compact(kv, None, torch.zeros(1, 1, 8, dtype=torch.int32, device=device), table, table),
        lambda: kv4.kv4_compact(kv, None, torch.zeros(2, Hkv, 8, dtype=torch.int32, device=device), table, table),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("accepted:", i)


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows_is_no_work(device):
    kv = kv4.Kv4Layer.alloc(2, 1, 64, device, mass=True)
    table = torch.zeros(1, 2, dtype=torch.int32, device=device)
    none = torch.zeros(0, dtype=torch.int32, device=device)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=device)
    kv4.kv4_append(kv, x, x, none, none, table)
    kv4.kv4_gather(kv, table, none, none, x[None][:0], x[None][:0])
    assert kv4.kv4_attn(x, none, none, table, kv, AttnGeom(1, 1, 64, 64, 1.0), x, 1).shape[0] == 0
    assert tuple(kv4.kv4_select(kv, none, none, table, 3, 1).shape) == (0, 1, 3)


@pytest.mark.gpu
def test_calls_are_captured_and_replayed_and_streams_do_not_share_scratch():
    D, Hkv, G = 128, 2, 4
    c = Cache([400, 700], Hkv, D, "cuda", seed=30)
    geom = AttnGeom(Hkv * G, Hkv, D, D, 0.1)
    q = torch.randn(2, Hkv * G * D, device="cuda").bfloat16()
    seq, pos = c.slots.cuda(), torch.tensor([399, 699], dtype=torch.int32, device="cuda")
    want = torch.empty_like(q)
    kv4.kv4_attn(q, seq, pos, c.table, c.kv, geom, want, 700)
    outs, graphs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(2):
        out, gr = torch.zeros_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            for _ in range(4):
                kv4.kv4_attn(q, seq, pos, c.table, c.kv, geom, out, 700, observe="set")
        outs.append(out)
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    pos.fill_(123)                                                                    # the graph reads lengths on the device
    graphs[0].replay()
    torch.cuda.synchronize()
    ref, size, _, _ = c.expect([0, 1], [123, 123], q.cpu(), G, 0.1)
    close(outs[0].cpu(), ref, size)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB whose only mapped pages are its last ones."""
    D, Hkv, G = 256, 8, 2
    P = 2 ** 32 // (Hkv * 18 * D) + 40
    kv = kv4.Kv4Layer(torch.empty(P, Hkv, 18 * D, dtype=torch.uint8, device="cuda"))
    table = torch.tensor([[P - 1, P - 3, P - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(40, Hkv * D, generator=g).bfloat16() for _ in range(2))
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    kv4.kv4_append(kv, k.cuda(), v.cuda(), pos, torch.zeros_like(pos), table)
    ok, ov = (torch.zeros(1, 40, Hkv * D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv4.kv4_gather(kv, table, None, None, ok, ov)
    k4, v4 = quantised(k.reshape(40, Hkv, D)), quantised(v.reshape(40, Hkv, D))
    assert torch.equal(ok[0].cpu(), k4.reshape(40, -1).bfloat16()) and torch.equal(ov[0].cpu(), v4.reshape(40, -1).bfloat16())
    q = torch.randn(1, Hkv * G * D, generator=g).bfloat16()
    out = torch.zeros(1, Hkv * G * D, dtype=torch.bfloat16, device="cuda")
    kv4.kv4_attn(q.cuda(), pos[:1], pos[39:], table, kv, AttnGeom(Hkv * G, Hkv, D, D, 1 / 16), out, 40)
    r = [attend64(q.reshape(Hkv, G, D)[h], k4[:, h], v4[:, h], 39, 1 / 16, 0) for h in range(Hkv)]
    close(out.cpu(), torch.cat([x[0].flatten() for x in r])[None], torch.cat([x[1].flatten() for x in r])[None])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("width,n,keep", [(700, 1500, 300), (1300, 9000, 4000), (4000, 40000, 777)])
def test_selection_of_long_sequences_and_wide_tables(device, width, n, keep):
    """Sequences that several CTAs share, short ones in a wide table among them."""
    g = torch.Generator().manual_seed(n)
    P = (n + PAGE - 1) // PAGE + 2
    kv = kv4.Kv4Layer.alloc(P, 1, 64, device, mass=True)
    m = torch.exp(3 * torch.randn(P, 1, PAGE, generator=g)) * (torch.rand(P, 1, PAGE, generator=g) < 0.6)
    kv.mass.copy_(m)
    table = torch.full((3, width), -1, dtype=torch.int32)
    pages = (n + PAGE - 1) // PAGE
    table[1, :pages] = torch.randperm(P, generator=g)[:pages].to(torch.int32)
    table[2, :20] = table[1, :20]
    lens = [n, 300, 5]
    idx = kv4.kv4_select(kv, torch.tensor([1, 2, 2], dtype=torch.int32, device=device), torch.tensor(lens, dtype=torch.int32, device=device),
                         table.to(device), keep, 16, 4)
    for s, (slot, k) in enumerate(zip((1, 2, 2), lens)):
        t = torch.arange(k)
        mass = m[table[slot, t // PAGE].long(), 0, t % PAGE]
        assert idx[s, 0].tolist() == expected_kept(mass.tolist(), k, keep, 16, 4)


@pytest.mark.gpu
def test_selection_of_a_sequence_longer_than_the_cluster_keeps():
    n, keep = 150_000, 5000
    P = n // PAGE + 1
    kv = kv4.Kv4Layer.alloc(P, 1, 64, "cuda", mass=True)
    kv.mass.copy_(torch.randint(0, 40, kv.mass.shape, generator=torch.Generator().manual_seed(2)).float())
    table = torch.arange(P, dtype=torch.int32, device="cuda")[None]
    idx = kv4.kv4_select(kv, None, torch.tensor([n], dtype=torch.int32, device="cuda"), table, keep, 100, 4)
    assert idx[0, 0].tolist() == expected_kept(kv.mass.flatten()[:n].tolist(), n, keep, 100, 4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_append_of_many_rows_over_an_odd_number_of_heads(device, D):
    n, Hkv = 2800, 3
    c = Cache([n], Hkv, D, device, seed=D)
    ok, ov = (torch.zeros(1, n, Hkv * D, dtype=torch.bfloat16, device=device) for _ in range(2))
    kv4.kv4_gather(c.kv, c.table, c.slots.to(device), None, ok, ov)
    assert torch.equal(ok[0].cpu(), c.k[0].reshape(n, -1).bfloat16()) and torch.equal(ov[0].cpu(), c.v[0].reshape(n, -1).bfloat16())


# ---------------------------------------------------------------------------------------------
# blocks of many rows: the unpacked keys are shared by all their pairs
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,G,block,window", [(64, 16, 9, 0), (64, 1, 40, 33), (128, 5, 32, 0), (128, 16, 5, 70), (256, 12, 1, 0), (256, 3, 20, 0), (256, 16, 3, 25)])
def test_blocks_of_many_rows(device, D, G, block, window):
    lens, Hkv = [200, 65, 700], 2
    c = Cache(lens, Hkv, D, device, seed=D + G)
    seqs = [s for s in range(3) for _ in range(block)]
    pos = [lens[s] - block + r for s in range(3) for r in range(block)]
    pos[0] = -1
    q = torch.randn(len(seqs), Hkv * G * D, generator=torch.Generator().manual_seed(G)).bfloat16()
    gate = torch.randn(len(seqs), Hkv * G * D, generator=torch.Generator().manual_seed(G + 1)).bfloat16()
    scale = -1 / math.sqrt(D) if window else 1 / math.sqrt(D)
    out = c.attend(seqs, pos, q, G, scale, window, gate=gate, block=block)
    ref, size, _, _ = c.expect(seqs, pos, q, G, scale, window)
    top = c.expect(seqs, pos, q, G, abs(scale), window)[3]
    scores_in_range(D, top)
    sg = torch.sigmoid(gate.double())
    close(out, ref * sg, size * sg)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_block_keeps_nan_from_rows_and_channels_that_do_not_see_it(device, D):
    n, G, block = 60, 6, 8
    c = Cache([n], 1, D, device, seed=6)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    k, v = c.kx[0][55:57].clone(), c.vx[0][55:57].clone()
    v[0, 5], k[1, 3] = math.inf, math.nan                                             # token 55: a value, token 56: a key
    kv4.kv4_append(c.kv, k.to(device), v.to(device), i32([55, 56]), i32([int(c.slots[0])] * 2), c.table)
    c.v[0][55] = quantised(c.vx[0][55:56].reshape(1, 1, D))[0]
    q = torch.randn(block, G * D, generator=torch.Generator().manual_seed(2)).bfloat16()
    pos = list(range(50, 58))
    out = c.attend([0] * block, pos, q, G, 0.1, block=block).reshape(block, G, D)
    ref, size, _, top = c.expect([0] * block, pos, q, G, 0.1)
    scores_in_range(D, top)
    ref, size = ref.reshape(block, G, D), size.reshape(block, G, D)
    bad = (torch.arange(D) // 4) % (D // 32) == (5 // 4) % (D // 32)
    close(out[:5].flatten(1), ref[:5].flatten(1), size[:5].flatten(1))                # rows 50 .. 54 see neither
    assert bool(torch.isnan(out[5][:, bad]).all())                                    # row 55: 32 channels
    close(out[5][:, ~bad], ref[5][:, ~bad], size[5][:, ~bad])
    assert bool(torch.isnan(out[6:]).all())                                           # rows that see the key


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("amp", [2.0 ** -60, 1e-4, 300.0, 2.0 ** 50])
def test_block_over_small_and_large_values(device, amp):
    D, G, n, block = 128, 3, 150, 12
    c = Cache([n], 1, D, device, seed=8, amp=amp)
    q = (torch.randn(block, G * D, generator=torch.Generator().manual_seed(3)) / amp).bfloat16()
    pos = list(range(n - block, n))
    ref, size, w, top = c.expect([0] * block, pos, q, G, 0.1)
    scores_in_range(D, top)
    close(c.attend([0] * block, pos, q, G, 0.1, block=block, observe="set"), ref, size)
    want = sum(torch.nn.functional.pad(x, (0, n - x.shape[1])) for x in w)
    eps = 2 * (D + 16) * 2 ** -24 * top + 2 ** -19
    assert bool(((c.mass_of(0).double() - want).abs() <= eps * want + 1e-35).all())


@pytest.mark.parametrize("device", DEVICES)
def test_block_with_tokens_of_far_larger_values(device):
    D, n, G, block = 64, 400, 4, 9
    c = Cache([n], 1, D, device, seed=12)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    big = (c.vx[0][210:211].float() * 2.0 ** 30).bfloat16()
    kv4.kv4_append(c.kv, c.kx[0][210:211].to(device), big.to(device), i32([210]), i32([int(c.slots[0])]), c.table)
    c.v[0][210] = quantised(big.reshape(1, 1, D))[0]
    q = torch.randn(block, G * D, generator=torch.Generator().manual_seed(5)).bfloat16()
    for last in (209, 212, 399):
        pos = list(range(last - block + 1, last + 1))
        ref, size, _, top = c.expect([0] * block, pos, q, G, 0.1)
        scores_in_range(D, top)
        close(c.attend([0] * block, pos, q, G, 0.1, block=block), ref, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window", [0, 20])
def test_rows_at_the_largest_position_see_the_whole_table(device, window):
    """Positions end where the table does: 2^31 - 1 is the last place of the last page, which need not be mapped."""
    D, Hkv, G = 64, 1, 3
    c = Cache([48], Hkv, D, device, seed=60)
    q = torch.randn(2, Hkv * G * D, generator=torch.Generator().manual_seed(6)).bfloat16()
    geom = AttnGeom(Hkv * G, Hkv, D, D, 0.2, window=window)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    out = torch.zeros(2, Hkv * G * D, dtype=torch.bfloat16, device=device)
    slot = int(c.slots[0])
    kv4.kv4_attn(q.to(device), i32(slot, slot), i32(2 ** 31 - 1, -2 ** 31), c.table, c.kv, geom, out, 64, observe="set")
    last = c.table.shape[1] * PAGE - 1                                                # 63: the last 16 places are not mapped
    ref, size, weights, top = c.expect([0], [47], q[:1], G, 0.2, max(0, window - (last - 47)))
    scores_in_range(D, top)
    close(out[:1].cpu(), ref, size)
    assert not bool(out[1].any())
    assert float((c.mass_of(0).double() - weights[0]).abs().max()) < 2 ** -9 * G


@pytest.mark.parametrize("device", DEVICES)
def test_one_row_for_all_heads_and_rows_of_the_queries(device):
    """Broadcast rows (stride 0) are read like any others."""
    D, Hkv, G = 128, 2, 4
    c = Cache([100, 37], Hkv, D, device, seed=61)
    q = torch.randn(1, Hkv * G * D, generator=torch.Generator().manual_seed(7)).bfloat16()
    out = c.attend([0, 1, 0], [99, 36, 50], q.expand(3, -1), G, 0.1, gate=q.expand(3, -1))
    ref, size, _, top = c.expect([0, 1, 0], [99, 36, 50], q.expand(3, -1), G, 0.1)
    scores_in_range(D, top)
    gate = torch.sigmoid(q.double())
    close(out, ref * gate, size * gate)


@pytest.mark.gpu
def test_a_captured_cut_of_two_conversations_side_by_side():
    """Write, observe, select, compact and read back as one graph per cache; two of them replayed on two streams at once give what
    eager calls give."""
    D, Hkv, G, n, keep = 128, 2, 4, 90, 33
    geom = AttnGeom(Hkv * G, Hkv, D, D, 0.1)
    x = [torch.randn(1, Hkv * D, device="cuda").bfloat16() for _ in range(2)]
    q = torch.randn(1, Hkv * G * D, device="cuda").bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")

    def job(c):
        slot, pos, length, dst = c.slots[:1].cuda(), i32(n), i32(n + 1), c.fresh[:3][None].contiguous()
        rows = torch.arange(1, dtype=torch.int32, device="cuda")
        out, ok, ov = torch.zeros_like(q), *(torch.zeros(1, keep, Hkv * D, dtype=torch.bfloat16, device="cuda") for _ in range(2))

        def run():
            kv4.kv4_append(c.kv, x[0], x[1], pos, slot, c.table)
            kv4.kv4_attn(q, slot, pos, c.table, c.kv, geom, out, n + 1, observe="set")
            idx = kv4.kv4_select(c.kv, slot, length, c.table, keep, 8, 2)
            kv4.kv4_compact(c.kv, slot, idx, c.table, dst)
            kv4.kv4_gather(c.kv, dst, rows * 0, None, ok, ov)
            return idx
        return run, (out, ok, ov)

    caches = [Cache([n + 6], Hkv, D, "cuda", seed=70 + i) for i in range(2)]
    wants = []
    for c in caches:
        run, outs = job(c)
        idx = run()
        wants.append([idx.clone()] + [t.clone() for t in outs] + [c.kv.data.clone(), c.kv.mass.clone()])
    graphs, got = [], []
    for c in caches:
        run, outs = job(c)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            idx = run()
        graphs.append(gr)
        got.append([idx, *outs, c.kv.data, c.kv.mass])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for w, r in zip(wants, got):
        for a, b in zip(w, r):
            assert torch.equal(a.view(torch.uint8) if a.is_floating_point() else a, b.view(torch.uint8) if b.is_floating_point() else b)


# ---------------------------------------------------------------------------------------------
# blocks of many rows over keys that the caller announces as long: 128 pairs a tile
# ---------------------------------------------------------------------------------------------
LONG = 1 << 20


def attend_long(c, seqs, pos, q, G, scale, window=0, gate=None, table=None, **kw):
    geom = AttnGeom(c.Hkv * G, c.Hkv, c.D, c.D, scale, window=window)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=c.device)
    out = torch.full((len(seqs), c.Hkv * G * c.D), 9.0, dtype=torch.bfloat16, device=c.device)
    kv4.kv4_attn(q.to(c.device), i32([int(c.slots[s]) for s in seqs]), i32(list(pos)), c.table if table is None else table, c.kv, geom, out, LONG,
                 gate=None if gate is None else gate.to(c.device), **kw)
    return out.cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D,G,block,window", [(64, 16, 9, 0), (64, 1, 40, 33), (128, 5, 32, 0), (128, 16, 5, 70), (256, 12, 4, 0), (256, 3, 20, 0),
                                              (256, 16, 3, 25), (128, 1, 150, 0), (64, 7, 19, 64), (128, 3, 43, 1)])
def test_tiles_of_many_rows(device, D, G, block, window):
    lens, Hkv = [300, 165, 1700], 2
    c = Cache(lens, Hkv, D, device, seed=D + G)
    seqs = [s for s in range(3) for _ in range(block)]
    pos = [lens[s] - block + r for s in range(3) for r in range(block)]
    pos[0] = -1
    q = torch.randn(len(seqs), Hkv * G * D + 3, generator=torch.Generator().manual_seed(G)).bfloat16()[:, : Hkv * G * D]
    gate = torch.randn(len(seqs), Hkv * G * D, generator=torch.Generator().manual_seed(G + 1)).bfloat16()
    scale = -1 / math.sqrt(D) if window else 1 / math.sqrt(D)
    ref, size, weights, top = c.expect(seqs, pos, q, G, scale, window)
    scores_in_range(D, c.expect(seqs, pos, q, G, abs(scale), window)[3])
    sg = torch.sigmoid(gate.double())
    for kw in (dict(), dict(observe="set"), dict(observe="add", alone=True)):
        close(attend_long(c, seqs, pos, q, G, scale, window, gate=gate, block=block, **kw), ref * sg, size * sg)
    for s in range(3):
        want = sum(torch.nn.functional.pad(weights[m], (0, lens[s] - weights[m].shape[1])) for m in range(len(seqs)) if seqs[m] == s)
        err = (c.mass_of(s).double() - 2 * want).abs()
        assert float((err - 2 ** -8 * 2 * want).max()) < 2 ** -16 * block * G


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tiles_keep_nan_and_unmapped_pages_from_rows_and_channels(device, D):
    """Tokens with a NaN or infinite group in V reach only the rows that see them, and only that group's channels; a NaN in K only
    the rows that see it; pages that are not mapped hold nothing."""
    n, Hkv, G, block = 230, 1, 5, 40
    c = Cache([n], Hkv, D, device, seed=90)
    slot = int(c.slots[0])
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    rows = torch.cat([c.kx[0][200:201], c.kx[0][215:216], c.kx[0][225:226]]), torch.cat([c.vx[0][200:201], c.vx[0][215:216], c.vx[0][225:226]])
    rows[1][0, 3] = float("nan")                                                       # token 200: quad 0, group 0
    rows[1][1, 4 * (D // 32 - 1)] = float("inf")                                       # token 215: the last group
    rows[0][2, 9] = float("nan")                                                       # token 225: K
    kv4.kv4_append(c.kv, rows[0].to(device), rows[1].to(device), i32(200, 215, 225), i32(slot, slot, slot), c.table)
    hole = c.table.clone()
    hole[slot, 5] = -1
    hole[slot, 6] = 2 ** 30
    q = torch.randn(block, G * D, generator=torch.Generator().manual_seed(3)).bfloat16()
    pos = list(range(190, 230))
    scale = 1 / math.sqrt(D)
    got = attend_long(c, [0] * block, pos, q, G, scale, block=block, table=hole).reshape(block, G, D)
    group = (torch.arange(D) // 4) % (D // 32)
    keep = torch.tensor([t for t in range(n) if not 80 <= t < 112])
    for m, p in enumerate(pos):
        bad = torch.zeros(D, dtype=torch.bool)
        if p >= 200:
            bad |= group == 0
        if p >= 215:
            bad |= group == D // 32 - 1
        if p >= 225:
            bad[:] = True
        assert bool(torch.isnan(got[m][:, bad]).all()) and not bool(torch.isnan(got[m][:, ~bad]).any())
        at = keep[keep <= p]
        if not bool(bad.all()):
            v = c.v[0][at, 0].clone()
            v[:, bad] = 0
            o, size, _, top = attend64(q[m].reshape(G, D), c.k[0][at, 0], v, len(at) - 1, scale, 0)
            scores_in_range(D, top)
            close(got[m][:, ~bad], o[:, ~bad], size[:, ~bad])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("amp", [2.0 ** -60, 1e-4, 300.0, 2.0 ** 50])
def test_tiles_over_small_and_large_values(device, amp):
    D, Hkv, G, block = 128, 2, 4, 24
    c = Cache([333, 90], Hkv, D, device, seed=91, amp=amp)
    seqs, pos = [0] * block + [1] * block, list(range(333 - block, 333)) + list(range(90 - block, 90))
    q = torch.randn(2 * block, Hkv * G * D, generator=torch.Generator().manual_seed(8)).bfloat16()
    scale = 1 / (amp * math.sqrt(D))
    ref, size, _, top = c.expect(seqs, pos, q, G, scale)
    scores_in_range(D, top)
    close(attend_long(c, seqs, pos, q, G, scale, block=block), ref, size)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("far", [2.0 ** 24, 2.0 ** 100])
def test_tiles_with_tokens_of_far_larger_values(device, far):
    """The last token holds values ``far`` times the others', which its own row alone sees: the other rows must not lose theirs
    while those are within 2^-24 of the largest.  Beyond that a value is rounded where the operand's fp16 ends: the largest maximum
    stands at 2^13 or above and subnormals are 2^-24 apart, so half a code times a maximum is off by 2^-25 at most, 2^-38 of the
    largest maximum, a value by twice that; the softmax (at 2^13, weights of 2^-38 lost) adds as much: 2^-36 of the largest value."""
    D, Hkv, G, n, block = 128, 1, 5, 200, 24
    c = Cache([n], Hkv, D, device, seed=92)
    big = (far * torch.randn(1, D, generator=torch.Generator().manual_seed(1))).bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    kv4.kv4_append(c.kv, c.kx[0][n - 1:].to(device), big.to(device), i32(n - 1), i32(int(c.slots[0])), c.table)
    c.v[0][n - 1] = quantised(big.reshape(Hkv, D))
    q = torch.randn(block, G * D, generator=torch.Generator().manual_seed(2)).bfloat16()
    pos = list(range(n - block, n))
    ref, size, _, top = c.expect([0] * block, pos, q, G, 0.1)
    scores_in_range(D, top)
    got = attend_long(c, [0] * block, pos, q, G, 0.1, block=block)
    if far <= 2.0 ** 24:
        close(got, ref, size)
    else:
        size = size + 2 ** 9 * 2 ** -36 * float(big.abs().max())                       # close() allows 2^-9 of it
        close(got[-1:], ref[-1:], size[-1:])


@pytest.mark.parametrize("device", DEVICES)
def test_tiles_of_more_units_than_the_gpu_holds(device):
    """No cut of the keys: the rows are finished where they are computed; sequences of one block up to several."""
    D, Hkv, G, block, S = 64, 8, 4, 11, 40
    lens = [11 + 7 * i for i in range(S)]
    c = Cache(lens, Hkv, D, device, seed=93)
    seqs = [s for s in range(S) for _ in range(block)]
    pos = [lens[s] - block + r for s in range(S) for r in range(block)]
    q = torch.randn(len(seqs), Hkv * G * D, generator=torch.Generator().manual_seed(4)).bfloat16()
    ref, size, _, top = c.expect(seqs, pos, q, G, 0.125)
    scores_in_range(D, top)
    close(attend_long(c, seqs, pos, q, G, 0.125, block=block), ref, size)


@pytest.mark.gpu
def test_selection_of_a_sequence_whose_keys_no_cluster_holds():
    n, keep = 300001, 5000
    pages = (n + PAGE - 1) // PAGE
    kv = kv4.Kv4Layer.alloc(pages, 1, 64, "cuda", mass=True)
    mass = torch.exp(3 * torch.randn(pages, 1, PAGE, generator=torch.Generator().manual_seed(9)))
    mass[::3] = 0
    kv.mass.copy_(mass)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(10)).to(torch.int32)[None]
    got = kv4.kv4_select(kv, None, torch.tensor([n], dtype=torch.int32, device="cuda"), table.cuda(), keep, 100, 4)[0, 0].cpu().long()
    m = mass[table[0].long()].reshape(-1)[:n]
    rest = torch.sort(m[4: n - 100], descending=True, stable=True).indices[: keep - 104] + 4
    want = torch.cat([torch.arange(4), rest.sort().values, torch.arange(n - 100, n)])
    assert torch.equal(got, want)
