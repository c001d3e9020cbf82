"""The ends of the value range of the draft attention over the e4m3 cache, against
its 64-bit statement: value rows of zeros, value rows of very different sizes,
queries and keys at the ends of the bf16 range.

Tolerances, set before the first run. The output rounds to bf16 (2^-8 of the
value) and a weight to bf16 (2^-8 of itself) or, in the kernel of few query
rows, to a half (2^-11 of itself, 2^-33 of the row's largest contribution), so
with p the exact weights |out - ref| <= 2^-8 |ref| + (2^-8 + 2^-10) sum p |v|,
where 2^-10 covers the rounding of scores below 32 and the fp32 sums, and in
the 2-norm (independent roundings, 2^-8 / sqrt(3) each) below 2^-8."""
import math

import pytest
import torch

from test_spec_ops_gpu import A, D, DEV, SCALE, Draft, _lib, fp8_pool, gen, held_rows, tables_for  # noqa: F401

pytestmark = pytest.mark.gpu


class Held:
    """Sequences of one node count whose rows were written by the cache write, with their 64-bit reference."""

    def __init__(self, ks, vs, qs, hkv, bs=64, seed=0, scale=SCALE):
        self.lens, self.size, self.bs, self.scale = [k.shape[0] for k in ks], qs[0].shape[0], bs, scale
        self.table, blocks = tables_for(self.lens, bs, seed)
        self.views, _ = fp8_pool(blocks, bs, hkv, seed)
        slots = torch.cat([self.table[b].long()[torch.arange(n) // bs] * bs + torch.arange(n) % bs for b, n in enumerate(self.lens)])
        A().store_kvcache_fp8(torch.cat(ks).to(DEV), torch.cat(vs).to(DEV), *self.views, slots.to(torch.int32).to(DEV))
        self.qs = qs

    def run(self):
        n = len(self.lens)
        k, v, ks, vs = self.views
        return A().tree_attention(torch.cat(self.qs).to(DEV), k, v, self.table.to(DEV),
                                  torch.tensor(self.lens, dtype=torch.int32, device=DEV),
                                  torch.arange(n + 1, dtype=torch.int32, device=DEV) * self.size, self.size, self.scale,
                                  k_scale=ks, v_scale=vs)

    def expected(self, b):
        """(output, sum p |v|, weights of the first token) of sequence b, float64; drafts are chains."""
        n, t = self.lens[b], self.size
        k, v = (held_rows(self.views[i], self.views[i + 2], self.table[b], n, self.bs) for i in (0, 1))
        q = self.qs[b].double()
        g = q.shape[1] // k.shape[1]
        seen = torch.arange(n)[None] <= torch.arange(n - t, n)[:, None]
        s = torch.einsum("thgd,nhd->thgn", q.view(t, -1, g, D), k) * self.scale
        p = torch.softmax(s.masked_fill(~seen[:, None, None], -math.inf), -1)
        out, size = (torch.einsum("thgn,nhd->thgd", p, x).reshape(t, -1, D) for x in (v, v.abs()))
        return out, size, p[..., 0]

    def check(self):
        got = self.run().cpu().double()
        for b in range(len(self.lens)):
            out, size, _ = self.expected(b)
            d = (got[b * self.size:(b + 1) * self.size] - out).abs()
            assert torch.isfinite(d).all(), (b, self.lens[b])
            assert float(d.norm() / out.norm()) < 2.0 ** -8, (b, self.lens[b], float(d.norm() / out.norm()))
            assert (d <= 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -10) * size).all(), (b, self.lens[b])


# query heads, kv heads, nodes of a sequence: 1 to 33 query rows a kv head in the kernel of few rows (heads a
# unit 4, 2, 1; one and two units), then more
FEW = [(32, 8, 1), (8, 4, 6), (8, 2, 4), (8, 2, 8), (12, 2, 1), (4, 1, 4), (9, 3, 4), (8, 1, 4)]
MANY = [(8, 2, 12), (33, 1, 1), (4, 1, 40), (16, 4, 33)]
LENS = [300, 2000, 301, 130, 700, 2100, 64, 900]


def rows_and_sink(n, hq, hkv, t, size, weight, seed):
    """K, V, Q of a sequence whose first token has a zero V row and draws about `weight` of every row's attention."""
    g = gen(seed)
    k = torch.randn(n, hkv, D, generator=g) * 0.7
    v = torch.randn(n, hkv, D, generator=g) * size
    q = torch.randn(t, hq, D, generator=g) * 0.5 + 1.0
    q = q.to(torch.bfloat16)
    s = torch.einsum("thd,nhd->thn", q.double(), k.double().repeat_interleave(hq // hkv, 1)) * SCALE
    want = s[..., 1:].logsumexp(-1).mean() + math.log(weight / (1 - weight))
    k[0] = float(want) / (float(q.double().sum(-1).mean()) * SCALE)
    v[0] = 0 if seed % 2 else -0.0
    return k.to(torch.bfloat16), v.to(torch.bfloat16), q


def sinks(hq, hkv, t, weight):
    made = [rows_and_sink(n, hq, hkv, t, size, weight, 31 * i + t)
            for i, (n, size) in enumerate(zip(LENS, [1.0, 0.1, 0.02, 1e-3, 1e-5, 1e-9, 2.0 ** -60, 100.0]))]
    return Held(*zip(*made), hkv)


def far_apart(hq, hkv, t):
    """V rows 2^20 apart, then further apart than fp32 reaches; a huge row without weight; small rows among zeros."""
    g = gen(7)
    ks, vs, qs = [], [], []
    for i, n in enumerate([500, 1100, 400, 800]):
        k, v = (torch.randn(n, hkv, D, generator=g) for _ in range(2))
        q = torch.randn(t, hq, D, generator=g) + 0.5
        if i == 0:
            v[::2] *= 2.0 ** 20
        if i == 1:
            v[::2] *= 1e25
            v[1::2] *= 1e-20
        if i == 2:  # q sums to about 64 a row: a score of -35, a weight of 2^-50 times 2^40
            k[3] = -35.0 / (64 * SCALE)
            v[3] *= 2.0 ** 40
        if i == 3:
            v *= 2.0 ** -17
            v[::3] = 0
        ks.append(k.to(torch.bfloat16)), vs.append(v.to(torch.bfloat16)), qs.append(q.to(torch.bfloat16))
    return Held(ks, vs, qs, hkv, bs=128, seed=1)


def long_sink(hq, hkv, t, weight):
    return Held(*zip(*[rows_and_sink(n, hq, hkv, t, size, weight, 5 + n) for n, size in ((8000, 0.02), (20_011, 1.0), (9000, 1e-5))]),
                hkv, bs=256)


@pytest.mark.parametrize("weight", [0.5, 0.85, 0.99])
@pytest.mark.parametrize("hq,hkv,t", FEW)
def test_few_rows_with_a_zero_value_row_that_draws_the_attention(hq, hkv, t, weight):
    d = sinks(hq, hkv, t, weight)
    drawn = torch.cat([d.expected(b)[2].flatten() for b in range(len(LENS))])
    assert abs(float(drawn.mean()) - weight) < 0.15
    d.check()


@pytest.mark.parametrize("hq,hkv,t", FEW)
def test_few_rows_with_value_rows_far_apart(hq, hkv, t):
    far_apart(hq, hkv, t).check()


@pytest.mark.parametrize("hq,hkv,t", [(16, 4, 1), (8, 2, 4), (4, 1, 4)])
def test_few_rows_with_a_zero_value_row_in_a_long_context(hq, hkv, t):
    long_sink(hq, hkv, t, 0.9).check()


@pytest.mark.parametrize("weight", [0.5, 0.85, 0.99])
@pytest.mark.parametrize("hq,hkv,t", MANY)
def test_many_rows_with_a_zero_value_row_that_draws_the_attention(hq, hkv, t, weight):
    d = sinks(hq, hkv, t, weight)
    drawn = torch.cat([d.expected(b)[2].flatten() for b in range(len(LENS))])
    assert abs(float(drawn.mean()) - weight) < 0.15
    d.check()


@pytest.mark.parametrize("hq,hkv,t", MANY)
def test_many_rows_with_value_rows_far_apart(hq, hkv, t):
    far_apart(hq, hkv, t).check()


@pytest.mark.parametrize("hq,hkv,t", [(16, 1, 4), (8, 2, 12)])
def test_many_rows_with_a_zero_value_row_in_a_long_context(hq, hkv, t):
    long_sink(hq, hkv, t, 0.9).check()


@pytest.mark.parametrize("apart", [16, 32, 128, 400])
@pytest.mark.parametrize("hq,hkv,t", [*FEW, *MANY])
def test_blocks_of_value_rows_far_apart(hq, hkv, t, apart):
    """Blocks of zero or tiny rows beside blocks of large ones: the reference jumps from tile to tile, warp to warp
    and part to part, and half of the softmax's sum is under rows that add nothing."""
    g = gen(13)
    ks, vs, qs = [], [], []
    for n, low, high in ((900, 0.0, 1e12), (1300, 1e-25, 1e20), (800, 0.0, 1e25), (700, 1e25, 0.0), (1000, 1e20, 1e-25)):
        k, v = (torch.randn(n, hkv, D, generator=g) for _ in range(2))
        v *= torch.where(torch.arange(n) // apart % 2 == 0, low, high).view(n, 1, 1)
        ks.append(k.to(torch.bfloat16)), vs.append(v.to(torch.bfloat16))
        qs.append(torch.randn(t, hq, D, generator=g).to(torch.bfloat16))
    Held(ks, vs, qs, hkv, seed=2).check()


@pytest.mark.parametrize("hq,hkv,t", [(8, 2, 1), (8, 2, 4), (8, 2, 12)])
def test_queries_and_keys_at_the_ends_of_the_range(hq, hkv, t):
    """Queries up to 2^127 over keys of 2^-96, down to 2^-126 over keys of 2^118: scores of ordinary size."""
    g = gen(11)
    for q2, k2, scale in ((118, -94, 2.0 ** -29), (-118, 110, 2.0 ** 4), (126, -96, 2.0 ** -35), (-125, 118, 2.0 ** 3)):
        ks = [(torch.randn(n, hkv, D, generator=g).double() * 2.0 ** k2).to(torch.bfloat16) for n in (200, 333)]
        vs = [torch.randn(n, hkv, D, generator=g).to(torch.bfloat16) for n in (200, 333)]
        qs = [(torch.randn(t, hq, D, generator=g).double().clamp(-3, 3) * 2.0 ** q2).to(torch.bfloat16) for _ in range(2)]
        Held(ks, vs, qs, hkv, scale=scale).check()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,size", [(4, 1, 1), (8, 4, 2), (16, 2, 2), (20, 1, 2)])
def test_noise_behind_a_context_of_any_length_has_no_influence(hq, hkv, size, fp8):
    """Contexts that end at every place of a tile, over pages whose other rows hold NaN and infinities among noise."""
    lens = list(range(size, 132))
    d = Draft(lens, [size] * len(lens), hq, hkv, fp8, bs=64, seed=90)
    a, b = d.run(), d.run()
    d.check(a)
    assert torch.equal(a, b)


def test_read_back_of_the_largest_bf16_values():
    """1.9375 x 2^127 and more round to 2^128, the scale 2^120 times 256: infinity as bf16. The values below stay finite."""
    x = torch.full((3, 1, D), 1.0, dtype=torch.bfloat16)
    x[0, 0, 5], x[1, 0, 5], x[2, 0, 5] = torch.finfo(torch.bfloat16).max, -1.9375 * 2.0 ** 127, 1.9296875 * 2.0 ** 127
    views, _ = fp8_pool(1, 64, 1)
    A().store_kvcache_fp8(x.to(DEV), x.to(DEV), *views, torch.arange(3, dtype=torch.int32, device=DEV))
    k, v = A().load_kvcache_fp8(*views, torch.zeros(1, 1, dtype=torch.int32, device=DEV),
                                torch.tensor([0, 3], dtype=torch.int32, device=DEV), 3)
    assert k[:, 0, 5].tolist() == [math.inf, -math.inf, 1.875 * 2.0 ** 127] and torch.equal(k, v)
    assert (k[:, 0, :5] == 0).all()
