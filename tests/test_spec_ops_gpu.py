"""The quantised KV cache, tree attention and token log probabilities on the GPU
against their 64-bit statements.

Tolerances, set before the first run. Cache write and read-back: bit-exact.
Attention: the output rounds to bf16 (half a step, 2^-8 of the value); weights
round to bf16 (2^-8) or, over the e4m3 cache, to at worst 2^-8 of themselves, each a relative
error of one term, so at most 2^-8 of sum |p v| <= max |v| in the worst case
and far less in the norm; fp32 sums and the fp32 exponential add under 2^-14 at
these lengths. Checked as |out - ref| <= 2^-8 |ref| + 2^-8 max|v| everywhere and
as a relative 2-norm error below 2^-8 (two independent roundings of uniform
errors: each 2^-8 / sqrt(3) at most). Log probabilities: fp32 throughout; a sum
of n terms in at most n/512 + 32 sequential steps per lane and exponents up to
2^7 give below 2^-15 absolute plus 2^-20 relative."""
import math
import random

import pytest
import torch

import spec_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128
SCALE = D ** -0.5


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("needs CUDA")
    from kavor_b200 import _lib as L

    L.load()
    L.device_error(clear=True)
    yield
    assert L.device_error(clear=True) == 0, "a kernel raised a device-side error bit"


def A():
    from kavor_b200.layers import attention

    return attention


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ cache helpers
def fp8_pool(blocks, bs, hkv, seed=0, device=DEV):
    """Views (k, v, ks, vs) of a page pool laid out as the engine's, filled with noise bytes (NaN among them)."""
    rows, page = bs * hkv * D, 2 * bs * hkv * D + 2 * bs * hkv
    pool = torch.randint(0, 256, (blocks, page), generator=gen(seed), dtype=torch.uint8).to(device)
    f8, e8 = pool.view(torch.float8_e4m3fn), pool.view(torch.float8_e8m0fnu)
    shape, st = (blocks, bs, hkv, D), (page, hkv * D, D, 1)
    ss, sst = (blocks, hkv, bs), (page, bs, 1)
    return (f8.as_strided(shape, st, 0), f8.as_strided(shape, st, rows), e8.as_strided(ss, sst, 2 * rows),
            e8.as_strided(ss, sst, 2 * rows + bs * hkv)), pool


def u8(t):
    return t.view(torch.uint8).cpu()


def rows_with_edges(n, hkv, seed):
    x = torch.randn(n, hkv, D, generator=gen(seed)) * torch.exp2(torch.randint(-20, 20, (n, hkv, 1), generator=gen(seed + 1)).float())
    x = x.to(torch.bfloat16)
    flat = x.view(-1, D)
    edge = [torch.zeros(D), torch.full((D,), 448.0), torch.full((D,), 450.0), torch.full((D,), -0.0)]
    tiny = torch.zeros(D)
    tiny[5] = 1e-38
    inf = torch.randn(D, generator=gen(9))
    inf[3], inf[77] = math.inf, -math.inf
    nan = torch.randn(D, generator=gen(10))
    nan[0] = math.nan
    alln = torch.full((D,), math.nan)
    big = torch.full((D,), 3e38)
    ties = torch.arange(D).float() / 16 + 1  # halfway cases of the e4m3 rounding
    ties[0] = 256.0
    for i, e in enumerate(edge + [tiny, inf, nan, alln, big, ties]):
        if i < flat.shape[0]:
            flat[i] = e.to(torch.bfloat16)
    return x


def check_held(cache, scale, x, slots, bs, before_c, before_s):
    c, s = u8(cache).clone(), u8(scale).clone()
    val, e = ref.quantise(x)
    for t, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        b, o = divmod(slot, bs)
        held = c[b, o].view(torch.float8_e4m3fn).double()
        assert torch.equal(torch.isnan(held), torch.isnan(val[t]))
        assert torch.equal(torch.nan_to_num(held), torch.nan_to_num(val[t]))
        assert torch.equal(s[b, :, o].long(), e[t] + 127)
        c[b, o], s[b, :, o] = before_c[b, o], before_s[b, :, o]
    assert torch.equal(c, before_c) and torch.equal(s, before_s), "bytes outside the written slots changed"


@pytest.mark.parametrize("n,hkv,bs", [(1, 1, 256), (37, 2, 256), (300, 8, 64), (5, 3, 128)])
def test_store_fp8_holds_the_definition(n, hkv, bs):
    hq = 2 * hkv
    x, y = rows_with_edges(n, hkv, 1), rows_with_edges(n, hkv, 2).flip(0)
    qkv = torch.zeros(n, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=DEV)  # packed rows, as the model's
    k = qkv[:, hq * D:(hq + hkv) * D].view(n, hkv, D)
    v = qkv[:, (hq + hkv) * D:].view(n, hkv, D)
    k.copy_(x)
    v.copy_(y)
    blocks = -(-n // bs) + 2
    (kc, vc, ks, vs), _ = fp8_pool(blocks, bs, hkv)
    before = [u8(t).clone() for t in (kc, vc, ks, vs)]
    slots = torch.randperm(blocks * bs, generator=gen(3))[:n].to(torch.int32)
    slots[::7] = -1
    A().store_kvcache_fp8(k, v, kc, vc, ks, vs, slots.to(DEV))
    check_held(kc, ks, x, slots, bs, before[0], before[2])
    check_held(vc, vs, y, slots, bs, before[1], before[3])


def test_store_fp8_strided_heads_and_bad_slots():
    from kavor_b200 import _lib as L

    n, hkv, bs = 6, 2, 64
    big = torch.randn(n, 2 * hkv, 2 * D, generator=gen(4)).to(torch.bfloat16).to(DEV)
    k, v = big[:, ::2, :D], big[:, 1::2, D:]  # head stride 4 * D, value offset
    (kc, vc, ks, vs), pool = fp8_pool(2, bs, hkv)
    before = [u8(t).clone() for t in (kc, vc, ks, vs)]
    slots = torch.tensor([3, 127, -1, 128, -5, 64], dtype=torch.int32)  # 128 and -5 are outside
    A().store_kvcache_fp8(k, v, kc, vc, ks, vs, slots.to(DEV))
    assert L.device_error(clear=True) == 2
    slots[3] = slots[4] = -1
    check_held(kc, ks, k.cpu(), slots, bs, before[0], before[2])
    check_held(vc, vs, v.cpu(), slots, bs, before[1], before[3])


def held_rows(cache, scale, table, n, bs):
    """[n, hkv, D] float64 of a sequence's held rows (NaN codes as NaN)."""
    c, s = u8(cache), u8(scale)
    blk = table[: -(-n // bs)].long()
    val = c[blk].view(torch.float8_e4m3fn).double().flatten(0, 1)[:n]
    e = s[blk].permute(0, 2, 1).flatten(0, 1)[:n].double() - 127
    return val * torch.exp2(e).unsqueeze(-1)


def tables_for(lens, bs, seed, spare=2):
    need = [-(-n // bs) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=gen(seed)).tolist()
    width = max(max(need), 1)
    t, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, m in enumerate(need):
        t[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int32)
        at += m
    return t, sum(need) + spare


def clean_fp8(views, seed):
    """Fill an e4m3 cache with held rows: ordinary values and scales."""
    kc, vc, ks, vs = views
    for c, s, sd in ((kc, ks, seed), (vc, vs, seed + 1)):
        c.copy_((torch.randn(c.shape, generator=gen(sd)) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV))
        s.view(torch.uint8).copy_(torch.randint(117, 123, s.shape, generator=gen(sd + 7), dtype=torch.uint8).to(DEV))


@pytest.mark.parametrize("lens,hkv,bs", [([1], 1, 256), ([0, 5, 0, 300, 64, 1, 0], 2, 64), ([700, 33, 257], 8, 256),
                                         ([3] * 300, 1, 64)])
def test_load_fp8_is_exact(lens, hkv, bs):
    table, blocks = tables_for(lens, bs, 5)
    views, _ = fp8_pool(blocks, bs, hkv)
    clean_fp8(views, 20)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    total = int(cu[-1])
    k = torch.full((total + 3, hkv, D), 7.0, dtype=torch.bfloat16, device=DEV)
    v = k.clone()
    A().load_kvcache_fp8(*views, table.to(DEV), cu.to(DEV), total + 3, k_out=k, v_out=v)
    for b, n in enumerate(lens):
        for got, c, s in ((k, views[0], views[2]), (v, views[1], views[3])):
            assert torch.equal(got[cu[b]:cu[b] + n].cpu().double(), held_rows(c, s, table[b], n, bs))
    assert (k[total:] == 7).all() and (v[total:] == 7).all(), "rows behind the last sequence changed"
    k2, v2 = A().load_kvcache_fp8(*views, table.to(DEV), cu.to(DEV), total)
    assert torch.equal(k2, k[:total]) and torch.equal(v2, v[:total])


def test_store_then_load_gives_the_rounded_rows_and_bad_blocks_zeros():
    from kavor_b200 import _lib as L

    n, hkv, bs = 100, 2, 64
    x = rows_with_edges(n, hkv, 30)
    x = torch.where(torch.isfinite(x), x, torch.ones_like(x))
    table, blocks = tables_for([n], bs, 6)
    (kc, vc, ks, vs), _ = fp8_pool(blocks, bs, hkv)
    slots = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in range(n)], dtype=torch.int32)
    dx = x.to(DEV)
    A().store_kvcache_fp8(dx, dx, kc, vc, ks, vs, slots.to(DEV))
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    k, v = A().load_kvcache_fp8(kc, vc, ks, vs, table.to(DEV), cu, n)
    val, e = ref.quantise(x)
    want = val * torch.exp2(e.double()).unsqueeze(-1)
    assert torch.equal(k.cpu().double(), want) and torch.equal(v, k)
    # half an e4m3 step of the value (2^-4 of it), or of the row's smallest step, 2^-9 of the scale: the
    # scale is under top / 224, so half of that step is under top * 2^-17; the scale's floor of 2^-100
    # leaves half a step of 2^-110 to rows below it
    err = (want - x.double()).abs()
    top = x.double().abs().amax(-1, keepdim=True)
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, top * 2.0 ** -17).clamp(min=2.0 ** -110)
    worst = float((err / bound).max())
    assert worst <= 1
    table[0, 1] = blocks + 4
    k, v = A().load_kvcache_fp8(kc, vc, ks, vs, table.to(DEV), cu, n)
    assert L.device_error(clear=True) == 1
    assert torch.equal(k[:bs].cpu().double(), want[:bs]) and (k[bs:] == 0).all() and (v[bs:] == 0).all()


# ------------------------------------------------------------------ attention
def random_parents(n, r):
    return [r.randint(-1, i - 1) for i in range(n)]


class Draft:
    """A batch of drafted trees over a paged cache, with its 64-bit reference."""

    def __init__(self, lens, sizes, hq, hkv, fp8, bs=256, seed=0, chain=False, words=None, qstride=None):
        r = random.Random(seed)
        self.lens, self.sizes, self.hq, self.hkv, self.fp8, self.bs, self.chain = lens, sizes, hq, hkv, fp8, bs, chain
        self.table, blocks = tables_for(lens, bs, seed + 1)
        if fp8:
            self.views, self.pool = fp8_pool(blocks, bs, hkv, seed)  # noise (NaN) everywhere ...
            self.k, self.v, self.ks, self.vs = self.views
        else:
            raw = torch.randint(0, 1 << 16, (blocks, 2, bs, hkv, D), generator=gen(seed), dtype=torch.int32)
            self.pool = raw.to(torch.int16).view(torch.bfloat16).to(DEV)
            self.k, self.v, self.ks, self.vs = self.pool[:, 0], self.pool[:, 1], None, None
        for b, n in enumerate(lens):  # ... but in the sequences' own rows
            for t0 in range(0, n, bs):
                m = min(bs, n - t0)
                blk = int(self.table[b, t0 // bs])
                g = gen(seed * 7919 + b * 131 + t0)
                for c, s in ((self.k, self.ks), (self.v, self.vs)):
                    if fp8:
                        c[blk, :m] = (torch.randn(m, hkv, D, generator=g) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).to(DEV)
                        s.view(torch.uint8)[blk, :, :m] = torch.randint(116, 123, (hkv, m), generator=g, dtype=torch.uint8).to(DEV)
                    else:
                        c[blk, :m] = torch.randn(m, hkv, D, generator=g).to(torch.bfloat16).to(DEV)
        self.cu = torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32)
        total = int(self.cu[-1])
        self.q = (torch.randn(total, hq, D, generator=gen(seed + 3)) * 1.5).to(torch.bfloat16)
        self.qd = self.q.to(DEV)
        if qstride:  # q as a slice of wider rows
            wide = torch.zeros(total, hq + qstride, D, dtype=torch.bfloat16, device=DEV)
            wide[:, :hq] = self.qd
            self.qd = wide[:, :hq]
        self.mask = None if chain else A().build_tree_mask([random_parents(n, r) for n in sizes], words)

    def run(self, **kw):
        return A().tree_attention(self.qd, self.k, self.v, self.table.to(DEV),
                                  torch.tensor(self.lens, dtype=torch.int32, device=DEV), self.cu.to(DEV),
                                  max([*self.sizes, 0]), SCALE,
                                  tree_mask=None if self.mask is None else self.mask.to(DEV), k_scale=self.ks,
                                  v_scale=self.vs, **kw)

    def seen(self, b):
        n, t = self.lens[b], self.sizes[b]
        pos = torch.arange(n)
        rel = pos - (n - t)
        if self.chain:
            tree = rel[None] <= torch.arange(t)[:, None]
        else:
            bits = ref.mask_bits(self.mask[self.cu[b]:self.cu[b + 1]], max(t, 1))
            tree = bits[:, rel.clamp(min=0)] if t else torch.zeros(0, n, dtype=torch.bool)
        return (rel < 0)[None] | tree

    def rows(self, b):
        n = self.lens[b]
        if self.fp8:
            return (held_rows(self.k, self.ks, self.table[b], n, self.bs),
                    held_rows(self.v, self.vs, self.table[b], n, self.bs))
        blk = self.table[b, : -(-n // self.bs)].long()
        return tuple(c.cpu()[blk].flatten(0, 1)[:n].double() for c in (self.k, self.v))

    def expected(self):
        out = []
        for b in range(len(self.lens)):
            k, v = self.rows(b)
            out.append(ref.attention(self.q[self.cu[b]:self.cu[b + 1]], k, v, self.seen(b), SCALE))
        return torch.cat(out)

    def check(self, got, want=None):
        want = self.expected() if want is None else want
        got = got.cpu().double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
        fin = torch.isfinite(want)
        vmax = max([float(torch.nan_to_num(self.rows(b)[1], 0, 0, 0).abs().max()) for b in range(len(self.lens)) if self.lens[b]] or [0.0])
        d = (got - want)[fin].abs()
        assert (d <= 2.0 ** -8 * want[fin].abs() + 2.0 ** -8 * vmax).all(), float(d.max())
        if want[fin].norm() > 0:
            assert float(d.norm() / want[fin].norm()) < 2.0 ** -8


SHAPES = [
    # lens, sizes, hq, hkv, bs
    ([1], [1], 1, 1, 256),                                  # one token, its own key only
    ([300], [1], 4, 1, 256),
    ([1024, 5, 64, 65, 257], [1, 1, 1, 1, 1], 32, 8, 256),   # decode
    ([70, 8, 130], [8, 8, 3], 16, 8, 64),
    ([513, 40], [7, 16], 12, 2, 128),                        # 6 query heads per kv head: rows cross the unit
    ([200, 2300, 640], [9, 32, 20], 32, 8, 256),
    ([1000], [64], 8, 1, 256),                               # 512 rows of one kv head
    ([130, 131, 400], [33, 100, 65], 4, 2, 64),              # more than a mask word
    ([96], [96], 16, 2, 64),                                 # the draft is the whole context
    ([5000, 1, 0, 2], [3, 1, 0, 2], 16, 2, 256),             # a long one beside tiny and empty ones
    ([40, 7], [17, 1], 40, 1, 256),                          # 40 query heads on one kv head
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_tree_attention_matches_the_definition(i, chain, fp8):
    lens, sizes, hq, hkv, bs = SHAPES[i]
    d = Draft(lens, sizes, hq, hkv, fp8, bs, seed=i + 10, chain=chain)
    d.check(d.run())


@pytest.mark.parametrize("fp8", [False, True])
def test_tree_attention_long_context_is_split_and_repeats_bit_for_bit(fp8):
    d = Draft([20011, 300], [5, 2], 16, 2, fp8, seed=3)
    a, b = d.run(), d.run()
    d.check(a)
    assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("size", [1, 6, 40])
def test_tree_attention_rows_that_see_nothing_and_wide_masks(fp8, size):
    d = Draft([size, size + 3, 500], [size, size, size], 8, 2, fp8, seed=4, words=(size + 31) // 32 + 2)
    d.mask[: size // 2 + 1] = 0           # in sequence 0 nothing else is in the cache: no key at all
    d.mask[-1] = 0                        # sees the context only
    d.mask[:, (size + 31) // 32:] = -1    # bits past the draft mean nothing
    got = d.run()
    assert (got[: size // 2 + 1] == 0).all()
    d.check(got)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,size", [(4, 2, 4), (8, 1, 24)])
def test_tree_attention_ignores_what_unseen_nodes_hold(fp8, hq, hkv, size):
    """Node 2 holds NaN (and, in bf16, infinities): rows that do not see it keep their values (to the same bound:
    a tile with such a node adds its terms one by one, so the order of the sum differs), rows that do get NaN."""
    d = Draft([40 + size, 300], [size, size], hq, hkv, fp8, seed=5)
    d.mask = A().build_tree_mask([[-1] + [0] * (size - 1), [-1, 0, 1] + [0] * (size - 3)])
    bits = ref.mask_bits(d.mask, size)
    clean = d.run()
    want = d.expected()
    for b in range(2):
        pos = d.lens[b] - size + 2
        blk, off = int(d.table[b, pos // d.bs]), pos % d.bs
        if fp8:
            for c in (d.k, d.v):
                c.view(torch.uint8)[blk, off, :, ::3] = 0x7F
            d.ks.view(torch.uint8)[blk, :, off] = 254
            d.vs.view(torch.uint8)[blk, :, off] = 254
        else:
            d.k[blk, off, :, ::3] = math.nan
            d.v[blk, off, :, ::2] = math.inf
            d.v[blk, off, :, ::5] = math.nan
    got = d.run()
    sees = bits[:, 2]
    assert sees.any() and (~sees).any()
    assert torch.isnan(got.cpu()[sees].float()).any(-1).all()
    d.check(clean, want)
    d.check(torch.where(sees[:, None, None], clean.cpu(), got.cpu()), want)
    # V alone: only the dims that hold it turn
    d2 = Draft([40 + size], [size], hq, hkv, fp8, seed=6)
    d2.mask = A().build_tree_mask([[-1] + [0] * (size - 1)])
    pos = d2.lens[0] - size + 2
    blk, off = int(d2.table[0, pos // d2.bs]), pos % d2.bs
    if fp8:
        d2.v.view(torch.uint8)[blk, off, :, 1::2] = 0xFF
    else:
        d2.v[blk, off, :, 1::2] = math.nan
    got, want = d2.run(), d2.expected()
    assert torch.isnan(want[2, :, 1::2]).all() and torch.isfinite(want[2, :, ::2]).all()
    d2.check(got, want)


@pytest.mark.parametrize("fp8", [False, True])
def test_tree_attention_extreme_scores(fp8):
    """Scores of +-1e3 and queries at the ends of the bf16 range keep finite, correct weights."""
    d = Draft([400, 90], [6, 20], 8, 2, fp8, seed=8)
    d.q *= 60
    d.q[0], d.q[1] = d.q[0] * 1e-30, 0
    d.qd = d.q.to(DEV)
    # weights of scores this large move by the scores' own rounding: |s| 2^-24 sqrt(128) relative to ~1
    got, want = d.run().cpu().double(), d.expected()
    assert torch.isfinite(got).all()
    assert float((got - want).norm() / want.norm()) < 2.0 ** -8


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("size", [1, 30])
def test_tree_attention_strides_given_out_and_padded_rows(fp8, size):
    d = Draft([77, 300], [size, size], 8, 2, fp8, seed=9, qstride=3)
    total = 2 * size
    big = torch.full((total + 5, 10, D), 3.0, dtype=torch.bfloat16, device=DEV)
    qpad = torch.cat([d.q, torch.full((5, 8, D), math.nan, dtype=torch.bfloat16)]).to(DEV)
    d.qd = qpad
    d.mask = torch.cat([d.mask, torch.full((5, d.mask.shape[1]), -1, dtype=torch.int32)])
    out = d.run(out=big[:, 1:9])
    assert out.data_ptr() == big[:, 1:9].data_ptr()
    assert (big[total:] == 3).all() and (big[:, 0] == 3).all() and (big[:, 9] == 3).all()
    d.mask = d.mask[:total]
    d.check(out[:total])


@pytest.mark.parametrize("fp8", [False, True])
def test_one_node_is_decode(fp8):
    from kavor_b200 import _kernels as K

    d = Draft([1024, 700, 1, 33] * 4, [1] * 16, 32, 8, fp8, seed=11)
    got = d.run()
    lens = torch.tensor(d.lens, dtype=torch.int32, device=DEV)
    if fp8:  # the same values in a bf16 cache
        bf = [(c.float() * torch.exp2(s.view(torch.uint8).float() - 127).transpose(1, 2).unsqueeze(-1)).to(torch.bfloat16)
              for c, s in ((d.k, d.ks), (d.v, d.vs))]
    else:
        bf = [d.k, d.v]
    want = K.paged_decode_attention(d.qd, bf[0].contiguous(), bf[1].contiguous(), d.table.to(DEV), lens, SCALE)
    # two bf16 roundings of the same value and of the weights: see the module's bounds, twice
    torch.testing.assert_close(got.float(), want.float(), atol=2.0 ** -6, rtol=2.0 ** -7)


def test_tree_attention_bad_block_reads_zeros_and_bad_rows_are_skipped():
    from kavor_b200 import _lib as L

    for fp8 in (False, True):
        for size in (2, 24):
            d = Draft([300, 200], [size, size], 8, 2, fp8, bs=64, seed=12, chain=True)
            good = d.run()
            keep = d.table.clone()
            d.table[0, 1] = 99
            got = d.run()
            assert L.device_error(clear=True) == 1
            assert torch.equal(got[size:], good[size:]) and torch.isfinite(got.float()).all()
            d.table = keep
            # a context longer than its table is cut to the table
            d.lens[1] = 10_000
            d.run()
            assert L.device_error(clear=True) == 1
            d.lens[1] = 200
            # rows outside the queries: that sequence is skipped
            d.cu[2] = 2 * size + 50
            out = torch.full_like(good, 5.0)
            d.run(out=out)
            assert L.device_error(clear=True) == 32
            assert torch.equal(out[:size], good[:size]) and (out[size:] == 5).all()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("size", [1, 12])
def test_tree_attention_in_graphs_and_on_streams(fp8, size):
    """Two captured graphs replayed at once on two streams, and an eager call beside them, agree with eager results."""
    ds = [Draft([1500, 900], [size, size], 16, 2, fp8, seed=s) for s in (13, 14)]
    args = []
    for d in ds:
        args.append(dict(q=d.qd, t=d.table.to(DEV), l=torch.tensor(d.lens, dtype=torch.int32, device=DEV),
                         cu=d.cu.to(DEV), m=d.mask.to(DEV)))

    def call(d, a):
        return A().tree_attention(a["q"], d.k, d.v, a["t"], a["l"], a["cu"], size, SCALE, tree_mask=a["m"],
                                  k_scale=d.ks, v_scale=d.vs)

    eager = [call(d, a) for d, a in zip(ds, args)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for d, a in zip(ds, args):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(d, a))
        graphs.append(g)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        beside = call(ds[0], args[0])
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)
        assert torch.equal(beside, eager[0])


# ------------------------------------------------------------------ log probabilities
def check_logprobs(x, tokens, top):
    from kavor_b200.layers.sampler import token_logprobs

    got = token_logprobs(x.to(DEV) if not x.is_cuda else x, tokens.to(DEV), top_k=top)
    lp, rank, ent, ids, tlp = ref.logprobs(x.cpu(), tokens, top)
    assert torch.equal(got.ranks.cpu(), rank)
    assert torch.equal(got.top_ids.cpu(), ids)
    for a, b in ((got.logprobs, lp), (got.entropy, ent), (got.top_logprobs, tlp)):
        a = a.cpu().double()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.isinf(a), torch.isinf(b)) and torch.equal(a[torch.isinf(a)], b[torch.isinf(b)])
        fin = torch.isfinite(b)
        assert ((a - b)[fin].abs() <= 2.0 ** -15 + 2.0 ** -20 * b[fin].abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 7, 7), (3, 33, 32), (5, 1000, 0), (2, 4097, 20), (1, 151936, 20),
                                            (9, 32768, 5), (300, 5003, 1), (4, 65536, 32)])
def test_logprobs_match_the_definition(dtype, rows, vocab, top):
    x = (torch.randn(rows, vocab, generator=gen(vocab + top)) * 4).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen(1))
    tokens[0] = int(x[0].double().argmax())
    if rows > 2:
        tokens[1], tokens[2] = -1, vocab - 1
    check_logprobs(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_ties_banned_entries_and_empty_rows(dtype):
    vocab = 5000
    x = torch.randint(-3, 3, (12, vocab), generator=gen(2)).to(dtype)       # few distinct values: ties everywhere
    x[1] = 0
    x[2, ::2], x[2, 1::2] = 0.0, -0.0                                       # equal
    x[3, torch.rand(vocab, generator=gen(3)) < 0.9] = -math.inf
    x[4] = -math.inf
    x[5] = -math.inf
    x[5, 4321] = -7.0                                                       # one entry left
    x[6] = torch.arange(vocab).to(dtype)                                    # rising: every entry is a new best
    x[7] = -torch.arange(vocab).to(dtype)
    x[8] = torch.finfo(dtype).min
    x[9] = torch.finfo(dtype).max
    x[10, :], x[10, 77] = -30000.0, 30000.0
    tokens = torch.randint(0, vocab, (12,), generator=gen(4))
    tokens[5] = 4321
    tokens[3] = int((x[3] == -math.inf).nonzero()[5])
    check_logprobs(x, tokens, 32)
    check_logprobs(x, (tokens + 1) % vocab, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [1, 9])
def test_logprobs_long_rows_with_few_allowed_entries_or_many_ties(dtype, rows):
    """Masked vocabularies (constrained decoding), constant and rising rows: more entries tie for a place among the
    alternatives than any candidate list holds."""
    vocab = 100_003
    low = torch.finfo(dtype).min
    fills = [-math.inf, low, -10000.0, 0.0]
    x = torch.empty(9, vocab, dtype=dtype)
    allowed = torch.randint(0, vocab, (5,), generator=gen(7))
    for i, f in enumerate(fills):
        x[i] = f
        x[i, allowed] = torch.randn(5, generator=gen(8)).to(dtype) + 1
    x[4] = -math.inf
    x[4, ::2] = low
    x[5] = (torch.arange(vocab) / 50).to(dtype)             # rising, with ties in the 16-bit types
    x[6] = -3.0
    x[6, ::37] = 2.0                                        # thousands tie for the first places
    x[7] = torch.randn(vocab, generator=gen(9)).to(dtype)
    x[7, torch.rand(vocab, generator=gen(10)) < 0.3] = -math.inf
    x[8] = -math.inf
    x[8, -3:] = low                                         # only the lowest value is left, at the end
    if rows == 1:
        for i in range(9):
            check_logprobs(x[i:i + 1], allowed[:1], 32 if i % 2 else 3)
    else:
        check_logprobs(x, torch.randint(0, vocab, (9,), generator=gen(11)), 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_logprobs_rows_with_nan_or_inf(dtype):
    from kavor_b200.layers.sampler import token_logprobs

    vocab = 9001
    x = torch.randn(3, vocab, generator=gen(5)).to(dtype)
    x[0, 5000] = math.nan
    x[1, 8000] = math.inf
    got = token_logprobs(x.to(DEV), torch.tensor([10, 8000, 10], device=DEV), top_k=4)
    assert torch.isnan(got.logprobs[:2]).all() and torch.isnan(got.entropy[:2]).all() and torch.isnan(got.top_logprobs[:2]).all()
    assert got.top_ids[0, 0] == 5000 and got.top_ids[1, 0] == 8000 and got.ranks[1] == 0
    clean = x[0].double()
    assert got.ranks[0].item() == 1 + int((clean > clean[10]).sum()) + int((clean[:10] == clean[10]).sum())
    assert torch.isfinite(got.logprobs[2]) and torch.isfinite(got.entropy[2])


def test_logprobs_strided_rows_bad_ids_and_no_rows():
    from kavor_b200 import _lib as L
    from kavor_b200.layers.sampler import token_logprobs

    for off in (0, 1, 3):  # rows of any alignment
        wide = torch.randn(6, 3001, generator=gen(6)).to(torch.bfloat16).to(DEV)
        check_logprobs(wide[::2, off:off + 2900], torch.tensor([4, 2899, 0]), 20)
        w32 = wide.float()
        check_logprobs(w32[:, off:off + 2048], torch.arange(6), 3)
    got = token_logprobs(wide, torch.tensor([-2, 3001, 0, 1, 2, -1], device=DEV), top_k=1)
    assert L.device_error(clear=True) == 8
    assert got.ranks.tolist()[:2] == [-1, -1] and got.logprobs.tolist()[0] == 0 and got.ranks.tolist()[5] == -1
    empty = token_logprobs(wide[:0], torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert empty.top_ids.shape == (0, 2) and empty.logprobs.shape == (0,)


# ------------------------------------------------------------------ together
def test_a_verification_step_of_drafted_trees_over_the_8bit_cache():
    """Prompt rows are quantised into the cache and read back for the prompt's own attention; a tree of drafts is
    stored behind them, attended, projected to logits and scored: every stage against the 64-bit statements."""
    from kavor_b200 import _kernels as K
    from kavor_b200.layers.sampler import token_logprobs

    hq, hkv, bs, vocab = 8, 2, 64, 4096
    lens, sizes = [150, 61], [9, 5]
    r = random.Random(3)
    table, blocks = tables_for([n + t for n, t in zip(lens, sizes)], bs, 8)
    views, _ = fp8_pool(blocks, bs, hkv)
    total = sum(lens)
    k = torch.randn(total, hkv, D, generator=gen(40)).to(torch.bfloat16)
    v = torch.randn(total, hkv, D, generator=gen(41)).to(torch.bfloat16)
    q = torch.randn(total, hq, D, generator=gen(42)).to(torch.bfloat16)
    cu = torch.tensor([0, lens[0], total], dtype=torch.int32)
    slot = lambda b, p: int(table[b, p // bs]) * bs + p % bs
    slots = torch.tensor([slot(b, p) for b in range(2) for p in range(lens[b])], dtype=torch.int32)
    A().store_kvcache_fp8(k.to(DEV), v.to(DEV), *views, slots.to(DEV))
    kb, vb = A().load_kvcache_fp8(*views, table.to(DEV), cu.to(DEV), total)
    o = K.prefill_attention(q.to(DEV), kb, vb, cu.to(DEV), cu.to(DEV), max(lens), SCALE)
    held = [[c * torch.exp2(e.double()).unsqueeze(-1) for c, e in (ref.quantise(x[cu[b]:cu[b + 1]]) for x in (k, v))]
            for b in range(2)]
    for b in range(2):
        want = ref.attention(q[cu[b]:cu[b + 1]], *held[b], torch.ones(lens[b], lens[b], dtype=torch.bool).tril(), SCALE)
        assert float((o[cu[b]:cu[b + 1]].cpu().double() - want).norm() / want.norm()) < 2.0 ** -7
    # the draft
    parents = [random_parents(t, r) for t in sizes]
    nodes = sum(sizes)
    dk, dv = (torch.randn(nodes, hkv, D, generator=gen(s)).to(torch.bfloat16) for s in (43, 44))
    dq = torch.randn(nodes, hq, D, generator=gen(45)).to(torch.bfloat16)
    dcu = torch.tensor([0, sizes[0], nodes], dtype=torch.int32)
    dslots = torch.tensor([slot(b, lens[b] + i) for b in range(2) for i in range(sizes[b])], dtype=torch.int32)
    A().store_kvcache_fp8(dk.to(DEV), dv.to(DEV), *views, dslots.to(DEV))
    mask = A().build_tree_mask(parents)
    ctx = torch.tensor([n + t for n, t in zip(lens, sizes)], dtype=torch.int32)
    got = A().tree_attention(dq.to(DEV), views[0], views[1], table.to(DEV), ctx.to(DEV), dcu.to(DEV), max(sizes), SCALE,
                             tree_mask=mask.to(DEV), k_scale=views[2], v_scale=views[3])
    for b in range(2):
        rows = slice(int(dcu[b]), int(dcu[b + 1]))
        kk, vv = (torch.cat([h, c * torch.exp2(e.double()).unsqueeze(-1)])
                  for h, (c, e) in zip(held[b], (ref.quantise(x[rows]) for x in (dk, dv))))
        seen = torch.cat([torch.ones(sizes[b], lens[b], dtype=torch.bool), ref.mask_bits(mask[rows], sizes[b])], 1)
        want = ref.attention(dq[rows], kk, vv, seen, SCALE)
        assert float((got[rows].cpu().double() - want).norm() / want.norm()) < 2.0 ** -8
    w = (torch.randn(vocab, hq * D, generator=gen(46)) * 0.3).to(torch.bfloat16).to(DEV)
    logits = torch.nn.functional.linear(got.flatten(1), w)
    check_logprobs(logits, torch.randint(0, vocab, (nodes,), generator=gen(47)), 5)
    assert token_logprobs(logits, logits.argmax(1)).ranks.max() >= 0


@pytest.mark.parametrize("fp8", [False, True])
def test_a_step_as_programmatic_dependents_equals_plain_launches(fp8):
    """Every kernel reads what the one before left only after waiting for it, whichever way it is launched."""
    from kavor_b200 import _kernels as K
    from kavor_b200.layers.sampler import token_logprobs

    drafts = [Draft([700, 90, 2500], [1, 1, 1], 16, 8, fp8, seed=40), Draft([700, 90, 2500], [9, 30, 4], 32, 4, fp8, seed=41)]
    logits = torch.randn(40, 5000, generator=gen(42)).to(DEV, torch.bfloat16)
    tokens = torch.arange(40, device=DEV) * 7

    def step():
        out = []
        for _ in range(3):
            for d in drafts:
                out.append(d.run())
            out.extend(token_logprobs(logits, tokens, top_k=8))
        torch.cuda.synchronize()
        return out

    want = step()
    K.set_pdl(True)
    try:
        got = step()
    finally:
        K.set_pdl(False)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tree_attention_of_units_much_smaller_than_a_part_and_of_few_tiles():
    """More CTAs than tiles, and units of one tile beside one of thousands."""
    for lens, sizes, hq, hkv in (([1] * 300, [1] * 300, 8, 1), ([64], [1], 8, 8), ([130] * 3 + [9000], [20, 1, 2, 5], 8, 2),
                                 ([3] * 40 + [0, 5000], [2] * 40 + [0, 40], 16, 2)):
        for fp8 in (False, True):
            d = Draft(lens, sizes, hq, hkv, fp8, seed=len(lens))
            d.check(d.run())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("hq,hkv,size", [(8, 8, 8), (6, 2, 3), (9, 3, 3), (8, 4, 8), (4, 1, 4), (17, 1, 1), (16, 4, 8), (8, 2, 8),
                                         (11, 1, 3), (12, 3, 8), (33, 1, 1)])
def test_tree_attention_at_the_row_limits_of_its_kernels(hq, hkv, size, many, fp8):
    """8, 9, 12, 16, 17, 32 and 33 query rows a kv head, for few sequences and for more than the GPU has SMs."""
    n = 150 // hkv + 2 if many else 3
    rng = random.Random(hq * 100 + size)
    lens = [rng.randint(size, 700 if not many else 200) for _ in range(n)]
    sizes = [rng.randint(1, size) for _ in range(n - 1)] + [size]
    d = Draft(lens, sizes, hq, hkv, fp8, seed=hq + size)
    d.mask[0] = 0
    d.check(d.run())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv,size,n", [(8, 4, 8, 40), (4, 2, 4, 80), (8, 2, 8, 3)])
def test_tree_attention_ignores_unseen_nodes_in_every_sequence(hq, hkv, size, n, fp8):
    """16, 8 and 32 query rows a kv head: node 2 of every tree holds NaN, the others hang under node 0 and do not see it."""
    lens = [size + 13 * b % 190 for b in range(n)]
    d = Draft(lens, [size] * n, hq, hkv, fp8, seed=70)
    d.mask = A().build_tree_mask([[-1] + [0] * (size - 1)] * n)
    want = d.expected()
    for b in range(n):
        pos = lens[b] - size + 2
        blk, off = int(d.table[b, pos // d.bs]), pos % d.bs
        for c in (d.k, d.v):
            if fp8:
                c.view(torch.uint8)[blk, off] = 0x7F
            else:
                c[blk, off] = math.nan
    got = d.run().cpu()
    hit = torch.arange(n * size) % size == 2
    assert torch.isnan(got[hit].float()).all() and torch.isfinite(got[~hit].float()).all()
    err = (got.double() - want)[~hit]
    assert float(err.norm() / want[~hit].norm()) < 2.0 ** -8


@pytest.mark.parametrize("fp8", [False, True])
def test_blocks_whose_offsets_pass_32_bits(fp8):
    """The same pages at the end of a pool of more than 2^32 bytes and values give the same bytes."""
    d = Draft([600, 90, 1300], [5, 40, 1], 16, 8, fp8, seed=80)
    page = d.k.stride(0) * d.k.element_size()
    pages = 2 ** 32 * d.k.element_size() // page + 2 * d.k.shape[0]
    big = torch.empty(pages * page, dtype=torch.uint8, device=DEV)
    shift = pages - d.k.shape[0]
    big.view(pages, page)[shift:].copy_(torch.as_strided(d.k.view(torch.uint8), (d.k.shape[0], page), (page, 1)))

    def moved(t):
        flat = big.view(t.dtype)
        return flat.as_strided((pages, *t.shape[1:]), t.stride(), t.storage_offset())

    want = d.run()
    parts = [d.k, d.v, d.ks, d.vs] if fp8 else [d.k, d.v]
    new = [moved(t) for t in parts]
    table = torch.where(d.table >= 0, d.table + shift, d.table)
    d.k, d.v = new[:2]
    if fp8:
        d.ks, d.vs = new[2:]
    d.table = table
    assert torch.equal(d.run(), want)
    if fp8:
        cu = torch.tensor([0, 600], dtype=torch.int32, device=DEV)
        k, v = A().load_kvcache_fp8(*new, table[:1].to(DEV), cu, 600)
        for got, cache, scale in ((k, new[0], new[2]), (v, new[1], new[3])):
            assert torch.equal(got.cpu().double(), held_rows(cache, scale, table[0], 600, d.bs))
        rows = torch.randn(3, 8, D, generator=gen(81)).to(DEV, torch.bfloat16)
        slots = torch.tensor([pages * d.bs - 1, 5, pages * d.bs - d.bs], dtype=torch.int32, device=DEV)
        A().store_kvcache_fp8(rows, rows, *new, slots)
        low = [torch.zeros_like(t[:1]).contiguous() for t in new]
        A().store_kvcache_fp8(rows, rows, *low, torch.tensor([d.bs - 1, 5, 0], dtype=torch.int32, device=DEV))
        for at, block in ((d.bs - 1, pages - 1), (5, 0), (0, pages - 1)):
            for t, s in zip(new[:2], low[:2]):
                assert torch.equal(t[block, at].view(torch.uint8), s[0, at].view(torch.uint8))
            for t, s in zip(new[2:], low[2:]):
                assert torch.equal(t[block, :, at].view(torch.uint8), s[0, :, at].view(torch.uint8))
