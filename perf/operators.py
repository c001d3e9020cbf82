"""The operators of speculative serving over an 8-bit KV cache, as measured workloads.

Four operators that a serving step runs one after the other:

* ``store``: key/value rows are quantised to e4m3 with one power-of-two scale per
  (token, kv head) as they are written into the paged cache;
* ``load``: the rows of whole sequences are read back from the pages as
  contiguous bf16 rows (what a prefill over a cached prefix attends to);
* ``attention``: the nodes of a tree of drafted tokens of every sequence (a tree of
  one node is ordinary decode) attend to the sequence's cached context and to
  their own ancestors, over a bf16 or an e4m3 cache;
* ``logprobs``: log probability and rank of given tokens, the entropy of each
  row and its most likely alternatives.

``run`` computes each in plain torch operations, in 32 bits, or, where ``own``
is set, through the package. ``exact`` is each operator's definition in 64 bits.
"""
import math

import torch

own = False

HEAD_DIM = 128
BLOCK = 256          # tokens of a cache page (Config.kvcache_block_size)
E4M3_MAX = 448.0
SCALE_MIN = -100     # exponents of the power-of-two scales are clamped to this
SCALE_BIAS = 127     # a scale is held as an e8m0 byte: 2 ** (byte - 127)


# ---------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of the default benchmark batch (256 sequences, Qwen3-8B heads)
        dict(name="store_decode_256", op="store", tokens=256, hq=32, hkv=8, padded=True),
        # the largest prefill batch the engine builds (max_num_batched_tokens)
        dict(name="store_prefill_16384", op="store", tokens=16384, hq=32, hkv=8, padded=False),
        # three short prompts that continue cached prefixes, two kv heads (ERNIE-4.5-0.3B)
        dict(name="load_3_short", op="load", seqs=3, lo=65, hi=701, hkv=2),
        # 64 prompts on a shared 2048-token prefix, 8 kv heads (the shared-prefix benchmark)
        dict(name="load_64_prefix", op="load", seqs=64, lo=2112, hi=2304, hkv=8),
        # a single request drafting 8 tokens, Qwen3-0.6B heads: latency counts
        dict(name="tree_bf16_1x8", op="attention", cache="bf16", seqs=1, hq=16, hkv=8, lo=1531, hi=1531, tlo=8, thi=8),
        # a full decode batch over the 8-bit cache, one token per sequence (Qwen3-8B heads)
        dict(name="decode_fp8_256", op="attention", cache="fp8", seqs=256, hq=32, hkv=8, lo=1024, hi=1024, tlo=1, thi=1),
        # ragged drafts of 9 to 32 nodes over ragged contexts
        dict(name="tree_bf16_64_ragged", op="attention", cache="bf16", seqs=64, hq=32, hkv=8, lo=200, hi=2300, tlo=9, thi=32),
        # wide drafts of 64 nodes, Qwen3-32B heads, long contexts in the 8-bit cache
        dict(name="tree_fp8_16x64", op="attention", cache="fp8", seqs=16, hq=64, hkv=8, lo=3900, hi=8100, tlo=64, thi=64),
        # one very long context, a short chain of drafts, two kv heads of eight query heads
        dict(name="tree_fp8_long", op="attention", cache="fp8", seqs=1, hq=16, hkv=2, lo=130001, hi=130001, tlo=4, thi=4),
        # one sampled token's log probability with alternatives, 32-bit logits (Mistral vocabulary)
        dict(name="logprobs_1", op="logprobs", rows=1, vocab=32768, dtype="float32", top=20, banned=False),
        # a decode batch's sampled tokens with 20 alternatives (Qwen3 vocabulary)
        dict(name="logprobs_256", op="logprobs", rows=256, vocab=151936, dtype="bfloat16", top=20, banned=True),
        # scoring a prompt of 2000 tokens with 5 alternatives each
        dict(name="logprobs_prompt", op="logprobs", rows=2000, vocab=151936, dtype="bfloat16", top=5, banned=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 8), (32, 8), (64, 8), (16, 2), (8, 1), (4, 1), (8, 8), (2, 2), (12, 2)]


def draw(rng):
    op = rng.choice(["store", "load", "attention", "attention", "logprobs"])
    hq, hkv = rng.choice(HEADS)
    if op == "store":
        return dict(op=op, tokens=_log(rng, 1, 16384), hq=hq, hkv=hkv, padded=rng.random() < 0.5)
    if op == "load":
        hi = _log(rng, 1, 16000)
        seqs = max(1, min(_log(rng, 1, 200), 140000 // hi))
        return dict(op=op, seqs=seqs, lo=rng.randint(max(1, hi // 3), hi), hi=hi, hkv=hkv)
    if op == "attention":
        thi = rng.choice([1, 1, _log(rng, 2, 100), _log(rng, 2, 16)])
        cache = rng.choice(["bf16", "fp8"])
        # at most 0.4 GB of cached rows and 3e8 scores, as in the largest listed cases
        rows = 400_000_000 // (hkv * (4 if cache == "bf16" else 2) * HEAD_DIM)
        rows = min(rows, 300_000_000 // (thi * hq))
        hi = max(min(_log(rng, 16, 130000), rows), 2 * thi)
        seqs = max(1, min(_log(rng, 1, 256), rows // hi))
        return dict(op=op, cache=cache, seqs=seqs, hq=hq, hkv=hkv,
                    lo=rng.randint(max(thi, hi // 3), hi), hi=hi, tlo=rng.randint(1, thi), thi=thi)
    vocab = rng.choice([32768, 103424, 151936, 32000 + rng.randint(1, 4000), 151936 // 8])
    return dict(op=op, rows=max(1, min(_log(rng, 1, 4096), (300_000_000 if vocab > 60000 else 70_000_000) // vocab)), vocab=vocab,
                dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]) if vocab < 60000 else "bfloat16",
                top=rng.choice([0, 1, 5, 20, 32]), banned=rng.random() < 0.5)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly: the lengths of a ragged batch (their order is the seed's)."""
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _tree_sizes(case):
    return [min(t, c) for t, c in zip(_spread(case["tlo"], case["thi"], case["seqs"]),
                                      _spread(case["lo"], case["hi"], case["seqs"]))]


def work(case):
    d, op = HEAD_DIM, case["op"]
    if op == "store":
        n = case["tokens"] * case["hkv"]
        return {"bytes": 2 * n * (2 * d + d + 1) + 4 * case["tokens"], "flops": 4 * n * d}
    if op == "load":
        n = sum(_spread(case["lo"], case["hi"], case["seqs"])) * case["hkv"]
        return {"bytes": 2 * n * (d + 1 + 2 * d), "flops": 2 * n * d}
    if op == "attention":
        lens, sizes = _spread(case["lo"], case["hi"], case["seqs"]), _tree_sizes(case)
        row = 2 * d if case["cache"] == "bf16" else d + 1
        return {"bytes": 2 * sum(lens) * case["hkv"] * row + 4 * sum(sizes) * case["hq"] * d,
                "flops": 4 * d * case["hq"] * sum(t * c for t, c in zip(sizes, lens))}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 24 + 12 * case["top"]),
            "flops": 6 * case["rows"] * case["vocab"]}


# --------------------------------------------------------------------- inputs
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed) & 0x7FFFFFFF)


def _pages(blocks, hkv, fp8, g):
    """A page pool of one layer, as the cache pool lays it out, with its views:
    a page holds its K rows [BLOCK, hkv, 128], its V rows and, in the 8-bit
    form, the scales of each, [hkv, BLOCK] e8m0 bytes."""
    rows = BLOCK * hkv * HEAD_DIM
    if not fp8:
        pool = torch.randn(blocks, 2 * rows, generator=g, device="cuda", dtype=torch.bfloat16)
        shape, strides = (blocks, BLOCK, hkv, HEAD_DIM), (2 * rows, hkv * HEAD_DIM, HEAD_DIM, 1)
        return dict(k=pool.as_strided(shape, strides, 0), v=pool.as_strided(shape, strides, rows))
    page = 2 * rows + 2 * hkv * BLOCK
    pool = torch.empty(blocks, page, device="cuda", dtype=torch.uint8)
    # as written rows are: normal values over a scale that leaves the largest in the e4m3 range
    values = (torch.randn(blocks, 2 * rows, generator=g, device="cuda") * 100.0).clamp_(-E4M3_MAX, E4M3_MAX)
    pool[:, :2 * rows].copy_(values.to(torch.float8_e4m3fn).view(torch.uint8))
    pool[:, 2 * rows:].copy_(torch.randint(118, 123, (blocks, 2 * hkv * BLOCK), generator=g, device="cuda",
                                           dtype=torch.uint8))
    f8, e8 = pool.view(torch.float8_e4m3fn), pool.view(torch.float8_e8m0fnu)
    shape, strides = (blocks, BLOCK, hkv, HEAD_DIM), (page, hkv * HEAD_DIM, HEAD_DIM, 1)
    sshape, sstrides = (blocks, hkv, BLOCK), (page, BLOCK, 1)
    return dict(k=f8.as_strided(shape, strides, 0), v=f8.as_strided(shape, strides, rows),
                ks=e8.as_strided(sshape, sstrides, 2 * rows), vs=e8.as_strided(sshape, sstrides, 2 * rows + hkv * BLOCK))


def _tables(lens, g):
    """Block tables of sequences of these lengths over a shuffled pool (a few pages spare)."""
    need = [-(-n // BLOCK) for n in lens]
    blocks, width = sum(need) + 3, max(need)
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return blocks, torch.tensor(table, dtype=torch.int32, device="cuda")


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return at


def _random_tree(size, words, cpu):
    """A drafted tree's visibility words: node i hangs under a random earlier node (or starts a branch),
    and sees itself and its ancestors; bit j % 32 of word j // 32 stands for node j."""
    up = torch.rand(size, generator=cpu).tolist()
    seen = []
    for i in range(size):
        p = int(up[i] * (i + 1)) - 1
        seen.append((seen[p] if p >= 0 else 0) | (1 << i))
    out = []
    for bits in seen:
        for w in range(words):
            x = (bits >> (32 * w)) & 0xFFFFFFFF
            out.append(x - (1 << 32) if x >> 31 else x)
    return out


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    cpu = _gen(seed, "cpu")
    if op == "store":
        t, hkv = case["tokens"], case["hkv"]
        qkv = torch.randn(t, (case["hq"] + 2 * hkv) * HEAD_DIM, generator=g, device="cuda")
        qkv *= torch.exp2(torch.randint(-3, 4, (t, 1), generator=g, device="cuda").float())
        qkv = qkv.to(torch.bfloat16)  # k and v are views of the packed projection rows, as in the model
        q, k, v = qkv.split([case["hq"] * HEAD_DIM, hkv * HEAD_DIM, hkv * HEAD_DIM], dim=-1)
        blocks = -(-t // BLOCK) + 2
        slots = torch.randperm(blocks * BLOCK, generator=g, device="cuda")[:t].to(torch.int32)
        if case["padded"]:
            slots[torch.rand(t, generator=g, device="cuda") < 0.1] = -1  # rows that pad a captured batch
        return dict(case=case, key=k.view(t, hkv, HEAD_DIM), value=v.view(t, hkv, HEAD_DIM), slots=slots,
                    **_pages(blocks, hkv, True, g))
    if op == "load":
        lens = _spread(case["lo"], case["hi"], case["seqs"])
        lens = [lens[i] for i in torch.randperm(len(lens), generator=cpu).tolist()]
        blocks, table = _tables(lens, g)
        return dict(case=case, tables=table, cu=_int32(_starts(lens)), total=sum(lens),
                    **_pages(blocks, case["hkv"], True, g))
    if op == "attention":
        lens, sizes = _spread(case["lo"], case["hi"], case["seqs"]), _tree_sizes(case)
        order = torch.randperm(len(lens), generator=cpu).tolist()
        lens, sizes = [lens[i] for i in order], [sizes[i] for i in order]
        blocks, table = _tables(lens, g)
        words = -(-max(sizes) // 32)
        mask = []
        for n in sizes:
            mask += _random_tree(n, words, cpu)
        q = torch.randn(sum(sizes), case["hq"], HEAD_DIM, generator=g, device="cuda") * 1.5
        return dict(case=case, q=q.to(torch.bfloat16), tables=table, lens=_int32(lens), cu=_int32(_starts(sizes)),
                    most=max(sizes), mask=_int32(mask).view(-1, words), **_pages(blocks, case["hkv"], case["cache"] == "fp8", g))
    rows, vocab = case["rows"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    logits = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    for at in range(0, rows, 256):
        part = torch.randn(min(256, rows - at), vocab, generator=g, device="cuda").mul_(2.5)
        part.scatter_add_(1, torch.randint(0, vocab, (part.shape[0], 8), generator=g, device="cuda"),
                          torch.rand(part.shape[0], 8, generator=g, device="cuda") * 12)
        if case["banned"]:
            part[:, torch.rand(vocab, generator=g, device="cuda") < 0.1] = -math.inf
        logits[at:at + 256] = part.to(dtype)
    # what a sampler picks: mostly likely tokens, some from anywhere
    likely = torch.stack([logits[i].float().topk(16).indices for i in range(rows)]) if rows <= 64 else \
        torch.cat([c.float().topk(16).indices for c in logits.split(64)])
    pick = torch.randint(0, 16, (rows, 1), generator=g, device="cuda")
    tokens = likely.gather(1, pick).view(-1)
    anywhere = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.3, anywhere, tokens)
    return dict(case=case, logits=logits, tokens=tokens)


# ---------------------------------------------------------------- plain forms
def _power(e):
    """2 ** e in 32 bits, exactly, for whole numbers e of the normal range."""
    return ((e.to(torch.int32) + SCALE_BIAS) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 values and the exponent of the power-of-two scale of each row of 128: the smallest scale that
    keeps the row's largest finite magnitude within the e4m3 range."""
    x = x.float()
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    mantissa, power = torch.frexp(top)  # top = mantissa * 2 ** power, mantissa in [0.5, 1); 448 = 0.875 * 2 ** 9
    e = torch.where(mantissa > 0.875, power - 8, power - 9)
    e = torch.where(top == 0, 0, e.clamp(min=SCALE_MIN))
    y = (x * _power(-e).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX)
    return y.to(torch.float8_e4m3fn), e


def _plain_store(s):
    kept = (s["slots"] >= 0).nonzero().view(-1)
    slots = s["slots"][kept].long()
    block, at = slots // BLOCK, slots % BLOCK
    for x, cache, scale in ((s["key"], s["k"], s["ks"]), (s["value"], s["v"], s["vs"])):
        y, e = _quantise(x[kept])
        cache.view(torch.uint8)[block, at] = y.view(torch.uint8)
        scale.view(torch.uint8)[block, :, at] = (e + SCALE_BIAS).to(torch.uint8)
    return dict(k=s["k"], v=s["v"], ks=s["ks"], vs=s["vs"])


def _scales(e8m0):
    return _power(e8m0.view(torch.uint8).to(torch.int32) - SCALE_BIAS)


def _plain_load(s):
    at = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["cu"][1:].long(), at, right=True)
    pos = at - s["cu"][seq]
    block, off = s["tables"][seq, pos // BLOCK].long(), pos % BLOCK

    def rows(cache, scale):
        x = cache.view(torch.uint8)[block, off].view(torch.float8_e4m3fn).float()
        return (x * _scales(scale)[block, :, off].unsqueeze(-1)).to(torch.bfloat16)

    return dict(k=rows(s["k"], s["ks"]), v=rows(s["v"], s["vs"]))


def _plain_attention(s):
    case, q, dev = s["case"], s["q"], s["q"].device
    hq, hkv = case["hq"], case["hkv"]
    n, most, group = s["lens"].numel(), s["most"], hq // hkv
    tables = s["tables"].long().clamp(min=0)
    width = tables.shape[1] * BLOCK
    start, sizes = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    row = torch.arange(q.shape[0], device=dev)
    seq = torch.searchsorted(s["cu"][1:].long(), row, right=True)
    node = row - start[seq]
    padded = (start[:, None] + torch.arange(most, device=dev)).clamp(max=q.shape[0] - 1)

    def keys(cache, scale):
        if scale is None:
            x = cache[tables].float()
        else:
            x = cache.view(torch.uint8)[tables].view(torch.float8_e4m3fn).float()
            x = x * _scales(scale)[tables].transpose(2, 3).unsqueeze(-1)
        return x.reshape(n, width, hkv, HEAD_DIM).permute(0, 2, 1, 3)

    qp = q[padded].float().view(n, most, hkv, group, HEAD_DIM).permute(0, 2, 1, 3, 4)
    scores = qp.reshape(n, hkv, most * group, HEAD_DIM) @ keys(s["k"], s.get("ks")).transpose(2, 3)
    scores = scores.view(n, hkv, most, group, width) * HEAD_DIM ** -0.5
    pos = torch.arange(width, device=dev)
    lens = s["lens"].long()
    rel = pos[None] - (lens - sizes)[:, None]  # index among the drafted nodes, negative in the context
    word = (rel.clamp(min=0) // 32).clamp(max=s["mask"].shape[1] - 1)
    bits = s["mask"][padded].long().gather(2, word[:, None].expand(n, most, width))
    seen = ((bits >> (rel.clamp(min=0) % 32)[:, None]) & 1).bool() | (rel < 0)[:, None]
    seen = seen & (pos[None] < lens[:, None])[:, None]
    scores = torch.where(seen[:, None, :, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = p.view(n, hkv, most * group, width) @ keys(s["v"], s.get("vs"))
    out = out.view(n, hkv, most, group, HEAD_DIM).permute(0, 2, 1, 3, 4).reshape(n, most, hq, HEAD_DIM)
    return out[seq, node].to(torch.bfloat16)


def _plain_logprobs(s):
    x, tokens, top = s["logits"].float(), s["tokens"], s["case"]["top"]
    vocab = x.shape[1]
    high = x.amax(1, keepdim=True)
    z = x - high
    p = torch.exp(z)
    total = p.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse.view(-1) - torch.where(p > 0, p * z, 0.0).sum(1) / total.view(-1)
    logprob = (z.gather(1, tokens[:, None]) - lse).view(-1)
    # order by value, then by lowest index: one whole number per entry
    i = (x + 0.0).view(torch.int32)
    key = (torch.where(i < 0, -(i & 0x7FFFFFFF), i).long() << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
    rank = (key > key.gather(1, tokens[:, None])).sum(1)
    out = dict(logprob=logprob, rank=rank, entropy=entropy)
    if top:
        best = vocab - 1 - (key.topk(top, 1).values & 0xFFFFFFFF)
        out["top_ids"] = best
        out["top_logprobs"] = z.gather(1, best) - lse
    return out


# ------------------------------------------------------------------------ run
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"store": _plain_store, "load": _plain_load, "attention": _plain_attention,
                "logprobs": _plain_logprobs}[op](state)
    if op == "store":
        from kavor_b200.layers.attention import store_kvcache_fp8

        store_kvcache_fp8(state["key"], state["value"], state["k"], state["v"], state["ks"], state["vs"],
                          state["slots"])
        return dict(k=state["k"], v=state["v"], ks=state["ks"], vs=state["vs"])
    if op == "load":
        from kavor_b200.layers.attention import load_kvcache_fp8

        k, v = load_kvcache_fp8(state["k"], state["v"], state["ks"], state["vs"], state["tables"], state["cu"],
                                state["total"])
        return dict(k=k, v=v)
    if op == "attention":
        from kavor_b200.layers.attention import tree_attention

        return tree_attention(state["q"], state["k"], state["v"], state["tables"], state["lens"], state["cu"],
                              state["most"], HEAD_DIM ** -0.5, tree_mask=state["mask"], k_scale=state.get("ks"),
                              v_scale=state.get("vs"))
    from kavor_b200.layers.sampler import token_logprobs

    got = token_logprobs(state["logits"], state["tokens"], top_k=state["case"]["top"])
    out = dict(logprob=got.logprobs, rank=got.ranks, entropy=got.entropy)
    if state["case"]["top"]:
        out["top_ids"], out["top_logprobs"] = got.top_ids, got.top_logprobs
    return out


# ---------------------------------------------------------------------- exact
def _two_to(e):
    """2 ** e in 64 bits for whole numbers e."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "load":
        return _exact_load(s)
    return _exact_store(s)


def _exact_store(s):
    """The pool's values after the write: e4m3 has 3 mantissa bits down to 2 ** -6 and steps of 2 ** -9 below."""
    kept = (s["slots"] >= 0).nonzero().view(-1)
    block, at = s["slots"][kept].long() // BLOCK, s["slots"][kept].long() % BLOCK
    out = {}
    for name, x in (("k", s["key"]), ("v", s["value"])):
        x = x[kept].double()
        top = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / E4M3_MAX))  # within one of the border, then put right
        e = torch.where(top > E4M3_MAX * _two_to(e), e + 1, torch.where(top <= E4M3_MAX * _two_to(e - 1), e - 1, e))
        e = torch.where(top == 0, 0.0, e.clamp(min=SCALE_MIN))
        y = x / _two_to(e)
        step = _two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6)).exponent - 4)
        pool = s[name].view(torch.uint8).view(torch.float8_e4m3fn).double()
        pool[block, at] = torch.round(y / step) * step
        scale = _two_to(s[name + "s"].view(torch.uint8).int() - SCALE_BIAS)
        scale[block, :, at] = _two_to(e[..., 0])
        out[name], out[name + "s"] = pool, scale
    return out


def _exact_rows(cache, scale, blocks, length):
    """[length, hkv, 128] float64 values of a sequence's cached rows."""
    pages = cache.view(torch.uint8)[blocks].view(torch.float8_e4m3fn) if scale is not None else cache[blocks]
    x = pages.double().flatten(0, 1)[:length]
    if scale is not None:
        e = scale.view(torch.uint8)[blocks].int().permute(0, 2, 1).flatten(0, 1)[:length]
        x = x * _two_to(e - SCALE_BIAS)[..., None]
    return x


def _exact_load(s):
    at, k, v = s["cu"].tolist(), [], []
    for b in range(len(at) - 1):
        n = at[b + 1] - at[b]
        blocks = s["tables"][b, :-(-n // BLOCK)].long()
        k.append(_exact_rows(s["k"], s["ks"], blocks, n))
        v.append(_exact_rows(s["v"], s["vs"], blocks, n))
    return dict(k=torch.cat(k), v=torch.cat(v))


def _exact_attention(s):
    hkv, at, lens = s["case"]["hkv"], s["cu"].tolist(), s["lens"].tolist()
    out = []
    for b, n in enumerate(lens):
        t = at[b + 1] - at[b]
        blocks = s["tables"][b, :-(-n // BLOCK)].long()
        k, v = _exact_rows(s["k"], s.get("ks"), blocks, n), _exact_rows(s["v"], s.get("vs"), blocks, n)
        q = s["q"][at[b]:at[b + 1]].double()
        words = s["mask"][at[b]:at[b + 1]].long()
        j = torch.arange(t, device="cuda")
        tree = (words[:, j // 32] >> (j % 32)) & 1 == 1
        seen = torch.cat([torch.ones(t, n - t, dtype=torch.bool, device="cuda"), tree], 1)
        group = q.shape[1] // hkv
        heads = []
        for h in range(hkv):
            x = torch.einsum("tgd,nd->tgn", q[:, h * group:(h + 1) * group], k[:, h]) / math.sqrt(HEAD_DIM)
            x = x.masked_fill(~seen[:, None], -math.inf)
            heads.append(torch.einsum("tgn,nd->tgd", torch.softmax(x, -1), v[:, h]))
        out.append(torch.cat(heads, 1))
    return torch.cat(out)


def _exact_logprobs(s):
    top, parts = s["case"]["top"], []
    for x, tokens in zip(s["logits"].split(128), s["tokens"].split(128)):
        lp = torch.log_softmax(x.double(), 1)
        p = lp.exp()
        mine = x.double().gather(1, tokens[:, None])
        index = torch.arange(x.shape[1], device="cuda")
        ahead = (x.double() > mine) | ((x.double() == mine) & (index < tokens[:, None]))
        part = dict(logprob=lp.gather(1, tokens[:, None]).view(-1), rank=ahead.sum(1),
                    entropy=-torch.where(p > 0, p * lp, 0.0).sum(1))
        if top:
            part["top_ids"] = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
            part["top_logprobs"] = lp.gather(1, part["top_ids"])
        parts.append(part)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
