"""What the speculative-serving operators refuse, and their host-side helpers (no GPU needed): bad sizes, strides,
alignments and NULL pointers give a negative status and a message before any launch; empty work succeeds."""
import ctypes

import pytest
import torch

import spec_ops_ref as ref
from kavor_b200 import _lib

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
NULL = None
FAKE = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)
HUGE = 1 << 40

PAGE, SCALES = 256 * 8 * 128, 256 * 8
STORE = dict(key=FAKE, kst=1024, ksh=128, value=FAKE, vst=1024, vsh=128, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, nblk=4,
             bst=2 * PAGE + 2 * SCALES, sst=2 * PAGE + 2 * SCALES, bs=256, hkv=8, hd=128, slots=FAKE, n=4, stream=NULL)
LOAD = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, nblk=4, bst=2 * PAGE + 2 * SCALES, sst=2 * PAGE + 2 * SCALES, bs=256, hkv=8,
            hd=128, tables=FAKE, btst=4, maxb=4, cu=FAKE, batch=2, total=10, ko=FAKE, kost=1024, vo=FAKE, vost=1024,
            stream=NULL)
TREE = dict(q=FAKE, qst=4096, qsh=128, total=10, k=FAKE, v=FAKE, ks=NULL, vs=NULL, nblk=4, bst=2 * PAGE, sst=0, bs=256,
            tables=FAKE, btst=4, maxb=4, ctx=FAKE, cu=FAKE, maxq=8, mask=FAKE, mst=1, words=1, out=FAKE, ost=4096,
            osh=128, batch=2, hq=32, hkv=8, hd=128, scale=0.088, ws=FAKE, wsn=HUGE, stream=NULL)
FP8 = dict(ks=FAKE, vs=FAKE, bst=2 * PAGE + 2 * SCALES, sst=2 * PAGE + 2 * SCALES)
LOGP = dict(x=FAKE, dtype=0, rst=1000, tok=FAKE, rows=4, vocab=1000, k=5, lp=FAKE, rank=FAKE, ent=FAKE, ids=FAKE,
            top=FAKE, stream=NULL)
BASE = {"kvb_store_kv_fp8": STORE, "kvb_load_kv_fp8": LOAD, "kvb_tree_attn": TREE, "kvb_token_logprobs": LOGP}

CASES = [
    ("kvb_store_kv_fp8", dict(n=-1), INVALID, "sizes"),
    ("kvb_store_kv_fp8", dict(hkv=0), INVALID, "sizes"),
    ("kvb_store_kv_fp8", dict(bs=0), INVALID, "sizes"),
    ("kvb_store_kv_fp8", dict(hd=64), UNSUPPORTED, "head_dim"),
    ("kvb_store_kv_fp8", dict(vs=NULL), INVALID, "NULL"),
    ("kvb_store_kv_fp8", dict(slots=NULL), INVALID, "NULL"),
    ("kvb_store_kv_fp8", dict(key=ODD), INVALID, "aligned"),
    ("kvb_store_kv_fp8", dict(vst=1028), INVALID, "aligned"),
    ("kvb_store_kv_fp8", dict(ksh=132), INVALID, "aligned"),
    ("kvb_store_kv_fp8", dict(v=ODD), INVALID, "aligned"),
    ("kvb_store_kv_fp8", dict(bst=PAGE - 16), INVALID, "block stride"),
    ("kvb_store_kv_fp8", dict(sst=SCALES - 1), INVALID, "block stride"),
    ("kvb_load_kv_fp8", dict(total=-1), INVALID, "sizes"),
    ("kvb_load_kv_fp8", dict(maxb=-1), INVALID, "sizes"),
    ("kvb_load_kv_fp8", dict(hd=256), UNSUPPORTED, "head_dim"),
    ("kvb_load_kv_fp8", dict(cu=NULL), INVALID, "NULL"),
    ("kvb_load_kv_fp8", dict(ko=ODD), INVALID, "aligned"),
    ("kvb_load_kv_fp8", dict(vost=1016), INVALID, "hold all heads"),
    ("kvb_tree_attn", dict(hq=33), INVALID, "sizes"),
    ("kvb_tree_attn", dict(nblk=0), INVALID, "sizes"),
    ("kvb_tree_attn", dict(total=1 << 31), INVALID, "sizes"),
    ("kvb_tree_attn", dict(hd=64), UNSUPPORTED, "head_dim"),
    ("kvb_tree_attn", dict(bs=32), UNSUPPORTED, "block_size"),
    ("kvb_tree_attn", dict(batch=65536), UNSUPPORTED, "sequences"),
    ("kvb_tree_attn", dict(maxb=1 << 23), UNSUPPORTED, "block tables"),
    ("kvb_tree_attn", dict(q=NULL), INVALID, "NULL"),
    ("kvb_tree_attn", dict(FP8, vs=NULL), INVALID, "NULL"),
    ("kvb_tree_attn", dict(q=ODD), INVALID, "aligned"),
    ("kvb_tree_attn", dict(osh=132), INVALID, "aligned"),
    ("kvb_tree_attn", dict(bst=PAGE - 8), INVALID, "block stride"),
    ("kvb_tree_attn", dict(FP8, sst=2 * PAGE + 2 * SCALES + 8), INVALID, "scales"),
    ("kvb_tree_attn", dict(FP8, ks=ODD), INVALID, "scales"),
    ("kvb_tree_attn", dict(words=0), INVALID, "mask"),
    ("kvb_tree_attn", dict(mst=-1), INVALID, "mask"),
    ("kvb_tree_attn", dict(scale=0.0), INVALID, "scale"),
    ("kvb_tree_attn", dict(scale=-1.0), INVALID, "scale"),
    ("kvb_tree_attn", dict(scale=float("nan")), INVALID, "scale"),
    ("kvb_tree_attn", dict(scale=float("inf")), INVALID, "scale"),
    ("kvb_tree_attn", dict(ws=NULL), WORKSPACE, "workspace"),
    ("kvb_tree_attn", dict(wsn=1024), WORKSPACE, "workspace"),
    ("kvb_tree_attn", dict(ws=ODD), INVALID, "workspace"),
    ("kvb_token_logprobs", dict(rows=-1), INVALID, "sizes"),
    ("kvb_token_logprobs", dict(vocab=0), INVALID, "sizes"),
    ("kvb_token_logprobs", dict(rst=999), INVALID, "sizes"),
    ("kvb_token_logprobs", dict(dtype=3), INVALID, "dtype"),
    ("kvb_token_logprobs", dict(k=33), UNSUPPORTED, "top_k"),
    ("kvb_token_logprobs", dict(vocab=4, k=5), UNSUPPORTED, "top_k"),
    ("kvb_token_logprobs", dict(k=-1), UNSUPPORTED, "top_k"),
    ("kvb_token_logprobs", dict(tok=NULL), INVALID, "NULL"),
    ("kvb_token_logprobs", dict(ids=NULL), INVALID, "NULL"),
    ("kvb_token_logprobs", dict(x=ctypes.c_void_p(0x1001)), INVALID, "misaligned"),
    ("kvb_token_logprobs", dict(x=ctypes.c_void_p(0x1002), dtype=2), INVALID, "misaligned"),
]


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("name,change,status,fragment", CASES, ids=[f"{c[0]}-{i}" for i, c in enumerate(CASES)])
def test_bad_arguments_are_refused_before_any_launch(lib, name, change, status, fragment):
    assert getattr(lib, name)(*{**BASE[name], **change}.values()) == status
    assert fragment in lib.kvb_last_error().decode()


@pytest.mark.parametrize("name,change", [("kvb_store_kv_fp8", dict(n=0)), ("kvb_load_kv_fp8", dict(total=0)),
                                         ("kvb_load_kv_fp8", dict(batch=0)), ("kvb_tree_attn", dict(batch=0)),
                                         ("kvb_tree_attn", dict(total=0)), ("kvb_token_logprobs", dict(rows=0))])
def test_empty_work_is_success(lib, name, change):
    assert getattr(lib, name)(*{**BASE[name], **change}.values()) == 0


def test_workspace_size(lib):
    n = ctypes.c_size_t(0)
    assert lib.kvb_tree_attn_workspace_size(4, 32, 8, 16, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.kvb_tree_attn_workspace_size(4, 33, 8, 16, ctypes.byref(n)) == INVALID
    assert lib.kvb_tree_attn_workspace_size(4, 32, 8, 16, None) == INVALID


def test_wrappers_refuse_cpu_tensors():
    from kavor_b200.layers.attention import load_kvcache_fp8, store_kvcache_fp8, tree_attention
    from kavor_b200.layers.sampler import token_logprobs

    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(1, 64, 2, 128, dtype=torch.float8_e4m3fn)
    s = torch.zeros(1, 2, 64, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: store_kvcache_fp8(x, x, c, c, s, s, i), lambda: load_kvcache_fp8(c, c, s, s, i[None], i, 1),
                 lambda: tree_attention(x, c, c, i[None], i[:1], i, 1, 0.1, k_scale=s, v_scale=s),
                 lambda: token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_build_tree_mask():
    from kavor_b200.layers.attention import build_tree_mask

    m = build_tree_mask([[-1, 0, 0, 1], [], [-1]])
    assert m.dtype == torch.int32 and m.tolist() == [[1], [3], [5], [11], [1]]
    chain = build_tree_mask([[i - 1 for i in range(70)]])
    assert chain.shape == (70, 3)
    assert torch.equal(ref.mask_bits(chain, 70), torch.ones(70, 70, dtype=torch.bool).tril())
    assert build_tree_mask([]).shape == (0, 1) and build_tree_mask([[-1]], words=4).shape == (1, 4)
    for bad in ([[0]], [[-1, 1]], [[-1, -2]]):
        with pytest.raises(ValueError, match="parent"):
            build_tree_mask(bad)
    with pytest.raises(ValueError, match="words"):
        build_tree_mask([[-1] * 33], words=1)


def test_reference_quantisation_is_the_nearest_held_value():
    """The tests' own quantisation against a search over every e4m3 value."""
    codes = torch.arange(256, dtype=torch.uint8)
    values = codes.view(torch.float8_e4m3fn).double()
    values = values[torch.isfinite(values)]
    x = torch.randn(6, ref.D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    x[1] *= 1e-4
    x[2, 0] = 448.0
    held, e = ref.quantise(x)
    for i in range(6):
        scale = 2.0 ** int(e[i])
        top = float(x[i].double().abs().max())
        assert top <= 448 * scale and top > 448 * scale / 2
        best = (x[i].double()[:, None] / scale - values).abs().amin(1)
        assert torch.equal((x[i].double() / scale - held[i]).abs(), best)
