"""Token log probabilities of logits far from the ordinary range, against their
64-bit statement: finite masks and large finite values. Tolerances as in the
module the check is imported from: 2^-15 + 2^-20 of the value."""
import math

import pytest
import torch

from test_spec_ops_gpu import _lib, check_logprobs, gen  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 100_003, 20), (8, 100_003, 5), (8, 5000, 32), (200, 20_001, 0)])
def test_logprobs_of_vocabularies_masked_by_finite_values(dtype, rows, vocab, top):
    """Constrained decoding with masks of -1e9 .. -1e30: most threads see only masked entries."""
    fills = [-1e9, -4e9, -1e10, -1e12, -1e20, -1e30, -3e37, -2e8]
    x = torch.empty(rows, vocab, dtype=dtype)
    allowed = torch.randint(0, vocab, (7,), generator=gen(1))
    for i in range(rows):
        x[i] = fills[i % 8]
        x[i, allowed] = (torch.randn(7, generator=gen(2 + i)) * 3).to(dtype)
    if rows == 1:
        for f in fills:
            x[x < -1e8] = f
            check_logprobs(x, allowed[:1], top)
    else:
        tokens = allowed[torch.arange(rows) % 7].clone()
        tokens[::3] = (tokens[::3] + 1) % vocab  # masked ones
        check_logprobs(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [100_003, 3001])
def test_logprobs_of_large_finite_logits(dtype, vocab):
    x = torch.randn(12, vocab, generator=gen(3))
    for i, f in enumerate([1e7, 1e8, 1e9, 1e10, 1e12, 1e20, 1e30, 1e37]):
        x[i] *= f
    x[8], x[9] = -1e10, 1e10                    # constant rows
    x[10] = -1e30
    x[10, 2 * vocab // 3:] = -1e12              # nothing but masks, of two kinds
    x[11, 5] = 1e20
    x = x.to(dtype)
    tokens = torch.randint(0, vocab, (12,), generator=gen(4))
    tokens[:8] = x[:8].double().argmax(1)
    check_logprobs(x, tokens, 20)
    check_logprobs(x, (tokens + 17) % vocab, 0)


@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("at", [2.0 ** 26, 2.0 ** 27])
def test_logprobs_of_neighbouring_large_logits(sign, at):
    """Entries 8 apart on both sides of a large value: each still counts beside its neighbours."""
    x = sign * at + 8.0 * torch.randint(-3, 4, (5, 30_011), generator=gen(5)).float()
    x[1] = sign * at - 8.0 * torch.arange(30_011).float().clamp(max=60)
    x[2, 1000:] = sign * at - 512.0
    x[3, ::2] = -math.inf
    x[4, 77] = 0.0
    check_logprobs(x, torch.tensor([5, 0, 999, 1, 77]), 32)
