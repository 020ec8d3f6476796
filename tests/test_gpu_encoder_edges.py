"""The embedding encoder's operators at the edges of what their documentation allows, against 64 bits (encoder_plain.py)."""
import math

import pytest
import torch

import encoder_plain as plain

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(hip):
    from rag_service_amd import ops
    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g) * scale


# ---- attention: scores of every size -------------------------------------------------------------------------------

@pytest.mark.parametrize("lq,lk", [(1, 90), (20, 3000), (150, 700)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_of_scores_beyond_their_own_resolution(ops, dtype, lq, lk):
    """Scores so large that the next fp32 number is far away: the softmax is its largest key's value, exactly, and nothing
    overflows. The products q k are whole numbers, 3843 the largest and 1891 the second at most; the scales put the largest
    score near 2^28 and 2^34, where fp32 numbers lie 32 and 2048 apart."""
    h, d = 2, 64
    g = gen(lq)
    for power in (28, 34):
        k = torch.zeros(1, lk, h, d)
        k[..., 3] = torch.randint(-31, 32, (1, lk, h), generator=g)
        at = lk // 3
        k[0, at, :, 3] = 63
        v = rand(g, 1, lk, h, d).to(dtype)
        q = torch.zeros(1, lq, h, d)
        q[..., 3] = 61
        scale = 2.0 ** power / 3843
        got = ops.cross_attention(q.to(dtype).cuda(), k.to(dtype).cuda(), v.cuda(), scale=scale)
        assert torch.equal(got.cpu(), v[:, at:at + 1].expand(-1, lq, -1, -1))
