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


# ---- attention: one key far above the others ------------------------------------------------------------------------

@pytest.mark.parametrize("lq,lk", [(1, 100), (9, 100), (1, 4097), (30, 4097), (33, 100), (200, 1100), (130, 4097)])
@pytest.mark.parametrize("gap", [8, 12, 14, 16, 17, 18, 22])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_weights_far_below_the_largest(ops, dtype, gap, lq, lk):
    """A key whose value is zero lies `gap` nats above all others, which carry the result: their weights are as exact as
    weights near the largest, first or last among the keys. The bound is plain.attention's, half a step of each weight
    relative to it. fp16 alone has weights that it does not hold so, those below 2^-27 of the largest (18.7 nats): its steps are
    2^-24 there and a rounding 2^-25, which, the largest being at least 2^13, is 2^-38 of the largest, each times its value (below
    1.5)."""
    g = gen(gap + lq + lk)
    h, d = 2, 64
    for at in (0, lk // 2, lk - 1):
        q = torch.zeros(1, lq, h, d)
        q[..., 0] = 1
        q[..., 1:9] = rand(g, 1, lq, h, 8, scale=0.25)
        k = torch.zeros(1, lk, h, d)
        k[..., 1:9] = rand(g, 1, lk, h, 8, scale=0.25)
        k[0, at] = 0
        k[0, at, :, 0] = gap
        v = 0.5 + torch.rand(1, lk, h, d, generator=g)
        v[0, at] = 0
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
        got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
        want, err = plain.attention(q[0], k[0], v[0], torch.ones(lk, dtype=torch.bool), 1.0)
        if dtype == torch.float16:
            err = err + lk * 1.5 * 2.0 ** -38
        plain.within(got[0], want, err, dtype)


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


@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 90), (7, 128), (20, 3000), (40, 90), (150, 700)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_of_infinite_values(ops, dtype, lq, lk):
    """An infinity among the values is one in the result wherever its key takes part; both signs of it, or a NaN, are NaN. The
    other dimensions do not see it, nor do sequences whose lengths leave it out."""
    g = gen(lq + lk)
    h, d = 2, 64
    q, k, v = (rand(g, 3, n, h, d).to(dtype) for n in (lq, lk, lk))
    v2 = v.clone()
    v2[:, lk // 2, 0, 3] = float("inf")
    v2[:, lk // 3, 0, 9] = float("-inf")
    v2[:, lk // 2, 1, 17] = float("nan")
    v2[:, 0, 1, 5], v2[:, lk - 1, 1, 5] = float("inf"), float("-inf")
    lens = torch.tensor([lk, lk, 0], dtype=torch.int32)
    got = ops.cross_attention(q.cuda(), k.cuda(), v2.cuda(), key_lengths=lens.cuda()).cpu()
    assert (got[2] == 0).all()
    got, bad = got[:2], torch.zeros(h, d, dtype=torch.bool)
    assert (got[:, :, 0, 3] == float("inf")).all() and (got[:, :, 0, 9] == float("-inf")).all()
    assert got[:, :, 1, 17].isnan().all()
    assert got[:, :, 1, 5].isnan().all() if lk > 1 else (got[:, :, 1, 5] == float("-inf")).all()
    for i, j in ((0, 3), (0, 9), (1, 17), (1, 5)):
        bad[i, j] = True
    for b in range(2):
        want, err = plain.attention(q[b], k[b], v[b], torch.ones(lk, dtype=torch.bool), d ** -0.5)
        plain.within(got[b][:, ~bad], want[:, ~bad], err[:, ~bad], dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_packed_with_hints_of_nothing(ops, dtype):
    """max_q and max_k size the launch of packed sides, whatever they say: 0 as well."""
    g = gen(31)
    h, d = 4, 64
    ql, kl = [0, 1, 17, 130, 2], [5, 0, 16, 257, 600]
    qo, ko = (torch.tensor([0] + n).cumsum(0).to(torch.int32) for n in (ql, kl))
    q, k, v = (rand(g, n, h, d).to(dtype) for n in (sum(ql), sum(kl), sum(kl)))
    for max_q, max_k in ((0, 0), (0, 600), (0, 5000)):
        got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), q_offsets=qo.cuda(), k_offsets=ko.cuda(), max_q=max_q, max_k=max_k)
        for i in range(len(ql)):
            a, b, c, e = qo[i], qo[i + 1], ko[i], ko[i + 1]
            want, err = plain.attention(q[a:b], k[c:e], v[c:e], torch.ones(kl[i], dtype=torch.bool), d ** -0.5)
            plain.within(got[a:b], want, err, dtype)


# ---- 8-bit rows: the longest --------------------------------------------------------------------------------------------

def test_quantize_rows_of_the_longest_row(ops):
    """A row of 2^31 - 1 columns: every one of them is converted, the largest being the last (about five seconds)."""
    n = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of GPU memory")
    x = torch.zeros(1, n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 5000, n // 2, n - 300, n - 256, n - 2, n - 1], device="cuda")
    some = torch.tensor([3.0, -60.0, 1.0, 100.0, -7.0, 9.0, 63.0, -127.0], device="cuda")
    x[0, at] = some.to(torch.bfloat16)
    q, s = ops.quantize_rows(x)
    _, want = plain.rows8(some[None])
    assert torch.equal(s.cpu(), want)
    assert torch.equal(q[0, at].cpu(), plain.rows8(some[None])[0][0])
    q[0, at] = 0
    assert not any(bool(part.any()) for part in q[0].split(1 << 28))
    del x, q
    torch.cuda.empty_cache()


# ---- norm: gates ------------------------------------------------------------------------------------------------------

def test_block_norm_refuses_a_gate_without_rows(ops):
    """A gate of no rows for rows that need one is refused, and not taken for no gate; for no rows it is enough."""
    y, none = torch.ones(4, 16).cuda(), torch.ones(0, 16).cuda()
    for per in (1, 4, 2 ** 40):
        with pytest.raises(ValueError, match="gate"):
            ops.block_norm(y, gate=none, rows_per_gate=per)
    assert ops.block_norm(y[:0], gate=none).normed.shape == (0, 16)


# ---- the largest numbers of rows ---------------------------------------------------------------------------------------

def room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


def test_block_norm_of_four_million_wide_rows(ops):
    """2^22 rows that do not fit the registers, written in place: as many workgroups of 1024 as rows would be 2^32 threads, more
    than a launch may have."""
    from rag_service_amd import _lib
    lib, rows, cols = _lib.load_library(), 1 << 22, 16640
    room(140)
    y = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 7, 2047, 2048, rows // 2, rows - 2, rows - 1], device="cuda")
    some = rand(gen(5), len(at), cols).to(torch.bfloat16).cuda()
    y[at] = some
    rc = lib.rr_block_norm(0, torch.cuda.current_stream().cuda_stream, _lib.RR_TYPE_BF16, rows, cols, y.data_ptr(), cols, None, 0,
                           1.0, None, 0, 0, 1, _lib.RR_NORM_NONE, None, None, _lib.RR_NORM_LAYER, None, None, 1e-5, None, 0,
                           y.data_ptr(), cols, None, 0, None)
    assert rc == _lib.RR_OK, lib.rr_last_error()
    assert torch.equal(y[at], ops.block_norm(some).normed)
    y[at] = 0
    assert not any(bool(part.any()) for part in y.split(1 << 16))
    del y
    torch.cuda.empty_cache()


def test_linear_int8_of_two_billion_rows(ops):
    """As many rows as the header allows, 2^31 - 1, at any byte: every result is right."""
    m = 2 ** 31 - 1
    room(40)
    x = torch.arange(m, device="cuda", dtype=torch.int32).to(torch.int8)[:, None]
    sx = torch.full((m,), 0.37, device="cuda")
    w, sw = torch.tensor([[-3]], dtype=torch.int8).cuda(), torch.tensor([0.11]).cuda()
    got = ops.linear_int8(x, w, sw, x_scale=sx, out_dtype=torch.bfloat16)
    scale = torch.tensor(0.37) * torch.tensor(0.11)                  # the product rounded once, then the result: as the operator
    for lo in range(0, m, 1 << 27):
        want = (x[lo:lo + (1 << 27)].float() * -3 * scale.cuda()).to(torch.bfloat16)
        assert torch.equal(got[lo:lo + (1 << 27)], want)
    del x, sx, got, want
    torch.cuda.empty_cache()


# ---- attention: strides that are never taken ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq", [1, 40])
def test_attention_of_one_key_in_front_of_a_large_batch(ops, dtype, lq):
    """States of one token, the token in front of the batch: the step from key to key is a whole batch's, which no one takes. Of
    two keys it is a step too far, and refused. A result is its one value times a weight, times the weight's reciprocal: a
    rounding of 32 bits each, 3 U and their products, within 4 U."""
    from rag_service_amd import HipRetrievalError
    g = gen(lq)
    b, h, d = 1100, 64, 128                                # 9.0 million elements from key to key, above 2^23
    q = rand(g, b, lq, 1, d).to(dtype).cuda().expand(b, lq, h, d)
    kv = rand(g, 2, 1, b, h, d).to(dtype).cuda()
    k, v = kv[0].transpose(0, 1), kv[1].transpose(0, 1)

    def near(got, want):
        got, want = got[::37], want[::37]                  # (every 37th sequence, even and odd ones)
        plain.within(got, want, 4 * plain.U * want.double().cpu().abs(), dtype)

    near(ops.cross_attention(q, k, v), v.expand(b, lq, h, d))
    lens = (torch.arange(b, dtype=torch.int32) % 2).cuda()
    near(ops.cross_attention(q, k, v, key_lengths=lens), v.expand(b, lq, h, d) * lens[:, None, None, None])
    offsets = torch.tensor([0, 1], dtype=torch.int32).cuda()
    one = k[:1].squeeze(0)                                 # (1, heads, d), packed
    assert one.stride(0) > 1 << 23
    near(ops.cross_attention(q[:1], one, v[:1].squeeze(0), k_offsets=offsets, max_k=1), v[:1].expand(1, lq, h, d))
    two = kv.transpose(1, 2).reshape(2, b, h, d).transpose(0, 1)
    with pytest.raises(HipRetrievalError, match="apart"):
        ops.cross_attention(q, two, two)
