"""The embedding encoder's operators (rag_service_amd.ops) against their definitions in 64 bits (encoder_plain.py)."""
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


# ---- 8-bit rows -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 1024), (65, 1000), (33, 4096), (300, 130), (2, 20011)])
def test_quantize_rows(ops, dtype, rows, cols):
    x = rand(gen(rows * 7 + cols), rows, cols, scale=3.0).to(dtype)
    q, s = ops.quantize_rows(x.cuda())
    wq, ws = plain.rows8(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq)


def test_quantize_rows_special_values(ops):
    x = torch.zeros(9, 37)
    x[1, 5] = float("nan")
    x[2, 36] = float("inf")
    x[3, 0] = float("-inf")
    x[4] = 1e-45                       # the smallest subnormal: its scale underflows to 0
    x[5] = torch.linspace(-3.4e38, 3.4e38, 37)
    x[6] = 2.0 ** -140                 # a subnormal scale
    x[7, 3] = -127.0
    x[7, 4:8] = torch.tensor([0.5, 1.5, -2.5, 126.5])      # halves go to the even neighbour
    x[8] = -0.0
    q, s = ops.quantize_rows(x.cuda())
    wq, ws = plain.rows8(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(ws))
    assert torch.equal(torch.nan_to_num(s.cpu()), torch.nan_to_num(ws))
    assert torch.equal(q.cpu(), wq)


def test_quantize_rows_strided_and_shaped(ops):
    base = rand(gen(1), 4, 6, 50).cuda()
    x = base[:, 1:5, 3:40].contiguous().view(4, 4, 37)
    part = base.view(24, 50)[::2, 5:31]                    # every other row, an odd start
    for t in (x, part):
        q, s = ops.quantize_rows(t)
        wq, ws = plain.rows8(t)
        assert q.shape == t.shape and s.shape == t.shape[:-1]
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


# ---- the 8-bit product ----------------------------------------------------------------------------------------------

def weights(g, n, k):
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return w, (0.5 + torch.rand(n, generator=g)) / (64 * math.sqrt(k)), rand(g, n, scale=0.2)


SIZES = [(1, 1, 1), (1, 1024, 4096), (1, 1024, 1024), (2, 777, 1000), (5, 64, 17), (16, 1024, 1024), (17, 130, 4096),
         (31, 33, 65), (32, 1024, 2048), (48, 256, 512), (64, 2048, 1024), (65, 1000, 1000), (100, 96, 100), (129, 257, 128),
         (200, 1024, 1024), (257, 255, 192), (613, 1024, 256), (300, 640, 4096), (1031, 777, 1000), (1500, 1024, 128)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_int8_float_rows(ops, dtype, m, n, k, act):
    g = gen(m + 3 * n + 5 * k)
    x = rand(g, m, k, scale=2.0).to(dtype)
    w, sw, b = weights(g, n, k)
    got = ops.linear_int8(x.cuda(), w.cuda(), sw.cuda(), bias=b.cuda(), act=act)
    assert got.dtype == dtype and got.shape == (m, n)
    q, sx = plain.rows8(x)
    want, tol = plain.linear(q, sx, w, sw, b, act, dtype)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("out", TYPES, ids=str)
def test_linear_int8_rows(ops, out, m, n, k):
    g = gen(m + 5 * n + 3 * k)
    q = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
    sx = 0.01 + torch.rand(m, generator=g)
    w, sw, _ = weights(g, n, k)
    got = ops.linear_int8(q.cuda(), w.cuda(), sw.cuda(), x_scale=sx.cuda(), out_dtype=out)
    want, tol = plain.linear(q, sx, w, sw, None, "none", out)
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", [(1500, 1100, 144), (1300, 1290, 16), (1290, 1281, 1040), (1411, 1024, 272), (3600, 3400, 208),
                                   (3585, 3333, 128), (4000, 3700, 32), (2600, 5000, 656), (2000, 1900, 144), (1000, 2300, 400),
                                   (1900, 2000, 16)])
@pytest.mark.parametrize("out", TYPES, ids=str)
def test_linear_int8_many_tiles(ops, out, m, n, k):
    """Sizes of many tiles whose last rows, channels and inner columns fill none."""
    g = gen(m + n + k)
    q = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8).cuda()
    sx = (0.01 + torch.rand(m, generator=g)).cuda()
    w, sw, b = (t.cuda() for t in weights(g, n, k))
    for bias, act in ((None, "none"), (b, "gelu")):
        got = ops.linear_int8(q, w, sw, x_scale=sx, out_dtype=out, bias=bias, act=act)
        want, tol = plain.linear(q, sx, w, sw, bias, act, out)
        assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("k", [1, 15, 17, 127, 129, 250, 257, 300, 385, 399, 513, 600, 650, 777, 1027, 1300, 2049])
def test_linear_int8_inner_sizes(ops, k):
    """Inner sizes that end anywhere in a step, rows at any byte."""
    g = gen(k)
    for m, n in ((70, 65), (3, 20)):
        q = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8)
        w, sw, _ = weights(g, n, k)
        sx = 0.01 + torch.rand(m, generator=g)
        got = ops.linear_int8(q.cuda(), w.cuda(), sw.cuda(), x_scale=sx.cuda())
        want, tol = plain.linear(q, sx, w, sw, None, "none", torch.float32)
        assert ((got.double().cpu() - want).abs() <= tol).all()
        x = rand(g, m, k).to(torch.bfloat16)
        got = ops.linear_int8(x.cuda(), w.cuda(), sw.cuda())
        q8, s8 = plain.rows8(x)
        want, tol = plain.linear(q8, s8, w, sw, None, "none", torch.bfloat16)
        assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("m,n,k", [(49, 5000, 9001), (700, 4000, 777), (2100, 1024, 1001), (5000, 3001, 150), (70000, 70, 447),
                                   (16000, 15000, 9), (800, 900, 3001)])
def test_linear_int8_odd_inner_sizes_of_many_products(ops, m, n, k):
    """The sizes at which rows and weights are copied for the tiled product, rows at any byte, and those just below."""
    g = gen(m + n + k)
    q = torch.randint(-128, 128, (m, k + 5), generator=g, dtype=torch.int8).cuda()[:, 3:3 + k]
    w = torch.randint(-128, 128, (n, k + 1), generator=g, dtype=torch.int8).cuda()[:, :k]
    sx, (_, sw, b) = (0.01 + torch.rand(m, generator=g)).cuda(), weights(g, n, 1)
    sw, b = sw.cuda(), b.cuda()
    rows = torch.unique(torch.cat([torch.arange(3), torch.randint(0, m, (40,), generator=g), torch.arange(m - 3, m)]))
    got = ops.linear_int8(q, w, sw, x_scale=sx, bias=b, act="gelu")
    want, tol = plain.linear(q[rows.cuda()], sx[rows.cuda()], w, sw, b, "gelu", torch.float32)
    assert ((got[rows.cuda()].double().cpu() - want).abs() <= tol).all()
    # the rows among others, in other kernels (up to 48 rows, and any size): every result is the same to the bit
    for few in (48, 64):
        assert torch.equal(got[:few], ops.linear_int8(q[:few], w, sw, x_scale=sx[:few], bias=b, act="gelu"))
    x = rand(g, m, k).to(torch.bfloat16).cuda()
    got = ops.linear_int8(x, w, sw)
    q8, s8 = ops.quantize_rows(x)
    assert torch.equal(got, ops.linear_int8(q8, w, sw, x_scale=s8, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("m,n,k", [(70, 65, 4), (70, 65, 132), (613, 700, 1000), (1300, 1290, 20), (1500, 1100, 148), (2600, 5000, 260),
                                   (1000, 2300, 404), (3600, 3400, 636), (16000, 3100, 1028), (4001, 4090, 516), (900, 300, 2044)])
def test_linear_int8_rows_at_dwords(ops, m, n, k):
    """Inner sizes that end inside a 16-byte column, in every tile: what lies between the rows is no part of them."""
    g = gen(m + n + k)
    q = torch.randint(-128, 128, (m + 1, k + 8), generator=g, dtype=torch.int8).cuda()[:m, 4:4 + k]
    w = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    sx, (_, sw, b) = (0.01 + torch.rand(m, generator=g)).cuda(), weights(g, n, 1)
    sw, b = sw.cuda(), b.cuda()
    rows = torch.unique(torch.cat([torch.arange(3), torch.randint(0, m, (60,), generator=g), torch.arange(m - 3, m)])).cuda()
    for out in (torch.float32, torch.bfloat16):
        got = ops.linear_int8(q, w, sw, x_scale=sx, bias=b, out_dtype=out)
        want, tol = plain.linear(q[rows], sx[rows], w, sw, b, "none", out)
        assert ((got[rows].double().cpu() - want).abs() <= tol).all()
    wide = torch.zeros(n, k + 13, dtype=torch.int8).cuda()      # the same at odd bytes, in the other kernels
    wide[:, 1:k + 1] = w
    assert torch.equal(ops.linear_int8(q, wide[:, 1:k + 1], sw, x_scale=sx, bias=b, out_dtype=torch.bfloat16), got)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_int8_extremes(ops, m):
    """The longest inner size with every product at its largest: the 32-bit sum must still be exact. -128 is a valid value."""
    k, n = 131071, 40
    q = torch.full((m, k), -128, dtype=torch.int8)
    w = torch.full((n, k), -128, dtype=torch.int8)
    w[1] = 127
    one = torch.ones(max(m, n))
    got = ops.linear_int8(q.cuda(), w.cuda(), one[:n].cuda(), x_scale=one[:m].cuda())
    want = torch.full((m, n), 128 * 128 * k, dtype=torch.float64)
    want[:, 1] = -128 * 127 * k
    assert ((got.double().cpu() - want).abs() <= 2.0 ** -24 * want.abs()).all()


def test_linear_int8_strides_and_alignment(ops):
    g = gen(5)
    for m, n, k, off in [(70, 130, 256, 1), (3, 50, 64, 5), (300, 256, 512, 16), (1, 64, 1024, 3)]:
        xs = torch.randint(-127, 128, (m, k + 37), generator=g, dtype=torch.int8).cuda()
        ws = torch.randint(-127, 128, (n, k + 19), generator=g, dtype=torch.int8).cuda()
        x, w = xs[:, off:off + k], ws[:, off:off + k]
        sx, sw = torch.rand(m, generator=g), torch.rand(n, generator=g)
        got = ops.linear_int8(x, w, sw.cuda(), x_scale=sx.cuda())
        want, tol = plain.linear(x, sx, w, sw, None, "none", torch.float32)
        assert ((got.double().cpu() - want).abs() <= tol).all()
        xf = rand(g, m, k + 9).to(torch.bfloat16).cuda()[:, 1:k + 1]
        got = ops.linear_int8(xf, w, sw.cuda())
        q, sx = plain.rows8(xf)
        want, tol = plain.linear(q, sx, w, sw, None, "none", torch.bfloat16)
        assert ((got.double().cpu() - want).abs() <= tol).all()


def test_linear_int8_bad_rows_stay_in_their_rows(ops):
    g = gen(8)
    for m in (4, 80):
        x = rand(g, m, 96)
        x[1, 95] = float("nan")
        x[2, 0] = float("inf")
        x[3] = 0
        w, sw, b = weights(g, 33, 96)
        got = ops.linear_int8(x.cuda(), w.cuda(), sw.cuda(), bias=b.cuda()).cpu()
        assert got[1].isnan().all() and got[2].isnan().all()
        assert torch.equal(got[3], b)
        q, sx = plain.rows8(x)
        want, tol = plain.linear(q, sx, w, sw, b, "none", torch.float32)
        keep = [i for i in range(m) if i not in (1, 2)]
        assert ((got[keep].double() - want[keep]).abs() <= tol[keep]).all()


def test_linear_int8_empty(ops):
    w, sw, _ = weights(gen(1), 8, 16)
    assert ops.linear_int8(torch.zeros(0, 16).cuda(), w.cuda(), sw.cuda()).shape == (0, 8)
    assert ops.linear_int8(torch.zeros(2, 0, 16).cuda(), w.cuda(), sw.cuda()).shape == (2, 0, 8)


# ---- block norm -----------------------------------------------------------------------------------------------------

def norm_case(ops, dtype, rows, cols, post, nxt, gate_rows, rs, residual=True, weighted=True, rows8=False, seed=0):
    g = gen(rows + 11 * cols + seed)
    y, x = rand(g, rows, cols).to(dtype), rand(g, rows, cols, scale=2.0).to(dtype) if residual else None
    gate = rand(g, gate_rows, cols, scale=0.5).to(dtype) if gate_rows else None
    per = -(-rows // gate_rows) if gate_rows else 1
    vec = {}
    for which, kind in (("post", post), ("next", nxt)):
        vec[which + "_weight"] = (1 + rand(g, cols, scale=0.1)).to(dtype) if weighted and kind != "none" else None
        vec[which + "_bias"] = rand(g, cols, scale=0.1).to(dtype) if weighted and kind == "layer" else None
    to = lambda t: None if t is None else t.cuda()  # noqa: E731
    r = ops.block_norm(to(y), to(x), residual_scale=rs, gate=to(gate), rows_per_gate=per, post_norm=post, next_norm=nxt,
                       eps=1e-5, rows8=rows8, **{k: to(v) for k, v in vec.items()})
    want = plain.block_norm(y, x, rs, gate, per, post, vec["post_weight"], vec["post_bias"], nxt, vec["next_weight"],
                            vec["next_bias"], 1e-5)
    plain.within(r.stream, *want["stream"], dtype)
    if nxt == "none":
        assert r.normed is None and r.rows8 is None
        return
    plain.within(r.normed, *want["normed"], dtype)
    if rows8:
        o, e = want["normed"]
        s = r.scale.double().cpu()
        amax, worst = o.abs().amax(-1), e.amax(-1) * (1 + 2 ** -6)
        assert ((s * 127 - amax).abs() <= worst + 4 * plain.U * amax).all()
        # a value is its own within half a step of the scale, and what the fp32 value was off
        off = (r.rows8.double().cpu() * s[:, None] - o).abs()
        assert (off <= s[:, None] * (0.5 + 2 ** -12) + worst[:, None] * 2).all()
        assert (r.rows8.abs().amax(-1) == 127).all()


COLS = [1, 2, 63, 64, 65, 255, 256, 500, 768, 1000, 1001, 1024, 1537, 2048, 3000, 4096, 5000, 8192, 12345]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_block_norm_widths(ops, dtype, cols):
    norm_case(ops, dtype, 5, cols, "none", "layer", 0, 1.0, rows8=cols > 2)
    norm_case(ops, dtype, 3, cols, "rms", "rms", 2, 0.5, rows8=cols > 2)


@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("nxt", ["none", "layer", "rms"])
@pytest.mark.parametrize("gate_rows", [0, 1, 4])
def test_block_norm_forms(ops, post, nxt, gate_rows):
    for dtype in TYPES:
        for residual in (True, False):
            for weighted in (True, False):
                norm_case(ops, dtype, 13, 200, post, nxt, gate_rows, 0.7, residual, weighted, rows8=nxt != "none")


@pytest.mark.parametrize("rows", [1, 2, 7, 300, 5000])
def test_block_norm_rows(ops, rows):
    norm_case(ops, torch.bfloat16, rows, 1024, "none", "layer", 0, 1.0, rows8=True)
    norm_case(ops, torch.bfloat16, rows, 320, "rms", "layer", min(rows, 7), 1.0)


@pytest.mark.parametrize("cols", [20000, 32768])
def test_block_norm_widest(ops, cols):
    norm_case(ops, torch.bfloat16, 3, cols, "layer", "rms", 1, 1.0, rows8=True)


def test_block_norm_offset_rows(ops):
    """A mean far larger than the spread: the variance is taken from centred values."""
    g = gen(3)
    y = (rand(g, 6, 777) + 1000.0)
    r = ops.block_norm(y.cuda(), next_norm="layer", stream=False)
    want = plain.block_norm(y, None, 1.0, None, 1, "none", None, None, "layer", None, None, 1e-5)
    plain.within(r.normed, *want["normed"], torch.float32)
    assert r.stream is None


def test_block_norm_bad_rows_stay_in_their_rows(ops):
    g = gen(9)
    y = rand(g, 6, 130)
    y[1, 129] = float("nan")
    y[2, 0] = float("inf")
    y[3] = 0
    r = ops.block_norm(y.cuda(), next_norm="layer", rows8=True)
    assert r.normed[1].isnan().all() and r.normed[2].isnan().all()
    assert (r.normed[3] == 0).all() and r.scale[3] == 0 and (r.rows8[3] == 0).all()
    assert r.scale[1].isnan() and (r.rows8[1] == 0).all() and (r.rows8[2] == 0).all()
    ok = [0, 4, 5]
    want = plain.block_norm(y[ok], None, 1.0, None, 1, "none", None, None, "layer", None, None, 1e-5)
    plain.within(r.normed[ok], *want["normed"], torch.float32)


def test_block_norm_strides(ops):
    g = gen(4)
    base = rand(g, 9, 140).to(torch.bfloat16).cuda()
    res = rand(g, 9, 333).to(torch.bfloat16).cuda()
    for lo, cols in ((1, 128), (3, 99), (8, 64)):
        y, x = base[:, lo:lo + cols], res[:, 2 * lo + 1:2 * lo + 1 + cols]
        r = ops.block_norm(y, x)
        want = plain.block_norm(y, x, 1.0, None, 1, "none", None, None, "layer", None, None, 1e-5)
        plain.within(r.stream, *want["stream"], torch.bfloat16)
        plain.within(r.normed, *want["normed"], torch.bfloat16)


# ---- attention ------------------------------------------------------------------------------------------------------

def check_attention(got, q, k, v, there, scale):
    """there: (batch, keys) bool."""
    for i in range(q.shape[0]):
        want, err = plain.attention(q[i], k[i], v[i], there[i], scale)
        plain.within(got[i], want, err, q.dtype)


def qkv(g, b, lq, lk, h, hkv, d, dtype):
    return ((rand(g, b, lq, h, d) * 1.5).to(dtype), rand(g, b, lk, hkv, d).to(dtype), rand(g, b, lk, hkv, d).to(dtype))


ATTN = [  # batch, queries, keys, heads, kv heads, d
    (1, 1, 1, 1, 1, 8), (2, 1, 5, 2, 2, 64), (3, 1, 300, 4, 4, 64), (2, 1, 1000, 8, 2, 128), (1, 1, 5000, 4, 1, 64),
    (2, 7, 33, 4, 4, 32), (2, 16, 64, 2, 2, 64), (2, 17, 31, 2, 1, 40), (1, 33, 65, 4, 2, 80), (2, 64, 64, 2, 2, 64),
    (1, 100, 40, 4, 4, 96), (2, 129, 130, 2, 2, 64), (1, 200, 515, 2, 1, 128), (1, 260, 1, 2, 2, 64), (3, 40, 257, 6, 2, 24),
    (1, 5, 2100, 2, 2, 120), (2, 300, 300, 3, 1, 16)]


@pytest.mark.parametrize("shape", ATTN, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_dense(ops, dtype, shape):
    b, lq, lk, h, hkv, d = shape
    g = gen(sum(shape))
    q, k, v = qkv(g, *shape, dtype)
    got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda())
    check_attention(got, q, k, v, torch.ones(b, lk, dtype=torch.bool), d ** -0.5)


@pytest.mark.parametrize("shape", ATTN, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_lengths_and_masks(ops, dtype, shape):
    """Masked keys hold NaN and infinities; the first sequence has no key left, lengths are out of range both ways."""
    b, lq, lk, h, hkv, d = shape
    b += 2
    g = gen(sum(shape) + 1)
    q, k, v = qkv(g, b, lq, lk, h, hkv, d, dtype)
    lens = torch.randint(0, lk + 1, (b,), generator=g, dtype=torch.int32)
    lens[0], lens[1] = -3, lk + 100
    there = torch.arange(lk) < lens[:, None]
    k2, v2 = k.clone(), v.clone()
    k2[~there], v2[~there] = float("nan"), float("inf")
    got = ops.cross_attention(q.cuda(), k2.cuda(), v2.cuda(), key_lengths=lens.cuda(), scale=0.2)
    assert (got[0] == 0).all()
    check_attention(got, q, k, v, there, 0.2)
    mask = torch.rand(b, lk, generator=g) < 0.6
    mask[2] = False
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("-inf"), float("nan")
    got = ops.cross_attention(q.cuda(), k2.cuda(), v2.cuda(), key_mask=mask.cuda())
    assert (got[2] == 0).all()
    check_attention(got, q, k, v, mask, d ** -0.5)
    both = mask & there
    k2[~both], v2[~both] = float("nan"), float("nan")
    got = ops.cross_attention(q.cuda(), k2.cuda(), v2.cuda(), key_mask=mask.to(torch.uint8).cuda(),
                              key_lengths=lens.cuda())
    check_attention(got, q, k, v, both, d ** -0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("h,hkv,d", [(4, 4, 64), (6, 2, 32), (8, 1, 128), (2, 2, 72)])
def test_attention_packed(ops, dtype, h, hkv, d):
    """Packed sequences of every length from none to hundreds, rows before the first and behind the last one; hints below
    the longest sequence change nothing."""
    g = gen(h + d)
    ql, kl = [0, 1, 17, 3, 40, 130, 2, 300], [5, 0, 16, 33, 1, 257, 600, 64]
    start = 3
    qo = torch.tensor([start] + ql).cumsum(0).to(torch.int32)
    ko = torch.tensor([start] + kl).cumsum(0).to(torch.int32)
    tq, tk = int(qo[-1]) + 5, int(ko[-1]) + 2
    q = rand(g, tq, h, d).to(dtype)
    k, v = rand(g, tk, hkv, d).to(dtype), rand(g, tk, hkv, d).to(dtype)
    for rows in (slice(0, start), slice(int(ko[-1]), None)):
        k[rows], v[rows] = float("nan"), float("nan")
    for max_q, max_k in ((300, 600), (1, 2000), (20, 1), (513, 0)):
        got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), q_offsets=qo.cuda(), k_offsets=ko.cuda(), max_q=max_q,
                                  max_k=max_k)
        for i in range(len(ql)):
            a, b, c, e = qo[i], qo[i + 1], ko[i], ko[i + 1]
            want, err = plain.attention(q[a:b], k[c:e], v[c:e], torch.ones(kl[i], dtype=torch.bool), d ** -0.5)
            plain.within(got[a:b], want, err, dtype)
    lens = torch.tensor([2, 5, 16, 7, 1, 200, 0, 999], dtype=torch.int32)
    got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), q_offsets=qo.cuda(), k_offsets=ko.cuda(), max_q=300, max_k=600,
                              key_lengths=lens.cuda())
    for i in range(len(ql)):
        a, b, c, e = qo[i], qo[i + 1], ko[i], ko[i + 1]
        there = torch.arange(kl[i]) < lens[i]
        want, err = plain.attention(q[a:b], k[c:e], v[c:e], there, d ** -0.5)
        plain.within(got[a:b], want, err, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_mixed_forms_and_strides(ops, dtype):
    """Dense queries over packed states; heads and tokens in other orders; states of one tensor that holds both."""
    g = gen(2)
    b, lq, h, d = 3, 9, 4, 64
    kl = [20, 0, 77]
    ko = torch.tensor([0] + kl).cumsum(0).to(torch.int32)
    kv = rand(g, sum(kl), 2, h, d).to(dtype)
    q = rand(g, b, h, lq, d + 8).to(dtype)
    qv = q[..., 3:3 + d].transpose(1, 2)                   # (b, lq, h, d), not contiguous, an odd start
    got = ops.cross_attention(q.cuda()[..., 3:3 + d].transpose(1, 2), kv.cuda()[:, 0], kv.cuda()[:, 1], k_offsets=ko.cuda(),
                              max_k=77)
    for i in range(b):
        want, err = plain.attention(qv[i], kv[ko[i]:ko[i + 1], 0], kv[ko[i]:ko[i + 1], 1],
                                    torch.ones(kl[i], dtype=torch.bool), d ** -0.5)
        plain.within(got[i], want, err, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq,h,hkv,d", [(1, 4, 2, 64), (50, 2, 2, 64), (3, 2, 1, 128), (90, 2, 1, 24), (40, 1, 1, 128)])
def test_attention_unaligned_and_broadcast_keys(ops, dtype, lq, h, hkv, d):
    """Keys and values that start at odd elements, rows of odd spacing, heads in front of tokens; keys shared by the batch, and
    one row shared by every key (strides of 0)."""
    g = gen(lq + d)
    lk = 75
    q = rand(g, 2, lq, h, d).to(dtype).cuda()
    k = rand(g, 2, hkv, lk, d + 5).to(dtype).cuda()[..., 1:1 + d].transpose(1, 2)
    v = rand(g, 2, hkv, lk, d + 3).to(dtype).cuda()[..., 3:3 + d].transpose(1, 2)
    all_ = torch.ones(2, lk, dtype=torch.bool)
    check_attention(ops.cross_attention(q, k, v), q, k, v, all_, d ** -0.5)
    k1, v1 = k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1)
    check_attention(ops.cross_attention(q, k1, v1), q, k1, v1, all_, d ** -0.5)
    k1, v1 = k[:, :1].expand(-1, lk, -1, -1), v[:, :1].expand(-1, lk, -1, -1)
    lens = torch.tensor([lk, 7], dtype=torch.int32)
    check_attention(ops.cross_attention(q, k1, v1, key_lengths=lens.cuda()), q, k1, v1, torch.arange(lk) < lens[:, None],
                    d ** -0.5)


def test_attention_large_scores(ops):
    """Scores of thousands: the maximum is found before anything overflows; a first key far below the others."""
    g = gen(6)
    for dtype in TYPES:
        q, k, v = qkv(g, 2, 3, 400, 2, 2, 64, dtype)
        k = k * 30
        k[:, 0] = -k[:, 0]
        got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)
        check_attention(got, q, k, v, torch.ones(2, 400, dtype=torch.bool), 1.0)
        for scale in (0.0, -0.3):
            got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=scale)
            check_attention(got, q, k, v, torch.ones(2, 400, dtype=torch.bool), scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lq,lk,h,hkv,d", [(40, 70, 8, 8, 64), (1, 70, 8, 8, 64), (50, 3000, 2, 2, 128), (2, 3000, 4, 2, 32),
                                           (70, 200, 16, 8, 64), (600, 90, 40, 40, 32)])
def test_attention_scales_signs_and_holes(ops, dtype, lq, lk, h, hkv, d):
    """Scales of 0 and below, a mask with holes of whole blocks, few and many rows, keys in pieces or not."""
    g = gen(lq + lk)
    q, k, v = qkv(g, 2, lq, lk, h, hkv, d, dtype)
    there = torch.rand(2, lk, generator=g) < 0.7
    there[0, : lk // 2] = False
    there[1, lk // 3: 2 * lk // 3] = False
    k2, v2 = k.clone(), v.clone()
    k2[~there], v2[~there] = float("nan"), float("nan")
    for scale in (0.0, -0.25, 0.1):
        got = ops.cross_attention(q.cuda(), k2.cuda(), v2.cuda(), key_mask=there.cuda(), scale=scale)
        check_attention(got, q, k, v, there, scale)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("b,lq,lk,h,hkv,d", [(1, 700, 1500, 4, 1, 80), (2, 130, 2100, 8, 8, 64), (1, 260, 3001, 4, 4, 128),
                                             (1, 2100, 501, 4, 4, 64), (3, 65, 90, 4, 2, 104), (2, 300, 2000, 8, 4, 32)])
def test_attention_much_to_multiply(ops, dtype, b, lq, lk, h, hkv, d):
    """Many rows and many keys, where tiles of rows share keys and pieces of the keys are joined: a mask with holes, a sequence
    without keys, keys at odd elements; packed, with launches sized for less."""
    g = gen(lq + lk + d)
    q, k, v = qkv(g, b + 1, lq, lk, h, hkv, d, dtype)
    there = torch.rand(b + 1, lk, generator=g) < 0.8
    there[0, : lk // 2] = False
    there[b] = False
    k2 = torch.full((b + 1, lk, hkv, d + 1), float("nan"), dtype=dtype)
    k2[..., 1:][there] = k[there]
    v2 = torch.where(there[..., None, None], v, torch.full((), float("inf"), dtype=dtype))
    got = ops.cross_attention(q.cuda(), k2.cuda()[..., 1:], v2.cuda(), key_mask=there.cuda(), scale=-0.11)
    assert (got[b] == 0).all()
    check_attention(got, q, k, v, there, -0.11)
    aligned = ops.cross_attention(q.cuda(), k2[..., 1:].contiguous().cuda(), v2.cuda(), key_mask=there.cuda(), scale=-0.11)
    assert torch.equal(aligned, got)
    ql, kl = [0, lq, lq // 3], [7, lk // 2, lk]
    qo, ko = (torch.tensor([0] + n).cumsum(0).to(torch.int32) for n in (ql, kl))
    q, k, v = rand(g, sum(ql), h, d).to(dtype), rand(g, sum(kl), hkv, d).to(dtype), rand(g, sum(kl), hkv, d).to(dtype)
    for max_q, max_k in ((lq, lk), (lq // 4, 2 * lk), (lq, 200)):
        got = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), q_offsets=qo.cuda(), k_offsets=ko.cuda(), max_q=max_q,
                                  max_k=max_k)
        for i in range(3):
            x, y = slice(qo[i], qo[i + 1]), slice(ko[i], ko[i + 1])
            want, err = plain.attention(q[x], k[y], v[y], torch.ones(kl[i], dtype=torch.bool), d ** -0.5)
            plain.within(got[x], want, err, dtype)


@pytest.mark.parametrize("lq", [1, 7, 50])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=str)
def test_attention_masks_that_end_anywhere(ops, dtype, lq):
    """A padded batch's masks, rows at any byte: they give what the lengths give, whatever lies behind the last key."""
    g = gen(lq)
    ends = [0, 1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 1020, 1021, 1022, 1023, 1024, 1025, 2047, 2049, 2051]
    b, lk, h, d = len(ends), 2051, 2, 64
    q, k, v = (t.cuda() for t in qkv(g, b, lq, lk, h, h, d, dtype))
    lens = torch.tensor(ends, dtype=torch.int32).cuda()
    want = ops.cross_attention(q, k, v, key_lengths=lens)
    there = (torch.arange(lk) < torch.tensor(ends)[:, None])
    k, v = (torch.where(there.cuda()[..., None, None], t, torch.full((), float("nan"), dtype=dtype).cuda()) for t in (k, v))
    for off, wide in ((0, lk), (1, lk + 1), (2, lk + 2), (3, lk + 4)):
        mask = torch.ones(b, wide + 3, dtype=torch.uint8)
        mask[:, off:off + lk] = there * 7
        got = ops.cross_attention(q, k, v, key_mask=mask.cuda()[:, off:off + lk])
        assert torch.equal(got, want)


def test_attention_no_keys_no_queries(ops):
    q = torch.ones(2, 3, 2, 16).cuda()
    kv = torch.ones(2, 0, 2, 16).cuda()
    assert (ops.cross_attention(q, kv, kv) == 0).all()
    assert ops.cross_attention(q[:, :0], torch.ones(2, 4, 2, 16).cuda(), torch.ones(2, 4, 2, 16).cuda()).shape == (2, 0, 2, 16)
    assert ops.cross_attention(q[:0], kv[:0], kv[:0]).shape == (0, 3, 2, 16)


def test_attention_offsets_out_of_range_are_clamped(ops):
    """Offsets in device memory cannot be checked by the call: the kernels keep to the buffers."""
    q, k = torch.ones(10, 1, 16).cuda(), torch.ones(12, 1, 16).cuda()
    qo = torch.tensor([-5, 4, 1000], dtype=torch.int32).cuda()
    ko = torch.tensor([7, 3, 2000], dtype=torch.int32).cuda()
    got = ops.cross_attention(q, k, k * 2, q_offsets=qo, k_offsets=ko, max_q=10, max_k=12)
    assert (got[:4] == 0).all() and (got[4:] == 2).all()


# ---- streams, graphs ------------------------------------------------------------------------------------------------

def layer(ops, x, st):
    """One post-norm encoder layer: the operators together, as HipEncoder chains them."""
    n = ops.quantize_rows(x)
    t, h, d = x.shape[0], st["heads"], x.shape[1] // st["heads"]
    q = ops.linear_int8(n[0], *st["wq"], x_scale=n[1], bias=st["bq"], out_dtype=x.dtype).view(t, h, d)
    kv = ops.linear_int8(n[0], *st["wkv"], x_scale=n[1], bias=st["bkv"], out_dtype=x.dtype).view(t, 2, h, d)
    c = ops.cross_attention(q, kv[:, 0], kv[:, 1], q_offsets=st["qo"], k_offsets=st["qo"], key_lengths=st["lens"],
                            max_q=st["max"], max_k=st["max"])
    a = ops.linear_int8(c.view(t, h * d), *st["wo"], bias=st["bq"])
    r = ops.block_norm(a, x, next_weight=st["g"], next_bias=st["be"], stream=False, rows8=True)
    f = ops.linear_int8(r.rows8, *st["w1"], x_scale=r.scale, bias=st["b1"], act="gelu", out_dtype=x.dtype)
    f = ops.linear_int8(f, *st["w2"], bias=st["bq"])
    return ops.block_norm(f, r.normed, next_weight=st["g"], next_bias=st["be"], stream=False).normed


def layer_state(g, hidden, heads, inner, lens, dtype):
    def lin(n, k):
        w, s, _ = weights(g, n, k)
        return w.cuda(), s.cuda()
    qo = torch.tensor([0] + [n + 1 for n in lens]).cumsum(0).to(torch.int32)
    return {"heads": heads, "qo": qo.cuda(), "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "max": max(lens) + 1,
            "wq": lin(hidden, hidden), "wkv": lin(2 * hidden, hidden), "wo": lin(hidden, hidden), "w1": lin(inner, hidden),
            "w2": lin(hidden, inner), "bq": rand(g, hidden, scale=0.1).cuda(), "bkv": rand(g, 2 * hidden, scale=0.1).cuda(),
            "b1": rand(g, inner, scale=0.1).cuda(), "g": (1 + rand(g, hidden, scale=0.1)).to(dtype).cuda(),
            "be": rand(g, hidden, scale=0.1).to(dtype).cuda()}, int(qo[-1])


def test_layer_in_a_graph(ops):
    """The layer captured and replayed on new inputs, with eager work between the replays: every replay equals the eager
    result bit for bit; a second captured layer shares no scratch memory with the first."""
    g = gen(12)
    st, t = layer_state(g, 256, 4, 512, [5, 33, 1, 80], torch.bfloat16)
    xs = [rand(g, t, 256).to(torch.bfloat16).cuda() for _ in range(4)]
    want = [layer(ops, x, st) for x in xs]
    a, b = xs[0].clone(), xs[1].clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer(ops, a, st)
    torch.cuda.synchronize()
    graphs = []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(ops, x, st)
        graphs.append((graph, y))
    for i in range(4):
        a.copy_(xs[i])
        b.copy_(xs[(i + 1) % 4])
        graphs[0][0].replay()
        graphs[1][0].replay()
        assert torch.equal(layer(ops, xs[i], st), want[i])
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want[i]) and torch.equal(graphs[1][1], want[(i + 1) % 4])


def test_layer_on_two_streams(ops):
    g = gen(13)
    st, t = layer_state(g, 256, 4, 512, [40] * 6, torch.float16)
    xs = [rand(g, t, 256).to(torch.float16).cuda() for _ in range(2)]
    want = [layer(ops, x, st) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(layer(ops, xs[j], st))
    torch.cuda.synchronize()
    for j in range(2):
        for y in got[j]:
            assert torch.equal(y, want[j])


def test_layer_from_threads(ops):
    """Threads with a stream each, calling at once: nothing is shared between calls."""
    import threading
    g = gen(16)
    st, t = layer_state(g, 256, 4, 512, [40, 3, 90, 17], torch.bfloat16)
    xs = [rand(g, t, 256).to(torch.bfloat16).cuda() for _ in range(4)]
    want = [layer(ops, x, st) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(j):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(20):
                y = layer(ops, xs[(i + j) % 4], st)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[(i + j) % 4]):
                    wrong.append((j, i))

    threads = [threading.Thread(target=work, args=(j,)) for j in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not wrong


def test_everything_in_a_graph_first(ops):
    """Each kernel family captured, also the widest norm (dynamic LDS) and attention in pieces, and replayed on new inputs."""
    g = gen(14)
    x1, x2 = (rand(g, 40, 20000).to(torch.bfloat16).cuda() for _ in range(2))
    w = torch.randint(-127, 128, (48, 20000), generator=g, dtype=torch.int8).cuda()
    sw = torch.rand(48, generator=g).cuda() / 1000
    q = rand(g, 2, 3, 4, 64).to(torch.bfloat16).cuda()
    kv1, kv2 = (rand(g, 2, 5000, 4, 64).to(torch.bfloat16).cuda() for _ in range(2))

    def run(x, kv):
        n = ops.block_norm(x, x, next_norm="rms", rows8=True)
        return (n.stream, n.normed, n.rows8, n.scale, ops.linear_int8(x, w, sw), ops.linear_int8(x[:1, :4096], w[:, :4096], sw),
                ops.cross_attention(q, kv, kv), ops.cross_attention(q.float(), kv.float(), kv.float()))

    want = [run(x1, kv1), run(x2, kv2)]
    a, b = x1.clone(), kv1.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(a, b)
    for i in (1, 0, 1):
        a.copy_((x1, x2)[i])
        b.copy_((kv1, kv2)[i])
        graph.replay()
        again = run(a, b)
        torch.cuda.synchronize()
        for y, z, v in zip(got, again, want[i]):
            assert torch.equal(y, v) and torch.equal(z, v)


def test_copies_and_tiles_in_a_graph(ops):
    """The products that copy odd rows into scratch memory and fp32 attention in tiles and pieces, captured twice: the graphs
    share no scratch memory, and every replay equals the eager result bit for bit."""
    g = gen(15)
    w = torch.randint(-127, 128, (2300, 1001), generator=g, dtype=torch.int8).cuda()
    sw = torch.rand(2300, generator=g).cuda() / 1000
    q8 = torch.randint(-127, 128, (1100, 1001), generator=g, dtype=torch.int8).cuda()
    xs = [rand(g, 300, 1001).to(torch.bfloat16).cuda() for _ in range(4)]
    kv = [rand(g, 1, 1100, 4, 80).cuda() for _ in range(4)]
    q = rand(g, 1, 900, 4, 80).cuda()
    mask = (torch.rand(1, 1100, generator=g) < 0.9).cuda()

    def run(x, s, k):
        return (ops.linear_int8(x, w, sw, act="gelu"), ops.linear_int8(q8, w, sw, x_scale=s), ops.quantize_rows(x)[0],
                ops.cross_attention(q, k, k, key_mask=mask))

    scales = [torch.rand(1100, generator=g).cuda() for _ in range(4)]
    want = [run(xs[i], scales[i], kv[i]) for i in range(4)]
    ins = [[xs[0].clone(), scales[0].clone(), kv[0].clone()] for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for a in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = run(*a)
        graphs.append((graph, y))
    for i in range(4):
        for j, a in enumerate(ins):
            for t, u in zip(a, (xs[(i + j) % 4], scales[(i + j) % 4], kv[(i + j) % 4])):
                t.copy_(u)
        graphs[0][0].replay()
        graphs[1][0].replay()
        again = run(xs[i], scales[i], kv[i])
        torch.cuda.synchronize()
        for j in range(2):
            for y, v in zip(graphs[j][1], want[(i + j) % 4]):
                assert torch.equal(y, v)
        for y, v in zip(again, want[i]):
            assert torch.equal(y, v)


# ---- the C-ABI itself -----------------------------------------------------------------------------------------------

def test_abi_leaves_other_rows_alone_and_works_in_place(ops):
    """Caller-owned results: packed rows that no sequence holds and columns behind a row are left as they were; a norm may
    write its stream and its normed rows over its inputs; the thread's device and stream are its own."""
    from rag_service_amd import _lib
    lib, g = _lib.load_library(), gen(17)
    stream = torch.cuda.current_stream().cuda_stream
    qo, ko = torch.tensor([3, 10, 40], dtype=torch.int32).cuda(), torch.tensor([0, 5, 90], dtype=torch.int32).cuda()
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)):
        q, k, v = (rand(g, n, 2, 64).to(dtype).cuda() for n in (50, 90, 90))
        out = torch.full((50, 2, 72), 7.0, dtype=dtype, device="cuda")
        for max_q in (30, 60):
            need = lib.rr_cross_attention_workspace(code, 2, 2, 2, 64, max_q, 85)
            ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
            rc = lib.rr_cross_attention(0, stream, code, q.data_ptr(), 0, 128, 64, k.data_ptr(), 0, 128, 64, v.data_ptr(), 0, 128,
                                        64, out.data_ptr(), 0, 144, 72, 2, 2, 2, 64, max_q, 85, 50, 90, qo.data_ptr(),
                                        ko.data_ptr(), None, None, 0, 0.125, ws.data_ptr(), need)
            assert rc == 0, lib.rr_last_error()
            assert (out[:3] == 7).all() and (out[40:] == 7).all() and (out[..., 64:] == 7).all()
            want = ops.cross_attention(q, k, v, q_offsets=qo, k_offsets=ko, max_q=max_q, max_k=85, scale=0.125)
            assert torch.equal(out[3:40, :, :64], want[3:40])
        x, y = rand(g, 6, 200).to(dtype).cuda(), rand(g, 6, 200).to(dtype).cuda()
        r = ops.block_norm(y, x, residual_scale=0.5, post_norm="rms")
        a, b = x.clone(), y.clone()
        rc = lib.rr_block_norm(0, stream, code, 6, 200, b.data_ptr(), 200, a.data_ptr(), 200, 0.5, None, 0, 0, 1, 2, None, None,
                               1, None, None, 1e-5, a.data_ptr(), 200, b.data_ptr(), 200, None, 0, None)
        assert rc == 0, lib.rr_last_error()
        assert torch.equal(a, r.stream) and torch.equal(b, r.normed)
        wide = torch.full((6, 300), 3, dtype=torch.int8, device="cuda")
        scale = torch.empty(6, device="cuda")
        assert lib.rr_quantize_rows(0, stream, code, x.data_ptr(), 200, 6, 200, wide.data_ptr(), 300, scale.data_ptr()) == 0
        q8, s8 = ops.quantize_rows(x)
        assert torch.equal(wide[:, :200], q8) and torch.equal(scale, s8) and (wide[:, 200:] == 3).all()
    for m, n, k in ((2, 70, 64), (70, 70, 64), (70, 70, 65), (700, 1500, 64), (3600, 3400, 32)):
        q8 = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8).cuda()
        w, sw, _ = (t.cuda() for t in weights(g, n, k))
        sx = torch.rand(m, generator=g).cuda()
        out = torch.full((m, n + 9), 5.0, dtype=torch.bfloat16, device="cuda")
        assert lib.rr_linear_i8(0, stream, 3, q8.data_ptr(), k, sx.data_ptr(), w.data_ptr(), k, sw.data_ptr(), None, 0, 1,
                                out.data_ptr(), n + 9, m, n, k, None, 0) == 0
        assert torch.equal(out[:, :n], ops.linear_int8(q8, w, sw, x_scale=sx, out_dtype=torch.bfloat16)) and (out[:, n:] == 5).all()
    with pytest.raises(Exception, match="device"):
        _lib._check(lib.rr_quantize_rows(99, None, 0, q.data_ptr(), 200, 6, 200, wide.data_ptr(), 300, scale.data_ptr()))
    assert torch.cuda.current_device() == 0


@pytest.mark.parametrize("cols", [7, 50, 100, 200, 700, 1500, 4608, 9000, 20000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_abi_norm_in_place(ops, dtype, cols):
    """The stream over the residual and the normed rows over the block's output, at every number of lanes a row."""
    from rag_service_amd import _lib
    lib, g, rows = _lib.load_library(), gen(cols), 37
    x, y = rand(g, rows, cols).to(dtype).cuda(), rand(g, rows, cols).to(dtype).cuda()
    r = ops.block_norm(y, x, residual_scale=0.5, rows8=True)
    q, sc = torch.empty_like(r.rows8), torch.empty_like(r.scale)
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    rc = lib.rr_block_norm(0, torch.cuda.current_stream().cuda_stream, code, rows, cols, y.data_ptr(), cols, x.data_ptr(), cols,
                           0.5, None, 0, 0, 1, 0, None, None, 1, None, None, 1e-5, x.data_ptr(), cols, y.data_ptr(), cols,
                           q.data_ptr(), cols, sc.data_ptr())
    assert rc == 0, lib.rr_last_error()
    assert torch.equal(x, r.stream) and torch.equal(y, r.normed) and torch.equal(q, r.rows8) and torch.equal(sc, r.scale)


def test_abi_copied_product_leaves_other_columns_alone(ops):
    """Odd inner sizes: results of a wider matrix, scratch memory of exactly the size asked for with guards behind it."""
    from rag_service_amd import _lib
    lib, g = _lib.load_library(), gen(21)
    stream = torch.cuda.current_stream().cuda_stream
    for code, m, n, k in ((3, 1500, 1600, 1001), (1, 60, 70, 33), (0, 333, 500, 1003), (2, 700, 90, 2050)):
        dtype = (torch.float32, torch.bfloat16, torch.float16, torch.int8)[code]
        x = torch.randint(-127, 128, (m, k), generator=g).to(dtype).cuda() if code == 3 else rand(g, m, k).to(dtype).cuda()
        w, sw, b = (t.cuda() for t in weights(g, n, k))
        sx = torch.rand(m, generator=g).cuda()
        out = torch.full((m, n + 7), 5.0, device="cuda")
        need = lib.rr_linear_i8_workspace(code, m, n, k)
        assert need > 0
        ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device="cuda")
        rc = lib.rr_linear_i8(0, stream, code, x.data_ptr(), k, sx.data_ptr() if code == 3 else None, w.data_ptr(), k,
                              sw.data_ptr(), b.data_ptr(), 1, 0, out.data_ptr(), n + 7, m, n, k, ws.data_ptr(), need)
        assert rc == 0, lib.rr_last_error()
        assert (out[:, n:] == 5).all() and (ws[need:] == 77).all()
        want = ops.linear_int8(x, w, sw, x_scale=sx if code == 3 else None, bias=b, act="gelu", out_dtype=torch.float32)
        assert torch.equal(out[:, :n], want)


# ---- beyond 32 bits -------------------------------------------------------------------------------------------------

def test_linear_and_norm_beyond_32_bit_offsets(ops):
    """More than 2^32 bytes and 2^31 elements of rows and results: the last rows are as right as the first."""
    g = gen(15)
    m, k, n = 2_200_000, 1024, 1024
    q = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    rows = torch.tensor([0, 1, 5000, m // 2, m - 2, m - 1])
    some = torch.randint(-127, 128, (len(rows), k), generator=g, dtype=torch.int8)
    q[rows.cuda()] = some.cuda()
    sx = torch.full((m,), 0.01, device="cuda")
    w, sw, b = weights(g, n, k)
    y = ops.linear_int8(q, w.cuda(), sw.cuda(), x_scale=sx, bias=b.cuda(), out_dtype=torch.bfloat16)
    want, tol = plain.linear(some, torch.full((len(rows),), 0.01), w, sw, b, "none", torch.bfloat16)
    assert ((y[rows.cuda()].double().cpu() - want).abs() <= tol).all()
    assert torch.equal(y[2:4000], b.to(torch.bfloat16).cuda().expand(3998, -1))
    r = ops.block_norm(y, y, rows8=True)
    for at in (slice(0, 3), slice(m - 3, m)):
        ref = plain.block_norm(y[at], y[at], 1.0, None, 1, "none", None, None, "layer", None, None, 1e-5)
        plain.within(r.stream[at], *ref["stream"], torch.bfloat16)
        plain.within(r.normed[at], *ref["normed"], torch.bfloat16)
        few = ops.block_norm(y[at], y[at], rows8=True)     # a row's result does not depend on the others
        assert torch.equal(r.rows8[at], few.rows8) and torch.equal(r.scale[at], few.scale)


@pytest.mark.parametrize("lq", [1, 40])
def test_attention_beyond_32_bit_offsets(ops, lq):
    """A sequence whose keys fill more than 2^32 bytes; the weight lies on its last keys."""
    g = gen(16)
    lk, h, d = 1_100_000, 16, 128
    k = torch.zeros(1, lk, h, d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, lk, h, d, dtype=torch.bfloat16, device="cuda")
    q = rand(g, 1, lq, h, d).to(torch.bfloat16)
    tail_k, tail_v = rand(g, 1, 50, h, d).to(torch.bfloat16), rand(g, 1, 50, h, d).to(torch.bfloat16)
    k[:, -50:], v[:, -50:] = (4 * tail_k).cuda(), tail_v.cuda()
    got = ops.cross_attention(q.cuda(), k, v)
    kk = torch.cat([torch.zeros(1, 1, h, d, dtype=torch.bfloat16), 4 * tail_k], 1).double()
    s = (q.double().transpose(1, 2) @ kk.permute(0, 2, 3, 1)) * d ** -0.5                # (1, h, lq, 51)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w[..., 0] *= lk - 50                                                                # the zero keys, all alike
    want = ((w[..., 1:] / w.sum(-1, keepdim=True)) @ tail_v.double().transpose(1, 2)).transpose(1, 2)
    # a weight is rounded to 16 bits (2^-8), a score is off by 132 U of sum |q k| d ** -0.5 <= 4 |q| |k| d ** -0.5 < 400, and
    # the sum of a million weights of 32 lanes or waves in turn by lk / 128 of its last places: below 2^-8 + 4e-3 + 6e-4
    size = ((w[..., 1:] / w.sum(-1, keepdim=True)) @ tail_v.double().abs().transpose(1, 2)).transpose(1, 2)
    tol = (2.0 ** -8 + 4e-3 + 6e-4) * 2 * size + 2.0 ** -8 * want.abs() + 2.0 ** -133
    assert ((got.double().cpu() - want).abs() <= tol).all()
