"""What the embedding encoder's operators refuse, before anything reaches a GPU (no GPU needed): the C-ABI's argument checks
through ctypes, and the torch wrappers'."""
import ctypes

import pytest

from rag_service_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load_library()


# an address that is never followed: every call below is refused, or has nothing to do
P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 1)
NULL = None


def refused(lib, rc, code, word):
    assert rc == code, (rc, lib.rr_last_error())
    assert word in lib.rr_last_error().decode(), lib.rr_last_error()


def quantize(lib, device=0, type=0, x=P, ldx=8, rows=2, cols=8, q=P, ldq=8, scale=P):
    return lib.rr_quantize_rows(device, None, type, x, ldx, rows, cols, q, ldq, scale)


@pytest.mark.parametrize("change,word", [
    ({"device": -1}, "device"), ({"type": 3}, "type"), ({"type": 9}, "type"), ({"rows": -1}, "rows"), ({"cols": 0}, "cols"),
    ({"x": NULL}, "x is null"), ({"x": ODD}, "aligned"), ({"ldx": 7}, "stride"), ({"q": NULL}, "q is null"),
    ({"ldq": 7}, "stride"), ({"scale": NULL}, "scale is null"), ({"scale": ODD}, "aligned")])
def test_quantize_rows_refuses(lib, change, word):
    refused(lib, quantize(lib, **change), _lib.RR_E_INVALID, word)


def test_nothing_to_do_is_fine(lib):
    assert quantize(lib, rows=0, x=NULL, q=NULL, scale=NULL) == _lib.RR_OK
    assert linear(lib, m=0, x=NULL, out=NULL) == _lib.RR_OK
    assert norm(lib, rows=0) == _lib.RR_OK
    assert attention(lib, batch=0) == _lib.RR_OK
    assert attention(lib, max_q=0) == _lib.RR_OK


def linear(lib, device=0, x_type=0, x=P, ldx=64, x_scale=NULL, w=P, ldw=64, w_scale=P, bias=NULL, act=0, out_type=0, out=P,
           ldo=16, m=40, n=16, k=64, ws=P, ws_bytes=1 << 20):
    return lib.rr_linear_i8(device, None, x_type, x, ldx, x_scale, w, ldw, w_scale, bias, act, out_type, out, ldo, m, n, k,
                            ws, ws_bytes)


@pytest.mark.parametrize("change,word", [
    ({"device": -2}, "device"), ({"x_type": 4}, "x_type"), ({"x_type": -1}, "x_type"), ({"m": -1}, "m=-1"),
    ({"n": 0}, "n=0"), ({"k": 0}, "k=0"), ({"act": 2}, "act"), ({"out_type": 3}, "out_type"), ({"x": NULL}, "x is null"),
    ({"ldx": 63}, "stride"), ({"w": NULL}, "w is null"), ({"ldw": 63}, "stride"), ({"w_scale": NULL}, "w_scale is null"),
    ({"bias": ODD}, "bias"), ({"out": NULL}, "out is null"), ({"out": ODD}, "aligned"), ({"ldo": 15}, "stride"),
    ({"x_scale": P}, "x_scale"), ({"x_type": 3}, "x_scale"), ({"ws": NULL}, "workspace"), ({"ws_bytes": 40 * 64}, "workspace"),
    ({"ws": ctypes.c_void_p((1 << 20) + 8)}, "16-byte")])
def test_linear_refuses(lib, change, word):
    refused(lib, linear(lib, **change), _lib.RR_E_INVALID, word)


def test_linear_unsupported(lib):
    big = _lib.RR_LINEAR_KMAX + 1
    refused(lib, linear(lib, k=big, ldx=big, ldw=big), _lib.RR_E_UNSUPPORTED, "exact")
    refused(lib, linear(lib, m=1 << 31), _lib.RR_E_UNSUPPORTED, "2^31")
    assert lib.rr_linear_i8_workspace(0, 4, 16, big) == _lib.RR_E_UNSUPPORTED
    assert lib.rr_linear_i8_workspace(7, 4, 16, 64) == _lib.RR_E_INVALID
    assert lib.rr_linear_i8_workspace(3, 4, 16, 64) == 0
    refused(lib, linear(lib, n=(1 << 26) + 1, ldo=1 << 27), _lib.RR_E_UNSUPPORTED, "2^26")
    assert lib.rr_linear_i8_workspace(1, 40, 16, 64) >= 40 * (64 + 4)
    refused(lib, linear(lib, ldw=_lib.RR_LINEAR_LDMOST), _lib.RR_E_UNSUPPORTED, "apart")
    refused(lib, linear(lib, x_type=3, x_scale=P, ldx=_lib.RR_LINEAR_LDMOST), _lib.RR_E_UNSUPPORTED, "apart")
    # odd inner sizes: copies of the weights beside floating-point rows, of both sides for many products of 8-bit rows
    assert lib.rr_linear_i8_workspace(1, 40, 16, 65) < 40 * (80 + 4) + 512
    assert lib.rr_linear_i8_workspace(1, 64, 16, 65) >= 64 * (80 + 4) + 16 * 80
    assert lib.rr_linear_i8_workspace(3, 64, 16, 65) == 0
    assert lib.rr_linear_i8_workspace(3, 1 << 14, 1 << 11, 65) >= ((1 << 14) + (1 << 11)) * 80


def norm(lib, device=0, type=0, rows=4, cols=8, y=P, ldy=8, x=P, ldx=8, rs=1.0, gate=NULL, ldg=8, gate_rows=1,
         rows_per_gate=4, post=0, pw=NULL, pb=NULL, nxt=1, nw=NULL, nb=NULL, eps=1e-5, stream=P, lds=8, normed=P, ldn=8,
         q=NULL, ldq=8, scale=NULL):
    return lib.rr_block_norm(device, None, type, rows, cols, y, ldy, x, ldx, rs, gate, ldg, gate_rows, rows_per_gate, post,
                             pw, pb, nxt, nw, nb, eps, stream, lds, normed, ldn, q, ldq, scale)


@pytest.mark.parametrize("change,word", [
    ({"device": -1}, "device"), ({"type": 3}, "type"), ({"rows": -1}, "rows"), ({"cols": 0}, "cols"), ({"post": 3}, "norm"),
    ({"nxt": -1}, "norm"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"),
    ({"stream": NULL, "normed": NULL}, "no output"), ({"q": P}, "together"), ({"scale": P}, "together"),
    ({"nxt": 0}, "next norm"), ({"nxt": 0, "normed": NULL, "nw": P}, "next norm"), ({"pw": P}, "post norm"),
    ({"pb": P}, "post norm"), ({"gate": P, "rows_per_gate": 0}, "gate rows"), ({"gate": P, "rows_per_gate": 3}, "gate rows"),
    ({"y": NULL}, "y is null"), ({"ldy": 7}, "stride"), ({"x": ODD}, "aligned"), ({"ldx": 7}, "stride"),
    ({"gate": P, "ldg": 7}, "stride"), ({"lds": 7}, "stride"), ({"ldn": 7}, "stride"),
    ({"q": P, "scale": P, "ldq": 7}, "stride"), ({"nw": ODD}, "aligned")])
def test_norm_refuses(lib, change, word):
    refused(lib, norm(lib, **change), _lib.RR_E_INVALID, word)


def test_norm_unsupported(lib):
    c = _lib.RR_NORM_COLMAX + 1
    refused(lib, norm(lib, cols=c, ldy=c, ldx=c, lds=c, ldn=c), _lib.RR_E_UNSUPPORTED, "cols")
    refused(lib, norm(lib, rows=1 << 31), _lib.RR_E_UNSUPPORTED, "2^31")


def attention(lib, device=0, type=1, q=P, qs=(64, 32, 16), k=P, ks=(64, 32, 16), v=P, vs=(64, 32, 16), out=P,
              os=(64, 32, 16), batch=2, heads=2, kv_heads=2, d=16, max_q=2, max_k=2, total_q=0, total_k=0, qo=NULL, ko=NULL,
              lens=NULL, mask=NULL, mask_stride=2, scale=0.25, ws=NULL, ws_bytes=0):
    return lib.rr_cross_attention(device, None, type, q, *qs, k, *ks, v, *vs, out, *os, batch, heads, kv_heads, d, max_q,
                                  max_k, total_q, total_k, qo, ko, lens, mask, mask_stride, scale, ws, ws_bytes)


@pytest.mark.parametrize("change,word", [
    ({"device": -1}, "device"), ({"type": 3}, "type"), ({"batch": -1}, "batch"), ({"heads": 0}, "heads"),
    ({"kv_heads": 0}, "kv_heads"), ({"heads": 3}, "over"), ({"max_q": -1}, "max_q"), ({"max_k": -1}, "max_k"),
    ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"mask": P, "ko": P}, "key_mask"),
    ({"mask": P, "mask_stride": 1}, "mask"), ({"qo": P, "total_q": -1}, "total_q"), ({"ko": P, "total_k": -1}, "total_k"),
    ({"qs": (64, -32, 16)}, "stride"), ({"ks": (-64, 32, 16)}, "stride"), ({"qo": ODD, "total_q": 4}, "aligned"),
    ({"lens": ODD}, "aligned"), ({"q": NULL}, "q is null"), ({"out": NULL}, "out is null"), ({"k": NULL}, "k is null"),
    ({"v": ODD}, "aligned"), ({"heads": 1, "kv_heads": 1, "batch": 1, "max_q": 1, "max_k": 4096}, "workspace")])
def test_attention_refuses(lib, change, word):
    refused(lib, attention(lib, **change), _lib.RR_E_INVALID, word)


@pytest.mark.parametrize("change,word", [
    ({"d": 12}, "head size"), ({"d": 136}, "head size"), ({"d": 0}, "head size"), ({"batch": 65536}, "65535"),
    ({"heads": 65536, "kv_heads": 65536}, "65535"), ({"batch": 4096, "heads": 2048, "kv_heads": 2048}, "2^22"),
    ({"ks": (1 << 24, 1 << 23, 16)}, "apart"), ({"vs": (1 << 24, 1 << 23, 16)}, "apart"),
    ({"max_q": 1 << 29, "heads": 8}, "2^30 rows"), ({"qo": P, "total_q": 1 << 29, "heads": 8}, "2^30 rows"), ({"max_q": (1 << 30) + 1}, "2^30"), ({"max_k": (1 << 30) + 1}, "2^30")])
def test_attention_unsupported(lib, change, word):
    refused(lib, attention(lib, **change), _lib.RR_E_UNSUPPORTED, word)
    if not {"max_q", "ks", "vs", "qo"} & set(change):
        assert lib.rr_cross_attention_workspace(1, change.get("batch", 2), change.get("heads", 2), change.get("kv_heads", 2),
                                                change.get("d", 16), 2, change.get("max_k", 2)) == _lib.RR_E_UNSUPPORTED


def test_attention_workspace_grows_with_the_keys_only_where_there_are_few_rows(lib):
    ws = lib.rr_cross_attention_workspace
    assert ws(1, 1, 1, 1, 64, 1, 100) == 0
    assert ws(1, 1, 1, 1, 64, 1, 100000) > 0
    assert ws(1, 64, 16, 16, 64, 512, 512) == 0


# ---- the torch wrappers (tensors on the CPU are refused too) --------------------------------------------------------

def test_wrappers_refuse():
    import torch
    from rag_service_amd import ops
    x = torch.zeros(4, 64)
    w, s = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.linear_int8(x, w, s), lambda: ops.block_norm(x),
                 lambda: ops.cross_attention(x.view(1, 4, 1, 64), x.view(1, 4, 1, 64), x.view(1, 4, 1, 64))):
        with pytest.raises(ValueError, match="GPU only"):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        ops.quantize_rows([[1.0]])
    with pytest.raises(ValueError, match="type"):
        ops.quantize_rows(x.double())
    with pytest.raises(ValueError, match="gradient"):
        ops.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="act"):
        ops.linear_int8(x, w, s, act="tanh")
    with pytest.raises(ValueError, match="type"):
        ops.linear_int8(x, w, s, x_scale=torch.ones(4))          # scales with floating rows
    with pytest.raises(ValueError, match="norm"):
        ops.block_norm(x, next_norm="batch")
