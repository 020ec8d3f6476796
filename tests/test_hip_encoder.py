"""HipEncoder (rag_service_amd.core.encoder): packing and refusals on the CPU; on the GPU its stages against 64 bits, its result
against the fp32 model it stands for, and the embedding half and BatchProcessor running on it."""
import json
import os

import numpy as np
import pytest
import torch

import embed_fixture as fx
import encoder_plain as plain

DATA = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "data")


def make_model(hidden=256, heads=4, layers=2, inner=512, vocab=500, seed=0, **kw):
    from transformers import XLMRobertaConfig, XLMRobertaModel
    torch.manual_seed(seed)
    cfg = XLMRobertaConfig(vocab_size=vocab, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads,
                           intermediate_size=inner, max_position_embeddings=66, type_vocab_size=1, pad_token_id=1,
                           bos_token_id=0, eos_token_id=2, layer_norm_eps=1e-5, **kw)
    return XLMRobertaModel(cfg, add_pooling_layer=False).eval()


def batch_of(lengths, length, seed=0, vocab=500):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(5, vocab, (len(lengths), length), generator=g)
    mask = (torch.arange(length) < torch.tensor(lengths)[:, None]).long()
    return torch.where(mask == 1, ids, torch.ones_like(ids)), mask


# ---- CPU ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lengths,length", [([3], 3), ([3], 5), ([1, 4, 2], 4), ([5, 5], 5), ([2, 1], 9), ([7, 1, 7, 3], 7)])
def test_pack_is_the_batch(lengths, length):
    from rag_service_amd.core.encoder import pack
    offsets, source, place, spread = pack(lengths, length)
    assert offsets.dtype == np.int32 and offsets[0] == 0
    assert list(np.diff(offsets)) == [n + (n < length) for n in lengths]
    assert len(source) == len(place) == offsets[-1] and len(spread) == len(lengths) * length
    for b, n in enumerate(lengths):
        for j in range(length):
            r = spread[b * length + j]
            assert offsets[b] <= r < offsets[b + 1]
            if j < n:                                      # a real token is its own row
                assert source[r] == b * length + j and place[r] == j
            else:                                          # every pad is its sequence's one pad row
                assert place[r] == -1 and r == offsets[b + 1] - 1
                assert n <= source[r] - b * length < length


def test_refuses_models_it_does_not_run():
    from transformers import BertConfig, BertModel
    from rag_service_amd.core.encoder import HipEncoder
    bert = BertModel(BertConfig(vocab_size=50, hidden_size=32, num_hidden_layers=1, num_attention_heads=2,
                                intermediate_size=32))
    with pytest.raises(ValueError, match="bert"):
        HipEncoder(bert)
    with pytest.raises(ValueError, match="gelu"):
        HipEncoder(make_model(64, 2, 1, 64, hidden_act="relu"))
    with pytest.raises(ValueError, match="head size"):
        HipEncoder(make_model(60, 3, 1, 64))
    with pytest.raises(ValueError, match="head size"):
        HipEncoder(make_model(272, 2, 1, 64))
    with pytest.raises(ValueError, match="dtype"):
        HipEncoder(make_model(64, 2, 1, 64), dtype="int8")
    with pytest.raises(ValueError, match="GPU only"):
        HipEncoder(make_model(64, 2, 1, 64)).to("cpu")
    with pytest.raises(RuntimeError, match="to"):
        HipEncoder(make_model(64, 2, 1, 64))(torch.zeros(1, 3, dtype=torch.long))


def test_look_reads_the_batch_and_refuses_what_it_cannot_run():
    from rag_service_amd.core.encoder import look
    ids, mask = batch_of([3, 5, 1], 5)
    for t in (torch.int64, torch.int32):
        lengths, lens = look(ids.to(t), mask != 0, None, 1, 500, 1)
        assert lengths == [3, 5, 1] and lens.tolist() == [3, 5, 1] and lens.dtype == torch.int32
    types = torch.zeros_like(ids)
    assert look(ids, mask != 0, types, 1, 500, 1)[0] == [3, 5, 1]
    types[0, 1] = 1                                        # a real token's
    assert look(ids, mask != 0, types, 1, 500, 2)[0] == [3, 5, 1]
    with pytest.raises(ValueError, match="token types 0 to 1 of 1"):
        look(ids, mask != 0, types, 1, 500, 1)
    types[0, 4] = 1                                        # a pad's: pads of a sequence would no longer be alike
    with pytest.raises(ValueError, match="pads are 0"):
        look(ids, mask != 0, types, 1, 500, 2)
    with pytest.raises(ValueError, match="token types -1"):
        look(ids, mask != 0, -mask, 1, 500, 2)
    for bad in (-1, 500, 2 ** 40):
        other = ids.clone()
        other[1, 2] = bad
        with pytest.raises(ValueError, match="token ids"):
            look(other, mask != 0, None, 1, 500, 1)
    with pytest.raises(ValueError, match="without tokens"):
        look(ids, torch.zeros_like(mask) != 0, None, 1, 500, 1)
    with pytest.raises(ValueError, match="right"):
        look(ids.flip(1), mask.flip(1) != 0, None, 1, 500, 1)


def test_batch_processor_refuses_it_off_the_gpu():
    from rag_service_amd.core.batch_processor import BatchProcessor
    with pytest.raises(ValueError, match="GPU only"):
        BatchProcessor(None, {"model": make_model(64, 2, 1, 64)}, None, None, device="cpu", encoder="hip")
    with pytest.raises(ValueError, match="encoder"):
        BatchProcessor(None, {"model": make_model(64, 2, 1, 64)}, None, None, device="cpu", encoder="onnx")


# ---- GPU ------------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def encoder_class(hip):
    from rag_service_amd.core.encoder import HipEncoder
    return HipEncoder


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_stages_against_64_bits(encoder_class, monkeypatch, dtype):
    """Every operator call of a forward pass, on the inputs it really got, against its definition in 64 bits."""
    from rag_service_amd import ops
    enc = encoder_class(make_model(), dtype).to("cuda")
    seen = {"linear": 0, "norm": 0, "attention": 0}
    linear, norm, attention = ops.linear_int8, ops.block_norm, ops.cross_attention

    def checked_linear(x, w, w_scale, *, x_scale=None, bias=None, act="none", out_dtype=None):
        y = linear(x, w, w_scale, x_scale=x_scale, bias=bias, act=act, out_dtype=out_dtype)
        q, sx = (x, x_scale) if x_scale is not None else plain.rows8(x)
        want, tol = plain.linear(q, sx, w, w_scale, bias, act, y.dtype)
        assert ((y.double().cpu() - want).abs() <= tol).all()
        seen["linear"] += 1
        return y

    def checked_norm(y, residual, *, next_weight, next_bias, eps, stream, rows8):
        r = norm(y, residual, next_weight=next_weight, next_bias=next_bias, eps=eps, stream=stream, rows8=rows8)
        want = plain.block_norm(y, residual, 1.0, None, 1, "none", None, None, "layer", next_weight, next_bias, eps)
        plain.within(r.normed, *want["normed"], y.dtype)
        if rows8:
            o, e = want["normed"]
            s = r.scale.double().cpu()[:, None]
            worst = 2 * (1 + 2 ** -6) * e.amax(-1, keepdim=True)
            assert ((r.rows8.double().cpu() * s - o).abs() <= s * (0.5 + 2 ** -12) + worst).all()
        seen["norm"] += 1
        return r

    def checked_attention(q, k, v, *, q_offsets, k_offsets, key_lengths, max_q, max_k):
        o = attention(q, k, v, q_offsets=q_offsets, k_offsets=k_offsets, key_lengths=key_lengths, max_q=max_q, max_k=max_k)
        at = q_offsets.tolist()
        for b, n in enumerate(key_lengths.tolist()):
            a, c = at[b], at[b + 1]
            there = torch.arange(c - a) < n
            want, err = plain.attention(q[a:c], k[a:c], v[a:c], there, q.shape[-1] ** -0.5)
            plain.within(o[a:c], want, err, q.dtype)
        seen["attention"] += 1
        return o

    monkeypatch.setattr(ops, "linear_int8", checked_linear)
    monkeypatch.setattr(ops, "block_norm", checked_norm)
    monkeypatch.setattr(ops, "cross_attention", checked_attention)
    ids, mask = batch_of([9, 1, 20, 13, 20], 20)
    out = enc(input_ids=ids, attention_mask=mask).last_hidden_state
    assert seen == {"linear": 10, "norm": 5, "attention": 2}
    assert out.shape == (5, 20, 256) and out.dtype == torch.float32
    pads = out[0, 9:]
    assert torch.equal(pads, pads[:1].expand_as(pads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lengths,length", [([1], 1), ([12], 12), ([3, 30, 17, 30, 8], 30), ([5] * 40, 9), ([60, 2], 64)])
def test_near_the_fp32_model(encoder_class, lengths, length, dtype):
    """The 8-bit forward pass against the model's own in fp32, pads included.

    A value rounded to 8 bits is off by at most half a step, 1/254 of its row's largest: for the normal rows of a random
    model, whose largest is below 4.5 times their rms, at most 0.018 and, evenly spread in it, 0.0103 of the rms. Rows and
    weights are independent, so a product is off by sqrt(2) 0.0103 = 0.0145 of its own size. A layer has four of them in a row
    (q / k / v, output, up, down), each of which feeds a sum with the residual and a norm: taken as all of the result's size and
    added up, 4 x 0.0145 a layer, 0.116 for two layers; bf16 adds less than 0.004 for each of eight roundings. Relative error
    below 0.15."""
    model = make_model()
    ids, mask = batch_of(lengths, length, seed=length)
    with torch.no_grad():
        want = model(input_ids=ids, attention_mask=mask).last_hidden_state.double()
    got = encoder_class(model, dtype).to("cuda")(input_ids=ids.cuda(), attention_mask=mask.cuda()).last_hidden_state
    got = got.double().cpu()
    assert got.shape == want.shape
    off = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert off.max() <= 0.15, off.max()
    # the embedding (the mean over all positions) averages errors of its own positions: no worse than the worst of them
    a, b = got.mean(1), want.mean(1)
    assert ((a - b).norm(dim=-1) <= 0.15 * want.norm(dim=-1).amax(1)).all()


@pytest.mark.gpu
def test_without_a_mask_and_refusals(encoder_class):
    enc = encoder_class(make_model()).to("cuda")
    ids, mask = batch_of([4, 7], 9)
    a = enc(input_ids=ids.cuda()).last_hidden_state
    b = enc(input_ids=ids.cuda(), attention_mask=mask.cuda(), token_type_ids=torch.zeros_like(ids).cuda()).last_hidden_state
    assert torch.equal(a, b)
    left = mask.flip(1)
    with pytest.raises(ValueError, match="right"):
        enc(input_ids=torch.where(left == 1, torch.full_like(ids, 7), torch.ones_like(ids)), attention_mask=left)
    hole = mask.clone()
    hole[1, 3] = 0
    with pytest.raises(ValueError, match="right"):
        enc(input_ids=ids, attention_mask=hole)
    with pytest.raises(ValueError, match="right"):                      # masked, but no pad token there
        enc(input_ids=torch.full_like(ids, 7), attention_mask=mask)
    with pytest.raises(ValueError, match="without tokens"):
        enc(input_ids=torch.ones_like(ids), attention_mask=torch.zeros_like(mask))
    with pytest.raises(ValueError, match="positions"):
        enc(input_ids=torch.full((1, 65), 7))
    with pytest.raises(ValueError, match="shape"):
        enc(input_ids=ids, attention_mask=mask[:, :5])
    assert enc(input_ids=ids[:0]).last_hidden_state.shape == (0, 9, 256)


class _Queue:
    def __init__(self):
        self.results = {}

    def store_result(self, rid, result):
        self.results[rid] = result


@pytest.mark.gpu
@pytest.mark.parametrize("handoff", [True, False])
def test_batch_processor_on_the_hip_encoder(encoder_class, handoff):
    """Embed, retrieve, prompt, store: BatchProcessor(encoder="hip") over the SQuAD corpus stores what its own embeddings
    retrieve, and the embedding model it was given is left as it was."""
    from rag_service_amd.core.batch_processor import BatchProcessor, embed_queries
    from rag_service_amd.core.retriever import HipRetriever
    corpus = np.load(os.path.join(DATA, "squad_embeddings.npy"))
    contexts = json.load(open(os.path.join(DATA, "squad_contexts.json")))
    queries = json.load(open(os.path.join(DATA, "squad_queries.json")))

    class Tokenizer(fx.HashTokenizer):
        def __call__(self, *a, **kw):
            e = super().__call__(*a, **kw)
            ids = e["input_ids"]                           # words into the small vocabulary, never onto the special tokens
            return {"input_ids": torch.where(ids >= 5, 5 + ids % 495, ids), "attention_mask": e["attention_mask"]}

    model = make_model(hidden=1024, heads=16, layers=1, inner=256, vocab=500)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    retr = HipRetriever(corpus, contexts)
    llm, q = fx.EchoLLM(), _Queue()
    given = {"tokenizer": Tokenizer(), "model": model}
    proc = BatchProcessor(q, given, llm, retr, device="cuda:0", device_handoff=handoff, encoder="hip")
    assert given["model"] is model
    for batch in fx.batches(queries):
        emb = embed_queries(proc.embedding_model, [r["query"] for r in batch], torch.device("cuda:0"))
        docs = retr.batch_retrieve(emb.cpu().numpy(), [r["k"] for r in batch])
        proc._process_batch(batch)
        for r, found in zip(batch, docs):
            prompt = "Context:\n" + "\n---\n".join(found) + f"\n\nQuestion: {r['query']}\n\nThe Answer to this question is: "
            assert q.results[r["id"]] == {"result": f"<answer to: {prompt}>"}
    assert all(torch.equal(v, before[k]) for k, v in model.state_dict().items())
    retr.close()


@pytest.mark.gpu
def test_pads_without_a_mask_are_said_to_be_left_out(encoder_class):
    """Without attention_mask the pad tokens are the mask. The model itself would attend to them, so the call warns; what it
    returns is the model's result with that mask, and without pads there is nothing to say."""
    import warnings
    model = make_model()
    enc = encoder_class(model).to("cuda")
    ids, mask = batch_of([4, 7], 9)
    with pytest.warns(UserWarning, match="attention_mask"):
        got = enc(input_ids=ids.cuda()).last_hidden_state
    with torch.no_grad():
        masked = model(input_ids=ids, attention_mask=mask).last_hidden_state.double()
    off = (got.double().cpu() - masked).norm(dim=-1) / masked.norm(dim=-1)
    assert off.max() <= 0.15                               # (the bound of test_near_the_fp32_model)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        enc(input_ids=ids[:, :4].cuda())
        enc(input_ids=ids.cuda(), attention_mask=mask.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_to_copies_all_weights(encoder_class, dtype):
    """A model on the same device that changes afterwards changes nothing of the encoder's: neither its 8-bit layers nor its
    embedding tables, norms and biases."""
    model = make_model().cuda()
    enc = encoder_class(model, dtype).to("cuda")
    ids, mask = (t.cuda() for t in batch_of([4, 9], 9))
    before = enc(input_ids=ids, attention_mask=mask).last_hidden_state
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(-1.5).add_(0.25)
    assert torch.equal(enc(input_ids=ids, attention_mask=mask).last_hidden_state, before)
