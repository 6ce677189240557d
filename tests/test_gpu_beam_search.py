"""The beam-search operators run together, as a search uses them: the device-side search against one written out in
plain Python, the cache operators over several steps against attention over caches copied beam by beam, and a Qwen3
decoder driven by the search against the same decoder over dense caches that are copied at every step."""
import numpy as np
import pytest
import torch

from gpu_util import assert_matmul_close
from test_gpu_beam import LSE_OFF, plain_select

pytestmark = pytest.mark.gpu


def plain_search(tables, beams, eos):
    """tables [steps, groups * beams, vocab] float64: the logits of every row at every step.  Histories as token lists."""
    steps, rows, _ = tables.shape
    groups = rows // beams
    scores = np.full((groups, beams), -np.inf)
    scores[:, 0] = 0
    done = np.zeros((groups, beams), bool)
    paths = [[[] for _ in range(beams)] for _ in range(groups)]
    for s in range(steps):
        scores, par, tok, done = plain_select(tables[s].reshape(groups, beams, -1), scores.astype(np.float32).astype(np.float64), beams,
                                              done if eos >= 0 else None, eos)
        paths = [[paths[g][par[g, b]] + [int(tok[g, b])] for b in range(beams)] for g in range(groups)]
    return scores, np.array(paths), done


@pytest.mark.parametrize("groups,beams,vocab,steps,eos", [(1, 1, 50, 4, -1), (2, 4, 997, 12, -1), (3, 5, 997, 25, 3), (1, 32, 40, 9, 0)])
def test_search_against_plain_python(cuda, groups, beams, vocab, steps, eos):
    from izwi_b200 import beam, ops
    rng = np.random.default_rng(vocab + beams)
    tables = rng.normal(0, 2, (steps, groups * beams, vocab)).astype(np.float32)
    if eos >= 0:
        tables[:, :, eos] += 3                                   # ends are likely
    search = beam.BeamSearch(groups, beams, steps, cuda, eos)
    for s in range(steps):
        search.step(torch.from_numpy(tables[s]).to(cuda))
    ops.Context.get(0).check()
    want, paths, done = plain_search(tables.astype(np.float64), beams, eos)
    got, scores = search.sequences(beams)
    assert np.array_equal(got.cpu().numpy(), paths)
    # every step rounds its score and carries the log-sum's error
    assert np.abs(scores.cpu().numpy() - want).max() <= steps * (LSE_OFF + 2.0 ** -24 * np.abs(want).max())
    if eos >= 0:
        assert np.array_equal(search.finished.cpu().numpy().astype(bool), done) and search.all_finished() == done.all()
        length = np.where((paths == eos).any(-1), (paths == eos).argmax(-1) + 1, steps)
    else:
        length = np.full(paths.shape[:2], steps)
    ranked, value = search.sequences(1, length_penalty=0.7)
    per = want / length ** 0.7
    best = per.argmax(1)
    assert np.array_equal(ranked.cpu().numpy()[:, 0], paths[np.arange(groups), best])
    assert np.allclose(value.cpu().numpy()[:, 0], per.max(1), rtol=1e-5)
    with pytest.raises(ValueError):
        search.step(torch.from_numpy(tables[0]).to(cuda))


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
def test_attention_follows_the_choices(cuda, quant):
    """Steps of append, choice, reorder and attention; the beams' caches of the plain side are `KvPages` of the oracle, copied
    outright at each choice, the prompt's one more of them.  Tolerance as for the attention alone, with scales that are
    no bf16 numbers for Q4_0 (the oracle's values are rounded as stored)."""
    import copy

    import izwi_oracle as o
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(77)
    groups, beams, heads, kvh, d, page, prompt = 2, 4, 8, 2, 64, 8, 37
    n, half = groups * beams, 2.0 ** -8

    def rand(*shape):
        return torch.from_numpy(rng.normal(0, 1, shape).astype(np.float32)).to(torch.bfloat16)

    prefix = paged.PagedKvCache(groups, kvh, d, prompt, cuda, quant, page)
    own = paged.PagedLayers.allocate(1, n, kvh, d, 40, cuda, quant, page)
    ref_p = [(o.KvPages(page, quant), o.KvPages(page, quant)) for _ in range(groups)]
    ref_o = [(o.KvPages(page, quant), o.KvPages(page, quant)) for _ in range(n)]
    k, v = rand(groups, prompt, kvh, d), rand(groups, prompt, kvh, d)
    prefix.append(k.to(cuda), v.to(cuda))
    for g in range(groups):
        ref_p[g][0].append(k[g].float().numpy())
        ref_p[g][1].append(v[g].float().numpy())
    for step in range(19):
        k, v = rand(n, 1, kvh, d), rand(n, 1, kvh, d)
        own.caches[0].append(k.to(cuda), v.to(cuda))
        for i in range(n):
            ref_o[i][0].append(k[i].float().numpy())
            ref_o[i][1].append(v[i].float().numpy())
        q = rand(n, heads, d)
        got = paged.shared_prefix_attention(q.to(cuda), prefix, own.caches[0]).double().cpu().numpy()
        for i in range(n):
            ks, vs = (np.concatenate([ref_p[i // beams][c].materialize(), ref_o[i][c].materialize()]).astype(np.float64) for c in (0, 1))
            ks, vs = np.repeat(ks, heads // kvh, axis=1), np.repeat(vs, heads // kvh, axis=1)
            s = np.einsum("hd,thd->ht", q[i].double().numpy(), ks) * d ** -0.5
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            want, a = np.einsum("ht,thd->hd", p, vs), np.einsum("ht,thd->hd", p, np.abs(vs))
            off = 0.0
            if quant == "q4_0":                       # a stored value may be the neighbour of the oracle's: one bf16 step
                off = 2 * half
            mag = d ** -0.5 * np.einsum("hd,thd->ht", np.abs(q[i].double().numpy()), np.abs(ks)).max(1, keepdims=True)
            tol = half * np.abs(want) + a * (half + 2.0 ** -18 + np.expm1(2 * mag * (off + 2.0 ** -17)) + off) * (1 + half)
            assert (np.abs(got[i] - want) <= tol).all(), (step, i)
        logits = torch.from_numpy(rng.normal(0, 2, (n, 300)).astype(np.float32)).to(cuda)
        _, parents, _, _ = ops.beam_select(logits, torch.zeros(groups, beams, device=cuda))
        own.use(own.reorder(parents))
        par = parents.cpu().numpy()
        ref_o = [copy.deepcopy(ref_o[g * beams + par[g, b]]) for g in range(groups) for b in range(beams)]
    ops.Context.get(0).check()


def _decoder(cuda, rng, fused):
    from izwi_b200 import decoder
    hid, heads, kvh, d, inter, vocab = 512, 8, 4, 64, 1024, 701

    def w(n, k, std=0.04):
        return torch.from_numpy(rng.normal(0, std, (n, k)).astype(np.float32)).to(cuda).to(torch.bfloat16)

    def norm(n):
        return torch.from_numpy(rng.normal(1, 0.1, n).astype(np.float32)).to(cuda).to(torch.bfloat16)

    layers = [decoder.Qwen3LayerWeights("bf16", hid, heads, kvh, d, inter, norm(hid), norm(hid), norm(d), norm(d), w((heads + 2 * kvh) * d, hid),
                                        w(hid, heads * d), w(2 * inter, hid), w(hid, inter)) for _ in range(2)]
    embed, final, head = w(vocab, hid, 1.0), norm(hid), w(vocab, hid)
    return decoder.Qwen3Decoder(embed, [decoder.Qwen3DecoderLayer(x, fused_qk=fused, fused_linear=False) for x in layers], final, head, "bf16"), kvh, d


@pytest.mark.parametrize("quant", ["none", "int8"])
def test_decoder_follows_the_search(cuda, quant):
    from izwi_b200 import beam, decoder, ops
    rng = np.random.default_rng(31)
    dec, kvh, d = _decoder(cuda, rng, fused=False)
    groups, beams, prompt, new, eos = 2, 3, 9, 7, 5
    caches = [decoder.KvCache(groups, kvh, 32, d, cuda) for _ in dec.layers]
    for pos in range(prompt):
        ids = torch.from_numpy(rng.integers(0, 701, groups)).to(cuda)
        _, logits = dec.step(ids, caches, pos, return_logits=True)
    run = beam.Qwen3BeamDecoder(dec, caches, prompt, beams, new, eos, quantization=quant, page_size=4)
    # the plain side: dense caches of every beam, copied at each choice; the prompt as the pages hold it
    flat = [decoder.KvCache(groups * beams, kvh, 32, d, cuda) for _ in dec.layers]
    for c, f, prefix in zip(caches, flat, run.prefixes):
        for which, src, dst in (("k", c.k, f.k), ("v", c.v, f.v)):
            held = prefix.materialize(which, prompt).transpose(1, 2)                    # [groups, kvh, prompt, d]
            if quant == "none":
                assert torch.equal(held, src[:, :, :prompt])
            dst[:, :, :prompt] = held.repeat_interleave(beams, 0)
    tokens = run.choose(logits.repeat_interleave(beams, 0))
    for step in range(1, new):
        got = run.forward(tokens)
        _, want = dec.step(tokens.long(), flat, prompt + step - 1, return_logits=True)
        assert_matmul_close(got, want.float().cpu().numpy(), f"step {step}")
        before, marks = run.search.scores.double().cpu().numpy(), run.search.finished.cpu().numpy().astype(bool)
        tokens = run.choose(got)
        _, par, tok, _ = plain_select(got.double().cpu().numpy().reshape(groups, beams, -1), before, beams, marks, eos)
        assert np.array_equal(run.search.parents[step].cpu().numpy(), par) and np.array_equal(run.search.tokens[step].cpu().numpy(), tok)
        rows = torch.from_numpy((np.arange(groups)[:, None] * beams + par).reshape(-1)).to(cuda)
        for f in flat:
            f.k, f.v = f.k[rows].contiguous(), f.v[rows].contiguous()
    ops.Context.get(0).check()
    sequences, scores = run.search.sequences(2)
    assert sequences.shape == (groups, 2, new) and torch.isfinite(scores).all()
    run.forward(tokens)
    with pytest.raises(ValueError):        # no room for more
        run.forward(tokens)
    # the whole loop in one call gives the same
    again = beam.Qwen3BeamDecoder(dec, caches, prompt, beams, new, eos, quantization=quant, page_size=4)
    whole, value = again.generate(logits, n_best=2)
    assert torch.equal(whole, sequences) and torch.equal(value, scores)
