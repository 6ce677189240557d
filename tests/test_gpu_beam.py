"""Beam selection, reordering of paged caches and the walk back (izb_beam_select, izb_kv_pages_reorder, izb_beam_trace)
against plain implementations: 64-bit numbers and a stable sort for the selection, the oracle's paged cache copied beam
by beam for the reordering, a loop for the walk.

Scores.  scores_out is the 64-bit total rounded to fp32 (2^-24 of it) plus what the log-sum carries: exp in fp32 of
x - max is off by at most 2^-21 + |x - max| 2^-23 of itself, and sum e^y |y| <= ln(vocab) + 1 of the sum, a thread adds up to 64
of them one after the other and 16 sums join (80 2^-24): below 1e-5 in all for the vocabularies here."""
import copy

import numpy as np
import pytest
import torch

import izwi_oracle as o
from gpu_util import bf16_np, to_np

pytestmark = pytest.mark.gpu
LSE_OFF = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp16": torch.float16}


def plain_select(logits, scores, n_out, finished=None, eos=-1):
    """logits [g, k, v] float64 (already of the stored type), scores [g, k] float64."""
    g, k, v = logits.shape
    total = np.full((g, k, v), -np.inf)
    for i in range(g):
        for b in range(k):
            if not np.isfinite(scores[i, b]):
                continue
            if finished is not None and finished[i, b]:
                total[i, b, eos] = scores[i, b]
                continue
            ok = np.isfinite(logits[i, b])
            if ok.any():
                m = logits[i, b][ok].max()
                lse = m + np.log(np.exp(logits[i, b][ok] - m).sum())
                total[i, b][ok] = logits[i, b][ok] + (scores[i, b] - lse)
    flat = total.reshape(g, -1)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :n_out]
    best = np.take_along_axis(flat, order, 1)
    if best.shape[1] < n_out:
        more = n_out - best.shape[1]
        best, order = np.pad(best, ((0, 0), (0, more)), constant_values=-np.inf), np.pad(order, ((0, 0), (0, more)))
    live = best > -np.inf
    parents, tokens = np.where(live, order // v, 0), np.where(live, order % v, max(eos, 0))
    done = np.zeros_like(live) if finished is None else np.take_along_axis(np.asarray(finished, bool), parents, 1)
    done = live & (done | (tokens == eos))
    return best, parents, tokens, done


def check_select(cuda, x, scores, n_out, finished=None, eos=-1):
    from izwi_b200 import ops
    g, k = scores.shape
    fin = None if finished is None else torch.from_numpy(np.asarray(finished, np.uint8)).to(cuda)
    got = ops.beam_select(x, torch.from_numpy(scores.astype(np.float32)).to(cuda), n_out, fin, eos)
    ops.Context.get(0).check()
    want = plain_select(x.double().cpu().numpy().reshape(g, k, -1), scores.astype(np.float32).astype(np.float64), n_out, finished, eos)
    s, p, t, f = (y.cpu().numpy() for y in got)
    assert np.array_equal(p, want[1]) and np.array_equal(t, want[2]), (p, want[1], t, want[2])
    assert np.array_equal(f.astype(bool), want[3])
    live = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(s), live)
    assert (np.abs(s[live] - want[0][live]) <= LSE_OFF + 2.0 ** -24 * np.abs(want[0][live])).all()
    return got


@pytest.mark.parametrize("dtype", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("g,k,v,n_out", [(1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 7, 6), (1, 4, 51865, 8), (3, 5, 1000, 10), (2, 2, 16385, 64),
                                         (1, 32, 259, 64), (5, 8, 4099, 33), (1, 2, 40, 64), (40, 4, 70001, 4)])
def test_select(cuda, dtype, g, k, v, n_out):
    rng = np.random.default_rng(v + k)
    x = torch.from_numpy(rng.normal(0, 3, (g * k, v)).astype(np.float32)).to(DTYPES[dtype]).to(cuda)
    check_select(cuda, x, rng.normal(-5, 2, (g, k)), n_out)
    fin = rng.random((g, k)) < 0.3
    check_select(cuda, x, rng.normal(-5, 2, (g, k)), n_out, fin, v // 2)


@pytest.mark.parametrize("v", [5, 1000, 40000])
@pytest.mark.parametrize("n_out", [1, 7, 64])
def test_equal_totals_keep_the_lowest_index(cuda, v, n_out):
    """All logits equal, two values only, and beams that are copies of one another with one score."""
    rng = np.random.default_rng(v)
    same = torch.zeros(3, v, device=cuda)
    same[:, 1::2] = -0.0                                     # -0 and +0 are equal
    check_select(cuda, same, np.full((1, 3), -2.0), n_out)
    two = torch.from_numpy(rng.integers(0, 2, (1, v)).astype(np.float32)).to(cuda).repeat(4, 1)
    check_select(cuda, two, np.full((2, 2), -1.5), n_out)
    check_select(cuda, two.to(torch.bfloat16), np.array([[-1.5, -3.0], [0.0, -1.0]]), n_out)


@pytest.mark.parametrize("order", ["up", "down", "one thread"])
def test_values_where_they_are_hardest_to_sort_out(cuda, order):
    """Sorted rows and rows whose large values all lie with one thread of a tile: most of a tile passes the first bound."""
    v = 20000
    row = np.linspace(-4, 4, v, dtype=np.float32)
    if order == "down":
        row = row[::-1].copy()
    if order == "one thread":
        row[np.arange(0, v, 1024)] += 20
    x = torch.from_numpy(np.stack([row, row + 0.37])).to(cuda)
    check_select(cuda, x, np.array([[-1.0, -2.0]]), 16)
    check_select(cuda, x, np.array([[-1.0, -2.0]]), 64)


def test_masked_and_dead_rows(cuda):
    rng = np.random.default_rng(2)
    x = torch.from_numpy(rng.normal(0, 1, (8, 3001)).astype(np.float32)).to(cuda)
    x[0] = float("-inf")
    x[1, 5:] = float("-inf")
    x[2, ::3] = float("nan")
    x[3, 7] = float("inf")
    x[4, :] = torch.finfo(torch.float32).min
    x[5, :] = float("nan")
    scores = np.array([[-1.0, -1.5, -0.5, -2.0], [-1.0, -1.0, -np.inf, np.nan]])
    check_select(cuda, x, scores, 9)
    check_select(cuda, x, scores, 64, np.array([[0, 0, 1, 0], [1, 0, 0, 1]]), 3000)
    check_select(cuda, x[:4], np.full((1, 4), -np.inf), 4)              # nobody alive
    first = np.full((2, 4), -np.inf)
    first[:, 0] = 0
    check_select(cuda, torch.from_numpy(rng.normal(0, 1, (8, 500)).astype(np.float32)).to(cuda), first, 4)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("shift", [1, 3, 5])
def test_rows_off_the_boundary(cuda, dtype, shift):
    """Views into a larger matrix: any start, row distance larger than the vocabulary; NaN around the rows is not read."""
    rng = np.random.default_rng(shift)
    big = torch.full((6, 5003), float("nan"), device=cuda, dtype=DTYPES[dtype])
    big[:, shift:shift + 4097] = torch.from_numpy(rng.normal(0, 2, (6, 4097)).astype(np.float32)).to(cuda).to(DTYPES[dtype])
    check_select(cuda, big[:, shift:shift + 4097], rng.normal(-3, 1, (2, 3)), 6)


def test_scores_and_marks_in_place_on_a_graph(cuda):
    """A captured step that updates its scores and marks in place, replayed with new logits."""
    from izwi_b200 import ops
    rng = np.random.default_rng(4)
    g, k, v, eos = 3, 4, 9001, 17
    steps = [torch.from_numpy(rng.normal(0, 3, (g * k, v)).astype(np.float32)).to(cuda) for _ in range(3)]
    for s in steps:
        s[:, eos] += 8                                        # some beams finish
    x = steps[0].clone()
    scores = torch.full((g, k), float("-inf"), device=cuda)
    scores[:, 0] = 0
    marks = torch.zeros(g, k, device=cuda, dtype=torch.uint8)
    par, tok = torch.zeros(g, k, device=cuda, dtype=torch.int32), torch.zeros(g, k, device=cuda, dtype=torch.int32)
    keep = scores.clone()
    ops.beam_select(x, scores, finished=marks, eos=eos, out=(scores, par, tok, marks))     # outside the capture once
    scores.copy_(keep)
    marks.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.beam_select(x, scores, finished=marks, eos=eos, out=(scores, par, tok, marks))
    ws, wf = keep.double().cpu().numpy(), np.zeros((g, k), bool)
    for s in steps:
        x.copy_(s)
        graph.replay()
        best, wp, wt, wd = plain_select(s.double().cpu().numpy().reshape(g, k, v), ws, k, wf, eos)
        assert np.array_equal(par.cpu().numpy(), wp) and np.array_equal(tok.cpu().numpy(), wt)
        assert np.array_equal(marks.cpu().numpy().astype(bool), wd)
        assert np.abs(scores.cpu().numpy() - best).max() <= LSE_OFF + 2.0 ** -24 * np.abs(best).max()
        ws, wf = scores.double().cpu().numpy(), wd
    assert wf.any()


# ---- reordering ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
@pytest.mark.parametrize("groups,beams,kvh,d,page,first", [(1, 1, 2, 64, 4, 3), (2, 4, 2, 64, 4, 6), (3, 5, 8, 128, 16, 1), (1, 32, 1, 64, 5, 7)])
def test_reorder_follows_copies_of_the_caches(cuda, quant, groups, beams, kvh, d, page, first):
    """Several steps of append and reorder over two layers; the oracle copies each parent's cache outright."""
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(beams + page)
    n = groups * beams
    layers = paged.PagedLayers.allocate(2, n, kvh, d, 40, cuda, quant, page)
    ref = [[[o.KvPages(page, quant), o.KvPages(page, quant)] for _ in range(n)] for _ in range(2)]
    held = 0
    for step, count in enumerate([first, 1, 1, page, 1, 2, 1]):
        for i, cache in enumerate(layers.caches):
            k, v = bf16_np(rng.normal(0, 1, (n, count, kvh, d))), bf16_np(rng.normal(0, 1, (n, count, kvh, d)))
            cache.append(torch.from_numpy(k).to(cuda).to(torch.bfloat16), torch.from_numpy(v).to(cuda).to(torch.bfloat16))
            for b in range(n):
                ref[i][b][0].append(k[b])
                ref[i][b][1].append(v[b])
        held += count
        parents = rng.integers(0, beams, (groups, beams)) if step % 3 else np.sort(rng.integers(0, max(1, beams // 2), (groups, beams)), 1)
        old = layers.caches[0].page_table.clone()
        table = layers.reorder(torch.from_numpy(parents.astype(np.int32)).to(cuda))
        ops.Context.get(0).check()
        assert torch.equal(layers.caches[0].page_table, old)            # the old table is only read
        again = layers.reorder(torch.from_numpy(parents.astype(np.int32)).to(cuda))
        assert torch.equal(again, table)                                  # a repeated call gives the same
        layers.use(table)
        ref = [[copy.deepcopy(layer[g * beams + parents[g, b]]) for g in range(groups) for b in range(beams)] for layer in ref]
        for i, cache in enumerate(layers.caches):
            for which, sel in (("k", 0), ("v", 1)):
                dense = to_np(cache.materialize(which, held))
                for b in range(n):
                    assert np.array_equal(dense[b], ref[i][b][sel].materialize()), (step, i, which, b)
        full, part = divmod(held, page)
        tail = table.cpu().numpy().reshape(groups, beams, -1)[:, :, full:]
        assert len(np.unique(tail)) == tail.size                          # pages still to be written belong to one beam each


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
def test_reorder_leaves_everything_else_alone(cuda, quant):
    """Only the rows held of pages that a further child takes over change; the oracle replays the rule on the host."""
    from izwi_b200 import paged
    rng = np.random.default_rng(21)
    groups, beams, kvh, d, page, per, length = 2, 6, 2, 128, 8, 3, 13
    n = groups * beams * per
    nbytes = page * kvh * d * 2 // {"none": 1, "int8": 2, "q4_0": 4}[quant]
    nsc = {"none": 0, "int8": 1, "q4_0": page * kvh * d // 32}[quant]
    host = [rng.integers(0, 256, (n, nbytes)).astype(np.uint8) for _ in "kv"]
    hsc = [rng.random((n, nsc)).astype(np.float32) for _ in "kv"]
    table = rng.permutation(n).astype(np.int32).reshape(groups * beams, per)
    dev = [torch.from_numpy(x).to(cuda) for x in host]
    dsc = [torch.from_numpy(x).to(cuda) if nsc else None for x in hsc]
    cache = paged.PagedKvCache.view(dev[0], dev[1], dsc[0], dsc[1], torch.from_numpy(table).to(cuda),
                                    torch.full((groups * beams,), length, device=cuda, dtype=torch.int32), kvh, d, quant, page)
    parents = np.array([[2, 2, 0, 2, 5, 0], [1, 1, 1, 1, 1, 1]], np.int32)
    out = paged.PagedLayers([cache]).reorder(torch.from_numpy(parents).to(cuda)).cpu().numpy().reshape(groups, beams, per)
    full, held = divmod(length, page)
    want = table.reshape(groups, beams, per).copy()
    for g in range(groups):
        free = [b for b in range(beams) if b not in parents[g]]
        seen = set()
        for b in range(beams):
            p = parents[g, b]
            want[g, b, :full] = table.reshape(groups, beams, per)[g, p, :full]
            src = table.reshape(groups, beams, per)[g, p, full]
            dst = src if p not in seen else table.reshape(groups, beams, per)[g, free.pop(0), full]
            seen.add(p)
            want[g, b, full] = dst
            if dst != src:
                for x, s in zip(host, hsc):
                    x[dst, :held * nbytes // page] = x[src, :held * nbytes // page]
                    m = 1 if quant == "int8" else held * nsc // page
                    s[dst, :m] = s[src, :m]
    assert np.array_equal(out, want)
    for x, y in zip(dev, host):
        assert np.array_equal(x.cpu().numpy(), y)
    if nsc:
        for x, y in zip(dsc, hsc):
            assert np.array_equal(x.cpu().numpy(), y)


@pytest.mark.parametrize("fault", ["parent too large", "parent negative", "unequal lengths", "length beyond the table"])
def test_reorder_reports_and_leaves_a_wrong_group(cuda, fault):
    from izwi_b200 import IzbError, _lib, ops, paged
    layers = paged.PagedLayers.allocate(1, 6, 2, 64, 16, cuda, "none", 4)
    k = torch.randn(6, 6, 2, 64, device=cuda).to(torch.bfloat16)
    layers.caches[0].append(k, k)
    parents = torch.zeros(2, 3, device=cuda, dtype=torch.int32)
    if fault == "parent too large":
        parents[1, 2] = 3
    elif fault == "parent negative":
        parents[1, 0] = -1
    elif fault == "unequal lengths":
        layers.caches[0].seq_lens[4] = 5
    else:
        layers.caches[0].seq_lens[3:] = 17
    pool = layers.caches[0].k_values.clone()
    before = layers.caches[0].page_table.clone()
    table = layers.reorder(parents)
    with pytest.raises(IzbError) as e:
        ops.Context.get(0).check()
    assert e.value.status == _lib.IZB_ERR_BAD_ARG
    ops.Context.get(0).check()
    assert torch.equal(table[3:], before[3:]) and not torch.equal(table[:3], before[:3])
    assert torch.equal(layers.caches[0].k_values.view(-1, 4 * 2 * 64 * 2)[before[3:].flatten().long()],
                       pool.view(-1, 4 * 2 * 64 * 2)[before[3:].flatten().long()])


# ---- walk back -------------------------------------------------------------------------------------------------------
def plain_trace(parents, tokens, last):
    steps, groups, _ = parents.shape
    out = np.zeros((*last.shape, steps), np.int32)
    for g in range(groups):
        for j in range(last.shape[1]):
            b = last[g, j]
            for s in range(steps - 1, -1, -1):
                out[g, j, s] = tokens[s, g, b]
                b = parents[s, g, b]
    return out


@pytest.mark.parametrize("steps,groups,beams,picks", [(1, 1, 1, 1), (37, 1, 5, 5), (64, 3, 4, 2), (65, 2, 32, 32), (1000, 7, 8, 1), (4097, 2, 3, 3),
                                                      (31, 130, 2, 2), (128, 2, 40, 3), (130, 1, 200, 9)])
def test_trace(cuda, steps, groups, beams, picks):
    from izwi_b200 import ops
    rng = np.random.default_rng(steps + beams)
    parents = rng.integers(0, beams, (steps, groups, beams)).astype(np.int32)
    tokens = rng.integers(0, 2 ** 31 - 1, (steps, groups, beams)).astype(np.int32)
    last = rng.integers(0, beams, (groups, picks)).astype(np.int32)
    got = ops.beam_trace(*(torch.from_numpy(x).to(cuda) for x in (parents, tokens, last)))
    ops.Context.get(0).check()
    assert np.array_equal(got.cpu().numpy(), plain_trace(parents, tokens, last))


@pytest.mark.parametrize("steps", [10, 300])
def test_trace_reports_beams_outside(cuda, steps):
    from izwi_b200 import IzbError, _lib, ops
    rng = np.random.default_rng(5)
    parents = torch.zeros(steps, 2, 3, device=cuda, dtype=torch.int32)
    tokens = torch.from_numpy(rng.integers(0, 100, (steps, 2, 3)).astype(np.int32)).to(cuda)
    last = torch.tensor([[0, 1], [2, 1]], device=cuda, dtype=torch.int32)
    parents[steps // 2, 1, :] = 3
    got = ops.beam_trace(parents, tokens, last).cpu().numpy()
    with pytest.raises(IzbError) as e:
        ops.Context.get(0).check()
    assert e.value.status == _lib.IZB_ERR_BAD_ARG
    ops.Context.get(0).check()
    parents[steps // 2, 1, :] = 0
    want = plain_trace(parents.cpu().numpy(), tokens.cpu().numpy(), last.cpu().numpy())
    want[1, :, :steps // 2] = -1
    assert np.array_equal(got, want)
    last[0, 0] = -1
    got = ops.beam_trace(parents, tokens, last).cpu().numpy()
    assert (got[0, 0] == -1).all() and np.array_equal(got[1, 0], plain_trace(parents.cpu().numpy(), tokens.cpu().numpy(), last.abs().cpu().numpy())[1, 0])
    with pytest.raises(IzbError):
        ops.Context.get(0).check()


def test_trace_of_nothing(cuda):
    from izwi_b200 import ops
    z = torch.zeros(0, 2, 3, device=cuda, dtype=torch.int32)
    assert ops.beam_trace(z, z, torch.zeros(2, 1, device=cuda, dtype=torch.int32)).shape == (2, 1, 0)
