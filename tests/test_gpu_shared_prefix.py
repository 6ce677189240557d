"""Attention of sequences that share a prompt (izb_shared_prefix_decode_gqa_attention) against softmax attention in 64 bits
over the stored values, token by token through the page tables.

Tolerance.  The kernel's result differs from the exact one by the rounding of the output (at most 2^-8 of it, half a
bf16 step), the rounding of the weights for the product with v (2^-8 of each term, so 2^-8 of A = sum p |v| / sum p), and
fp32 arithmetic: scores of D products (D 2^-24 of B = scale sum |q| |k|, which moves a weight by that much, both in the
numerator and in the sum) and accumulation over the tokens (T 2^-24 of A).  Q4_0 scales that are no bf16 numbers: a
stored value is the product of code and scale rounded to bf16; the kernel splits the scale into two bf16 parts (the second
at most 2^-8 of it and rounded by 2^-8 of itself, its product with the code once more: 2^-15 in all) and may land on the
neighbour when the product is that near a tie, so it is held to the unrounded product, from which it lies at most
2^-8 + 2^-15 (1 + 2^-8) away: weights move by that times 2 B, values by that."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8


class Pool:
    """A paged cache with random contents; every slot past a sequence's end holds NaN, the table is shuffled."""

    def __init__(self, rng, cuda, lens, kvh, d, page, quant, spare_pages=1, bf16_scales=True):
        from izwi_b200 import paged
        self.lens, self.page, self.kvh, self.d, self.quant = lens, page, kvh, d, quant
        rows, per = len(lens), max(1, -(-max(lens) // page)) + spare_pages
        n = rows * per
        table = rng.permutation(n).astype(np.int32).reshape(rows, per)
        self.exact = []  # per sequence: (k, v), [len, kvh, d] float64
        used = np.zeros((n, page), bool)
        for r, m in enumerate(lens):
            for t in range(m):
                used[table[r, t // page], t % page] = True
        bufs, scales, values = [], [], []
        for _ in "kv":
            if quant == "none":
                x = torch.from_numpy(rng.normal(0, 1, (n, page, kvh, d)).astype(np.float32)).to(torch.bfloat16)
                x[torch.from_numpy(~used)] = float("nan")
                values.append(x.double().numpy())
                bufs.append(x.reshape(-1).to(cuda))
                scales.append(None)
            elif quant == "int8":
                code = rng.integers(1, 256, (n, page, kvh, d)).astype(np.uint8)
                sc = rng.uniform(0.005, 0.02, n).astype(np.float32)
                sc[~used.any(1)] = np.nan
                sb = torch.from_numpy(sc).to(torch.bfloat16).double().numpy()
                values.append(torch.from_numpy((code.astype(np.float64) - 128) * sb[:, None, None, None]).float().to(torch.bfloat16).double().numpy())
                bufs.append(torch.from_numpy(code.reshape(-1)).to(cuda))
                scales.append(torch.from_numpy(sc).to(cuda))
            else:
                code = rng.integers(1, 16, (n, page, kvh, d)).astype(np.uint8)
                sc = rng.uniform(0.05, 0.3, (n, page, kvh, d // 32)).astype(np.float32)
                if bf16_scales:
                    sc = torch.from_numpy(sc).to(torch.bfloat16).float().numpy()
                sc[~used] = np.nan
                x = (code.astype(np.float64) - 8) * np.repeat(sc.astype(np.float64), 32, axis=-1)
                values.append(torch.from_numpy(x).float().to(torch.bfloat16).double().numpy() if bf16_scales else x)
                flat = code.reshape(-1, 2)
                bufs.append(torch.from_numpy((flat[:, 0] | (flat[:, 1] << 4)).astype(np.uint8)).to(cuda))
                scales.append(torch.from_numpy(sc.reshape(-1)).to(cuda))
        for r, m in enumerate(lens):
            t = np.arange(m)
            self.exact.append(tuple(v[table[r, t // page], t % page] for v in values))
        self.cache = paged.PagedKvCache.view(bufs[0], bufs[1], scales[0], scales[1], torch.from_numpy(table).to(cuda),
                                             torch.tensor(lens, dtype=torch.int32, device=cuda), kvh, d, quant, page)


def check(rng, cuda, seqs, heads, prefix, suffix, scale=None, value_off=0.0, **kw):
    """One call against the definition; returns the output."""
    from izwi_b200 import ops, paged
    d, kvh = prefix.d, prefix.kvh
    b = len(prefix.lens) * seqs
    q = torch.from_numpy(rng.normal(0, 2, (b, heads, d)).astype(np.float32)).to(torch.bfloat16)
    got = paged.shared_prefix_attention(q.to(cuda), prefix.cache, None if suffix is None else suffix.cache, scale, **kw)
    ops.Context.get(0).check()
    got = got.double().cpu().numpy()
    qd, g = q.double().numpy(), heads // kvh
    sc = d ** -0.5 if scale is None else scale
    for i in range(b):
        k, v = prefix.exact[i // seqs]
        if suffix is not None:
            k, v = np.concatenate([k, suffix.exact[i][0]]), np.concatenate([v, suffix.exact[i][1]])
        if len(k) == 0:
            assert (got[i] == 0).all(), "a sequence without any token gives zeros"
            continue
        kr, vr = np.repeat(k, g, axis=1), np.repeat(v, g, axis=1)             # [T, heads, d]
        s = np.einsum("hd,thd->ht", qd[i], kr) * sc
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want = np.einsum("ht,thd->hd", p, vr)
        a = np.einsum("ht,thd->hd", p, np.abs(vr))
        mag = abs(sc) * np.einsum("hd,thd->ht", np.abs(qd[i]), np.abs(kr)).max(1, keepdims=True)
        moved = np.expm1(2 * mag * (value_off + (d + 4) * 2.0 ** -24))
        tol = HALF * np.abs(want) + a * (HALF + len(k) * 2.0 ** -24 + 2.0 ** -20 + moved + value_off) * (1 + HALF)
        err = np.abs(got[i] - want)
        assert (err <= tol).all(), f"sequence {i}: {(err / tol).max():.2f} of the tolerance"
    return got


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
@pytest.mark.parametrize("seqs,heads,kvh,d,page,plens,slens", [
    (1, 1, 1, 64, 64, [1], [1]),                       # one row, one token each
    (1, 8, 8, 128, 64, [0], [3]),                      # no prefix
    (4, 16, 8, 128, 64, [100], [5, 5, 5, 5]),
    (5, 4, 4, 64, 5, [63, 64], [0, 1, 2, 64, 65, 7, 0, 3, 130, 4]),   # ragged, pages that end inside a tile
    (4, 16, 4, 128, 16, [65, 0, 129], [0, 0, 0, 0, 1, 0, 2, 0, 9, 9, 9, 9]),  # some sequences with nothing at all
    (3, 32, 2, 64, 7, [200], [33, 1, 0]),              # 48 rows, sixteen query heads per KV head
    (17, 8, 2, 128, 64, [300], [6] * 17),              # 68 rows: the wide block, partly filled
    (33, 8, 2, 64, 128, [257], [1] * 33),              # 132 rows: a second row block of four
    (2, 2, 1, 128, 1, [70], [3, 4]),                   # pages of one token
])
def test_against_the_definition(cuda, quant, seqs, heads, kvh, d, page, plens, slens):
    rng = np.random.default_rng(seqs * 100 + heads + sum(plens))
    prefix = Pool(rng, cuda, plens, kvh, d, page, quant)
    suffix = Pool(rng, cuda, slens, kvh, d, page, quant)
    check(rng, cuda, seqs, heads, prefix, suffix)


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
@pytest.mark.parametrize("seqs,heads,kvh,d,plens", [(5, 20, 20, 64, [1500, 1400]), (8, 8, 8, 128, [5000]), (20, 4, 2, 64, [2500])])
def test_prefix_alone_and_many_chunks(cuda, quant, seqs, heads, kvh, d, plens):
    rng = np.random.default_rng(seqs + heads)
    check(rng, cuda, seqs, heads, Pool(rng, cuda, plens, kvh, d, 64, quant), None)


@pytest.mark.parametrize("pq,sq", [("int8", "none"), ("none", "q4_0"), ("q4_0", "int8")])
def test_prefix_and_suffix_stored_differently(cuda, pq, sq):
    rng = np.random.default_rng(3)
    prefix, suffix = Pool(rng, cuda, [333, 90], 4, 128, 64, pq), Pool(rng, cuda, [20, 0, 70, 1, 64, 65], 4, 128, 16, sq)
    check(rng, cuda, 3, 8, prefix, suffix)


@pytest.mark.parametrize("d", [64, 128])
def test_q4_0_scales_of_full_precision(cuda, d):
    rng = np.random.default_rng(8)
    prefix = Pool(rng, cuda, [150], 2, d, 64, "q4_0", bf16_scales=False)
    suffix = Pool(rng, cuda, [9, 70], 2, d, 64, "q4_0", bf16_scales=False)
    check(rng, cuda, 2, 4, prefix, suffix, value_off=HALF + 2 ** -15 * (1 + HALF))


@pytest.mark.parametrize("scale", [0.0, -0.05, 0.5])
def test_scales_of_any_sign(cuda, scale):
    rng = np.random.default_rng(9)
    check(rng, cuda, 2, 4, Pool(rng, cuda, [130], 2, 64, 64, "none"), Pool(rng, cuda, [3, 67], 2, 64, 64, "none"), scale=scale)


def test_one_row_does_not_depend_on_the_others(cuda):
    """The same sequence alone, with others in its group, and with bounds given: within two roundings of each other."""
    from izwi_b200 import paged
    rng = np.random.default_rng(5)
    prefix, suffix = Pool(rng, cuda, [700], 2, 128, 64, "none"), Pool(rng, cuda, [40] * 6, 2, 128, 64, "none")
    q = torch.from_numpy(rng.normal(0, 1, (6, 8, 128)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    both = paged.shared_prefix_attention(q, prefix.cache, suffix.cache)
    tight = paged.shared_prefix_attention(q, prefix.cache, suffix.cache, max_prefix_len=700, max_seq_len=40)
    one = paged.PagedKvCache.view(suffix.cache.k_values, suffix.cache.v_values, None, None, suffix.cache.page_table[2:3].contiguous(),
                                  suffix.cache.seq_lens[2:3].contiguous(), 2, 128, "none", 64)
    alone = paged.shared_prefix_attention(q[2:3], prefix.cache, one)
    for other in (tight[2], alone[0]):
        diff = (both[2].double() - other.double()).abs()
        assert (diff <= 4 * HALF * both[2].double().abs() + 2 * HALF * 0.2).all()


def test_lengths_are_cut_to_the_bounds(cuda):
    """A length on the device beyond the bound counts up to the bound; a negative one counts nothing."""
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(6)
    prefix, suffix = Pool(rng, cuda, [100], 2, 64, 64, "none"), Pool(rng, cuda, [30, 30], 2, 64, 64, "none")
    q = torch.from_numpy(rng.normal(0, 1, (2, 4, 64)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    want = paged.shared_prefix_attention(q, prefix.cache, None, max_prefix_len=100)
    prefix.cache.seq_lens.fill_(2 ** 30)
    suffix.cache.seq_lens.fill_(-7)
    got = paged.shared_prefix_attention(q, prefix.cache, suffix.cache, max_prefix_len=100)
    ops.Context.get(0).check()
    diff = (got.double() - want.double()).abs()
    assert (diff <= 2 * HALF * want.double().abs() + 2 * HALF * 0.5).all()


def test_non_finite_queries_stay_in_their_rows(cuda):
    from izwi_b200 import paged
    rng = np.random.default_rng(7)
    prefix = Pool(rng, cuda, [90], 2, 64, 64, "none")
    q = torch.from_numpy(rng.normal(0, 1, (3, 4, 64)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    clean = paged.shared_prefix_attention(q, prefix.cache, None)
    q[1, 2, 5] = float("nan")
    got = paged.shared_prefix_attention(q, prefix.cache, None)
    assert got[1, 2].isnan().all()
    got[1, 2] = clean[1, 2]
    assert torch.equal(got, clean)


def test_strided_queries_streams_and_graph_replay(cuda):
    """Rows of q and out apart; a side stream; a captured call replayed with other lengths and queries."""
    from izwi_b200 import paged
    rng = np.random.default_rng(11)
    prefix, suffix = Pool(rng, cuda, [400, 130], 4, 128, 64, "int8"), Pool(rng, cuda, [9, 64, 0, 70], 4, 128, 64, "none")
    wide = torch.from_numpy(rng.normal(0, 1, (4, 3, 8, 128)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    q = wide[:, 1]
    want = paged.shared_prefix_attention(q.contiguous(), prefix.cache, suffix.cache)
    room = torch.full((4, 2, 8, 128), 7.0, device=cuda, dtype=torch.bfloat16)
    paged.shared_prefix_attention(q, prefix.cache, suffix.cache, out=room[:, 0])
    assert torch.equal(room[:, 0], want) and (room[:, 1] == 7.0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = paged.shared_prefix_attention(q, prefix.cache, suffix.cache)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.shared_prefix_attention(q, prefix.cache, suffix.cache)
    graph.replay()
    assert torch.equal(out, want)
    prefix.cache.seq_lens.copy_(torch.tensor([17, 128]))
    suffix.cache.seq_lens.copy_(torch.tensor([1, 2, 0, 64]))
    wide.mul_(0.5)
    graph.replay()
    assert torch.equal(out, paged.shared_prefix_attention(q, prefix.cache, suffix.cache)) and not torch.equal(out, want)
    # two calls under way on two streams with workspaces of their own
    outs = [paged.shared_prefix_attention(q, prefix.cache, suffix.cache) for _ in range(1)]
    with torch.cuda.stream(side):
        outs += [paged.shared_prefix_attention(q, prefix.cache, suffix.cache) for _ in range(3)]
    outs += [paged.shared_prefix_attention(q, prefix.cache, suffix.cache) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)


def test_empty_calls(cuda):
    from izwi_b200 import paged
    rng = np.random.default_rng(1)
    prefix = Pool(rng, cuda, [10], 2, 64, 64, "none")
    q = torch.zeros(0, 4, 64, device=cuda, dtype=torch.bfloat16)
    assert paged.shared_prefix_attention(q, prefix.cache, None).shape == (0, 4, 64)
    q = torch.ones(2, 4, 64, device=cuda, dtype=torch.bfloat16)
    assert (paged.shared_prefix_attention(q, prefix.cache, None, max_prefix_len=0) == 0).all()


def test_agrees_with_paged_attention_over_copies_of_the_prompt(cuda):
    """The same continuations with the prompt copied into each sequence's pages (the entry point that was there)."""
    from izwi_b200 import paged
    rng = np.random.default_rng(12)
    n, kvh, d, p, s = 3, 4, 128, 150, 20
    k = torch.from_numpy(rng.normal(0, 1, (n, p + s, kvh, d)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    v = torch.from_numpy(rng.normal(0, 1, (n, p + s, kvh, d)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    k[:, :p], v[:, :p] = k[:1, :p], v[:1, :p]
    whole = paged.PagedKvCache(n, kvh, d, p + s, cuda)
    whole.append(k, v)
    prefix, suffix = paged.PagedKvCache(1, kvh, d, p, cuda), paged.PagedKvCache(n, kvh, d, s, cuda)
    prefix.append(k[:1, :p].contiguous(), v[:1, :p].contiguous())
    suffix.append(k[:, p:].contiguous(), v[:, p:].contiguous())
    q = torch.from_numpy(rng.normal(0, 1, (n, 8, d)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    a, b = whole.decode_attention(q).double(), paged.shared_prefix_attention(q, prefix, suffix).double()
    # each within half a step of the output and 2^-8 A of the exact result; A <= max |v|, here bounded by 1
    assert ((a - b).abs() <= 2 * HALF * a.abs() + 2 * HALF * 1.0).all()
    assert math.isfinite(float(a.sum()))


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
@pytest.mark.parametrize("seqs,heads,kvh,groups,length", [(8, 16, 4, 1, 60001), (12, 8, 4, 2, 29000), (4, 8, 4, 1, 80000), (4, 8, 4, 1, 116000)])
def test_long_prefixes_of_few_rows(cuda, quant, seqs, heads, kvh, groups, length):
    """Up to 32 rows over prefixes long enough for the tensor-memory kernel, the last chunk cut anywhere; the definition
    computed on the GPU in 64 bits.  Pages of 24 tokens."""
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(length)
    d, page = 128, 24
    lens = [length - 1000 * g for g in range(groups)]
    prefix = Pool(rng, cuda, lens, kvh, d, page, quant, spare_pages=0)
    q = torch.from_numpy(rng.normal(0, 2, (groups * seqs, heads, d)).astype(np.float32)).to(torch.bfloat16).to(cuda)
    got = paged.shared_prefix_attention(q, prefix.cache, None).double()
    ops.Context.get(0).check()
    for g in range(groups):
        k, v = (torch.from_numpy(x).to(cuda) for x in prefix.exact[g])
        qd = q[g * seqs:(g + 1) * seqs].double().reshape(seqs, kvh, heads // kvh, d)
        p = torch.softmax(torch.einsum("skgd,tkd->skgt", qd, k) * d ** -0.5, -1)
        want = torch.einsum("skgt,tkd->skgd", p, v).reshape(seqs, heads, d)
        a = torch.einsum("skgt,tkd->skgd", p, v.abs()).reshape(seqs, heads, d)
        mag = (torch.einsum("skgd,tkd->skgt", qd.abs(), k.abs()).amax(-1) * d ** -0.5).reshape(seqs, heads, 1)
        tol = HALF * want.abs() + a * (HALF + len(k) * 2.0 ** -24 + 2.0 ** -20 + torch.expm1(2 * mag * (d + 4) * 2.0 ** -24)) * (1 + HALF)
        assert ((got[g * seqs:(g + 1) * seqs] - want).abs() <= tol).all()


@pytest.mark.parametrize("quant", ["none", "int8"])
@pytest.mark.parametrize("page", [8, 5])
def test_values_that_are_not_finite_behind_the_end(cuda, quant, page):
    """Many rows (the tensor-memory kernel) over a length that ends inside a tile and a page; behind it lie NaN."""
    rng = np.random.default_rng(page)
    check(rng, cuda, 20, 8, Pool(rng, cuda, [133, 1, 127], 2, 64, page, quant), Pool(rng, cuda, [2] * 60, 2, 64, page, "none"))


def test_two_graphs_share_a_workspace(cuda):
    """Two captured calls with one workspace, replayed in turn: each leaves its own result."""
    import ctypes as C

    from izwi_b200 import _lib as L
    from izwi_b200 import ops, paged  # noqa: F401
    rng = np.random.default_rng(19)
    lib, ctx = L.lib(), ops.Context.get(0)
    sides = []
    for plens, slens, seqs in (([500, 90], [9, 64, 0, 70], 2), ([2000], [30] * 20, 20)):
        prefix, own = Pool(rng, cuda, plens, 2, 128, 64, "none"), Pool(rng, cuda, slens, 2, 128, 64, "none")
        q = torch.from_numpy(rng.normal(0, 1, (len(slens), 8, 128)).astype(np.float32)).to(cuda).to(torch.bfloat16)
        want = paged.shared_prefix_attention(q, prefix.cache, own.cache)
        sides.append((prefix.cache, own.cache, q, seqs, want, torch.zeros_like(want)))
    need = max(lib.izb_shared_prefix_decode_gqa_attention_workspace_bytes(ctx.handle, p.batch, n, 8, 2, 128, p.max_tokens, o.max_tokens)
               for p, o, _, n, _, _ in sides)
    ws = torch.empty(need, device=cuda, dtype=torch.uint8)
    graphs = []
    for p, o, q, n, _, out in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            L.check(lib.izb_shared_prefix_decode_gqa_attention(
                ctx.handle, C.c_void_p(torch.cuda.current_stream().cuda_stream), q.data_ptr(), C.byref(p._desc), p.seq_lens.data_ptr(),
                C.byref(o._desc), o.seq_lens.data_ptr(), out.data_ptr(), p.batch, n, 8, p.max_tokens, o.max_tokens, 1024, 1024, 128 ** -0.5,
                ws.data_ptr(), need), "capture")
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, _, _, _, want, out in sides:
        assert torch.equal(out, want)


@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
@pytest.mark.parametrize("seqs,heads,slens,plen", [(3, 8, [70, 0, 1], 1500), (11, 8, [70, 0, 1] * 3 + [64, 128], 1500), (11, 8, [900] + [0] * 10, 1500),
                                                   (4, 16, [5] * 4, 1500), (3, 8, [70, 0, 1], 100), (7, 8, [9] * 7, 3)])
def test_rows_of_any_stride_and_address(cuda, quant, seqs, heads, slens, plen):
    """Results two bytes off a word, rows an odd number of elements apart, what lies between them left as it was; few and
    many rows, own tokens in one item and in several, in the last launch and before it, all in one cluster."""
    import ctypes as C

    from izwi_b200 import _lib as L
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(len(slens))
    prefix, own = Pool(rng, cuda, [plen], 2, 128, 16, quant), Pool(rng, cuda, slens, 2, 128, 16, quant)
    q = torch.from_numpy(rng.normal(0, 1, (seqs, heads, 128)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    want = paged.shared_prefix_attention(q, prefix.cache, own.cache).reshape(seqs, -1)
    p, o, lib, ctx = prefix.cache, own.cache, L.lib(), ops.Context.get(0)
    ld = heads * 128 + 3
    room = torch.full((seqs * ld + 1,), 7.0, device=cuda, dtype=torch.bfloat16)
    need = lib.izb_shared_prefix_decode_gqa_attention_workspace_bytes(ctx.handle, 1, seqs, heads, 2, 128, p.max_tokens, o.max_tokens)
    ws = torch.empty(need, device=cuda, dtype=torch.uint8)
    L.check(lib.izb_shared_prefix_decode_gqa_attention(
        ctx.handle, C.c_void_p(torch.cuda.current_stream().cuda_stream), q.data_ptr(), C.byref(p._desc), p.seq_lens.data_ptr(), C.byref(o._desc),
        o.seq_lens.data_ptr(), room.data_ptr() + 2, 1, seqs, heads, p.max_tokens, o.max_tokens, heads * 128, ld, 128 ** -0.5, ws.data_ptr(), need), "call")
    got = room[1:].reshape(seqs, ld)
    assert torch.equal(got[:, :-3], want) and (got[:, -3:] == 7).all() and room[0] == 7


@pytest.mark.parametrize("seqs", [2, 20])
@pytest.mark.parametrize("quant", ["none", "int8", "q4_0"])
def test_without_prefix_or_without_own_tokens(cuda, quant, seqs):
    """Bounds of zero leave a cache out, whatever its lengths say; with both at zero every row is zero."""
    from izwi_b200 import ops, paged
    rng = np.random.default_rng(41)
    prefix, own = Pool(rng, cuda, [70, 3], 2, 64, 16, quant), Pool(rng, cuda, ([1, 0, 130, 17] * 10)[:2 * seqs], 2, 64, 16, quant)
    none = Pool(rng, cuda, [0, 0], 2, 64, 16, quant)
    none.cache = prefix.cache
    check(rng, cuda, seqs, 8, none, own, max_prefix_len=0)
    q = torch.from_numpy(rng.normal(0, 1, (2 * seqs, 8, 64)).astype(np.float32)).to(cuda).to(torch.bfloat16)
    assert torch.equal(paged.shared_prefix_attention(q, prefix.cache, own.cache, max_seq_len=0), paged.shared_prefix_attention(q, prefix.cache, None))
    assert (paged.shared_prefix_attention(q, prefix.cache, own.cache, max_prefix_len=0, max_seq_len=0) == 0).all()
    ops.Context.get(0).check()
