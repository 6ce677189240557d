"""Refusals of the beam-search entry points, without a GPU: every call below has to return its status before it touches
a device, so the context may be a block of zeros and the pointers plain numbers."""
import ctypes as C

import pytest

BAD_ARG, UNSUPPORTED = -1, -2
P = 4096  # an aligned address that nothing may read


@pytest.fixture(scope="module")
def lib():
    from izwi_b200 import build
    build.build()
    import izwi_b200
    return izwi_b200.lib()


@pytest.fixture(scope="module")
def ctx():
    return C.create_string_buffer(4096)


def pages(**kw):
    from izwi_b200 import _lib as L
    a = dict(k_values=P, v_values=P, k_scales=P, v_scales=P, page_table=P, quantization=1, page_size=64, kv_heads=8, head_dim=128,
             max_pages_per_seq=4)
    a.update(kw)
    return L.KvPages(*(a[f] for f, _ in L.KvPages._fields_))


def select(lib, ctx, **kw):
    a = dict(logits=P, dtype=0, groups=2, beams=4, vocab=1000, ld=1000, scores=8192, finished=None, eos=-1, n_out=4, scores_out=16384,
             parents_out=P, tokens_out=P, finished_out=None, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return lib.izb_beam_select(ctx, None, a["logits"], a["dtype"], a["groups"], a["beams"], a["vocab"], a["ld"], a["scores"], a["finished"], a["eos"],
                               a["n_out"], a["scores_out"], a["parents_out"], a["tokens_out"], a["finished_out"], a["workspace"], a["workspace_bytes"])


@pytest.mark.parametrize("kw,status", [
    (dict(groups=-1), BAD_ARG), (dict(beams=0), BAD_ARG), (dict(vocab=0), BAD_ARG), (dict(ld=999), BAD_ARG), (dict(n_out=0), BAD_ARG),
    (dict(dtype=3), BAD_ARG), (dict(eos=1000), BAD_ARG), (dict(finished=P), BAD_ARG), (dict(beams=33), UNSUPPORTED), (dict(n_out=65), UNSUPPORTED),
    (dict(vocab=2 ** 31 - 1, ld=2 ** 31), UNSUPPORTED), (dict(groups=2 ** 30), UNSUPPORTED), (dict(logits=None), BAD_ARG), (dict(scores=None), BAD_ARG),
    (dict(scores_out=None), BAD_ARG), (dict(parents_out=None), BAD_ARG), (dict(tokens_out=None), BAD_ARG), (dict(logits=P + 1), BAD_ARG),
    (dict(dtype=1, logits=P + 2), BAD_ARG), (dict(scores=P + 2), BAD_ARG), (dict(tokens_out=P + 1), BAD_ARG), (dict(workspace=None), BAD_ARG),
    (dict(workspace=P + 4), BAD_ARG), (dict(workspace_bytes=100), BAD_ARG),
    (dict(scores_out=8192, n_out=8), BAD_ARG),                    # in place needs as many results as beams
    (dict(scores_out=8192 + 4), BAD_ARG), (dict(scores_out=8192 - 4), BAD_ARG),
    (dict(finished=P, finished_out=P + 1, eos=3), BAD_ARG),
    (dict(groups=0), 0),
])
def test_select_refusals(lib, ctx, kw, status):
    assert select(lib, ctx, **kw) == status


def test_select_workspace_query(lib, ctx):
    q = lib.izb_beam_select_workspace_bytes
    assert q(ctx, 0, 0, 4, 100, 4) == q(ctx, 0, 1, 33, 100, 4) == q(ctx, 0, 1, 4, 0, 4) == q(ctx, 0, 1, 4, 100, 65) == q(ctx, 0, 1, 4, 2 ** 40, 4) == 0
    assert q(ctx, 0, 1, 4, 100, 4) > 0


def reorder(lib, ctx, layers=None, n=2, **kw):
    from izwi_b200 import _lib as L
    arr = (L.KvPages * n)(*(layers or [pages() for _ in range(n)]))
    a = dict(n_layers=n, parents=P, groups=2, beams=4, lens=P, out=1 << 20)
    a.update(kw)
    return lib.izb_kv_pages_reorder(ctx, None, arr, a["n_layers"], a["parents"], a["groups"], a["beams"], a["lens"], a["out"])


@pytest.mark.parametrize("kw,status", [
    (dict(n_layers=0), BAD_ARG), (dict(groups=-1), BAD_ARG), (dict(beams=0), BAD_ARG), (dict(beams=33), UNSUPPORTED), (dict(groups=20000), UNSUPPORTED),
    (dict(parents=None), BAD_ARG), (dict(lens=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(out=P), BAD_ARG), (dict(out=P + 8 * 4 * 4 - 4), BAD_ARG),
    (dict(out=P - 4), BAD_ARG), (dict(parents=P + 1), BAD_ARG), (dict(groups=0), 0)])
def test_reorder_refusals(lib, ctx, kw, status):
    assert reorder(lib, ctx, **kw) == status


@pytest.mark.parametrize("kw", [dict(page_table=P + 64), dict(quantization=2), dict(page_size=32), dict(kv_heads=4), dict(head_dim=64), dict(max_pages_per_seq=5),
                                dict(k_values=None), dict(v_values=P + 8), dict(k_scales=None), dict(v_scales=P + 2)])
def test_reorder_refuses_layers_that_do_not_agree(lib, ctx, kw):
    assert reorder(lib, ctx, [pages(), pages(**kw)]) == BAD_ARG


@pytest.mark.parametrize("kw,status", [(dict(page_table=None), BAD_ARG), (dict(quantization=3), BAD_ARG), (dict(page_size=0), BAD_ARG),
                                       (dict(kv_heads=0), BAD_ARG), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=2 ** 30), UNSUPPORTED)])
def test_reorder_refuses_the_geometry(lib, ctx, kw, status):
    assert reorder(lib, ctx, [pages(**kw)], n=1) == status
    assert reorder(lib, ctx, [pages()] * 65, n=65) == UNSUPPORTED


@pytest.mark.parametrize("args,status", [
    ((P, P, -1, 1, 2, P, 1, P, 0), BAD_ARG), ((P, P, 5, -1, 2, P, 1, P, 5), BAD_ARG), ((P, P, 5, 1, 0, P, 1, P, 5), BAD_ARG),
    ((P, P, 5, 1, 2, P, -1, P, 5), BAD_ARG), ((P, P, 5, 1, 2, P, 1, P, 4), BAD_ARG), ((None, P, 5, 1, 2, P, 1, P, 5), BAD_ARG),
    ((P, None, 5, 1, 2, P, 1, P, 5), BAD_ARG), ((P, P, 5, 1, 2, None, 1, P, 5), BAD_ARG), ((P, P, 5, 1, 2, P, 1, None, 5), BAD_ARG),
    ((P + 2, P, 5, 1, 2, P, 1, P, 5), BAD_ARG), ((P, P, 2 ** 32, 1, 2, P, 1, P, 2 ** 32), UNSUPPORTED), ((P, P, 0, 1, 2, P, 1, P, 0), 0)])
def test_trace_refusals(lib, ctx, args, status):
    assert lib.izb_beam_trace(ctx, None, *args) == status


def attend(lib, ctx, prefix=None, own=None, **kw):
    a = dict(q=P, plens=P, slens=P, out=P, groups=2, seqs=3, heads=16, max_p=256, max_s=256, ld_q=2048, ld_out=2048, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    pre, suf = prefix or pages(), own or pages()
    return lib.izb_shared_prefix_decode_gqa_attention(ctx, None, a["q"], C.byref(pre), a["plens"], C.byref(suf),
                                                      a["slens"], a["out"], a["groups"], a["seqs"], a["heads"], a["max_p"], a["max_s"], a["ld_q"],
                                                      a["ld_out"], 0.1, a["ws"], a["ws_bytes"])


@pytest.mark.parametrize("kw,status", [
    (dict(groups=-1), BAD_ARG), (dict(seqs=-1), BAD_ARG), (dict(heads=0), BAD_ARG), (dict(q=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(q=P + 8), BAD_ARG),
    (dict(ld_q=2047), BAD_ARG), (dict(ld_q=2040), BAD_ARG), (dict(ld_out=2047), BAD_ARG), (dict(heads=12, ld_q=2048), UNSUPPORTED),
    (dict(heads=136, ld_q=136 * 128, ld_out=136 * 128), UNSUPPORTED), (dict(plens=None), BAD_ARG), (dict(slens=None), BAD_ARG), (dict(plens=P + 2), BAD_ARG),
    (dict(max_p=257), BAD_ARG), (dict(max_s=257), BAD_ARG), (dict(max_p=-1), BAD_ARG), (dict(ws=None), BAD_ARG), (dict(ws=P + 8), BAD_ARG), (dict(ws_bytes=10), BAD_ARG),
    (dict(groups=2 ** 20, seqs=2 ** 20), UNSUPPORTED), (dict(groups=0), 0), (dict(seqs=0), 0)])
def test_attention_refusals(lib, ctx, kw, status):
    assert attend(lib, ctx, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(page_table=None), BAD_ARG), (dict(k_values=P + 8), BAD_ARG), (dict(k_scales=None), BAD_ARG), (dict(v_scales=P + 1), BAD_ARG), (dict(quantization=-1), BAD_ARG),
    (dict(page_size=0), BAD_ARG), (dict(head_dim=256), UNSUPPORTED), (dict(max_pages_per_seq=3), BAD_ARG)])
def test_attention_refuses_pages(lib, ctx, kw, status):
    assert attend(lib, ctx, prefix=pages(**kw)) == status
    assert attend(lib, ctx, own=pages(**kw)) == status


def test_attention_refuses_caches_that_do_not_match(lib, ctx):
    assert attend(lib, ctx, own=pages(kv_heads=4)) == BAD_ARG
    assert attend(lib, ctx, own=pages(head_dim=64)) == BAD_ARG


def test_attention_without_own_pages_has_no_own_tokens(lib, ctx):
    pre = pages()
    assert lib.izb_shared_prefix_decode_gqa_attention(ctx, None, P, C.byref(pre), P, None, None, P, 1, 1, 16, 256, 5, 2048, 2048, 0.1, P, 1 << 40) == BAD_ARG


def test_null_context(lib):
    assert lib.izb_beam_select(None, None, P, 0, 1, 1, 1, 1, P, None, -1, 1, P, P, P, None, P, 1 << 20) == BAD_ARG
    assert lib.izb_beam_trace(None, None, P, P, 1, 1, 1, P, 1, P, 1) == BAD_ARG
    assert lib.izb_kv_pages_reorder(None, None, C.byref(pages()), 1, P, 1, 1, P, P) == BAD_ARG


def test_python_wrappers_refuse_tensors_that_do_not_fit():
    import torch
    from izwi_b200 import ops, paged
    z = torch.zeros
    with pytest.raises(ValueError):
        ops.beam_select(z(4, 10), z(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.beam_select(z(4, 10), z(2, 2))                                     # not on a GPU
    with pytest.raises(ValueError):
        ops.beam_trace(z(3, 2, 2, dtype=torch.int32), z(3, 2, 2, dtype=torch.int32), z(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.beam_trace(z(3, 2, 2, dtype=torch.int32), z(3, 2, 1, dtype=torch.int32), z(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        paged.PagedKvCache.view(z(10), z(10), None, None, z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32), 1, 64)
    with pytest.raises(ValueError):
        paged.PagedLayers([])
