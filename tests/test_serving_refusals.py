"""The cache's and the log probabilities' entry points refuse calls that their
header rules out, before any device work.  CPU only: addresses are made up and
never reached."""

import ctypes as C

import pytest

from ember_amd import capi

INVALID, UNSUPPORTED = 1, 2
P = 4096  # an aligned address


def view(**change):
    f = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, page_table=P, pages=4, heads=2, page_size=16, head_dim=64, sequences=3, max_pages=2)
    f.update(change)
    return capi.KVCacheView(**f)


def refused(status, want=INVALID):
    assert status == want
    assert capi.lib().ember_get_last_error() == want


def write(c=None, k=P, v=P, T=2, st=(256, 64, 128), start=P, count=P, nxt=8192):
    return capi.lib().kv_cache_write(c or view(), k, v, T, *st, start, count, nxt)


def read(c=None, k=P, v=P, T=2, st=(256, 64, 128), start=P, count=P):
    return capi.lib().kv_cache_read(c or view(), k, v, T, *st, start, count)


def attention(c=None, q=P, o=8192, lse=P, T=2, Hq=4, scale=0.125, st=(512, 64, 256), ost=None, start=P, count=P):
    return capi.lib().kv_cache_attention(c or view(), q, o, lse, T, Hq, scale, 1, *st, *(ost or st), start, count)


CALLS = [write, read, attention]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change", [
    dict(pages=-1), dict(pages=2 ** 31), dict(heads=0), dict(heads=65536), dict(page_size=0), dict(page_size=8), dict(page_size=48),
    dict(page_size=1 << 17), dict(sequences=-1), dict(sequences=65536), dict(max_pages=-1), dict(max_pages=2 ** 27), dict(page_table=None),
    dict(page_table=P + 2), dict(k_codes=None), dict(v_scales=None), dict(v_codes=P + 8), dict(k_scales=P + 4), dict(page_size=-16),
])
def test_caches_that_cannot_be(call, change):
    refused(call(view(**change)))


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("D", [0, 16, 48, 96, 256])
def test_head_dims(call, D):
    refused(call(view(head_dim=D)), UNSUPPORTED)


@pytest.mark.parametrize("call", [write, read])
@pytest.mark.parametrize("change", [
    dict(T=-1), dict(T=2 ** 30), dict(k=P + 4), dict(v=P + 8), dict(k=None), dict(v=None), dict(st=(257, 64, 128)), dict(st=(256, 66, 128)),
    dict(st=(256, 64, 130)), dict(st=(256, 64, 1 << 24)), dict(st=(-256, 64, 128)), dict(start=P + 1), dict(count=P + 2),
])
def test_copies(call, change):
    refused(call(**change))


def test_next_is_an_array_of_its_own():
    refused(write(nxt=P))
    refused(write(nxt=8194))


@pytest.mark.parametrize("nxt", [P + 4, P + 8, P - 4, P - 8])
def test_next_overlaps_no_input(nxt):
    refused(write(nxt=nxt, count=None))
    refused(write(nxt=nxt, start=None))
    refused(write(nxt=nxt, start=8192))


@pytest.mark.parametrize("nxt", [P, P + 20, P - 8])
def test_next_does_not_overlap_the_page_table(nxt):
    refused(write(nxt=nxt, start=16384, count=None))


@pytest.mark.parametrize("change", [
    dict(T=-1), dict(Hq=0), dict(Hq=3), dict(Hq=65536), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=None),
    dict(o=None), dict(o=P), dict(q=P + 4), dict(o=8200), dict(lse=P + 2), dict(st=(510, 64, 256)), dict(st=(512, 64, 1 << 24)),
    dict(ost=(512, 62, 256)), dict(ost=(512, -64, 256)), dict(start=P + 2), dict(count=P + 1), dict(T=1 << 30), dict(T=1 << 27, Hq=16),
])
def test_attention(change):
    refused(attention(**change))


def test_calls_of_nothing_do_nothing():
    L = capi.lib()
    none = view(sequences=0, page_table=None)
    assert write(none, k=None, v=None) == read(none, k=None, v=None) == attention(none, q=None, o=None) == 0
    assert write(T=0, k=None, v=None, nxt=None) == read(T=0, k=None, v=None) == attention(T=0, q=None, o=None) == 0
    assert L.token_logprobs(None, 8, None, 0, 8, None, None, None, None, None, 0) == 0
    assert L.token_logprobs_bwd(None, 8, None, None, None, None, None, None, 8, 0, 8) == 0
    assert L.ember_get_last_error() == 0


def test_null_cache():
    L = capi.lib()
    none = C.POINTER(capi.KVCacheView)()
    refused(L.kv_cache_write(none, P, P, 1, 256, 64, 128, None, None, None))
    refused(L.kv_cache_read(none, P, P, 1, 256, 64, 128, None, None))
    refused(L.kv_cache_attention(none, P, 8192, None, 1, 2, 0.125, 1, 256, 64, 128, 256, 64, 128, None, None))


def score(x=P, stride=100, tokens=P, rows=4, classes=100, logp=P, lse=P, ent=P, ids=P, best=P, top=5):
    return capi.lib().token_logprobs(x, stride, tokens, rows, classes, logp, lse, ent, ids, best, top)


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(classes=0), dict(classes=-4), dict(classes=2 ** 31, stride=2 ** 31), dict(stride=99), dict(top=-1), dict(top=65),
    dict(classes=4, top=5), dict(x=None), dict(tokens=None), dict(logp=None), dict(ids=None), dict(best=None), dict(x=P + 1), dict(tokens=P + 2),
    dict(lse=P + 3), dict(ent=P + 1), dict(rows=1 << 31), dict(rows=1 << 62),
])
def test_scores(change):
    refused(score(**change))


def grad(x=P, stride=100, tokens=P, lse=P, ent=P, d_logp=P, d_ent=P, out=8192, out_stride=100, rows=4, classes=100):
    return capi.lib().token_logprobs_bwd(x, stride, tokens, lse, ent, d_logp, d_ent, out, out_stride, rows, classes)


@pytest.mark.parametrize("change", [
    dict(rows=-1), dict(classes=0), dict(stride=99), dict(out_stride=99), dict(x=None), dict(tokens=None), dict(lse=None), dict(out=None),
    dict(ent=None), dict(out=P, out_stride=104), dict(out=8193), dict(d_logp=P + 2), dict(rows=1 << 24), dict(rows=1 << 62),
])
def test_gradients(change):
    refused(grad(**change))


@pytest.mark.parametrize("change", [
    dict(out=P + 4), dict(out=P + 400), dict(out=P + 404), dict(out=P + 1596), dict(x=8192, out=8192 - 4), dict(x=8192, out=8192 - 1596),
    dict(stride=150, out_stride=150, out=P + 396), dict(stride=150, out_stride=150, out=P + 204), dict(stride=150, out_stride=150, out=P + 996),
])
def test_gradients_partly_over_the_logits(change):
    refused(grad(**change))


def test_the_rest_of_lse_is_aligned():
    L = capi.lib()
    refused(L.token_logprobs_ex(P, 100, P, 4, 100, P, P, P + 2, P, None, None, 0))
    refused(L.token_logprobs_bwd_ex(P, 100, P, P, P + 1, P, P, P, 8192, 100, 4, 100))
