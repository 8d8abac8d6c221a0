"""Token operators (norm, matrix product, paged cache, attention of layers served in 8-bit integers): what they refuse, on a
machine without a GPU.  Every refusal comes before any GPU work."""
import ctypes as C

import pytest

from n2d2_b200 import runtime

OK, INVALID, CUDA, TOO_LARGE = 0, -1, -2, -5
HERE = (C.c_uint8 * 4096)()
BASE = (C.addressof(HERE) + 63) & ~63      # refused, or nothing to do, before anything looks at it


def norm(**over):
    d = dict(dtype=runtime.BF16, rows=4, columns=64, eps=1e-6, x=BASE, residual=None, total=None, weight=BASE, codes=BASE, scales=BASE, x_stride=0,
             residual_stride=0, total_stride=0, codes_stride=0)
    d.update(over)
    return runtime.load().n2d2b_rmsnorm_quantize(0, C.byref(runtime.Norm(**d)), None)


def matmul(**over):
    d = dict(dtype=runtime.BF16, m=4, n=8, k=16, a=BASE, a_scales=BASE, w=BASE, w_scales=BASE, bias=None, out=BASE, a_stride=0, w_stride=0,
             out_stride=0)
    d.update(over)
    return runtime.load().n2d2b_matmul_i8(0, C.byref(runtime.Matmul(**d)), None)


CACHE = dict(nb_pages=4, nb_heads=2, page_tokens=16, head_size=64, k=BASE, v=BASE, k_scales=BASE, v_scales=BASE)
BATCH = dict(nb_sequences=1, pages_per_sequence=2, nb_tokens=1, max_new=1, page_table=BASE, lengths=BASE, starts=None)
ATTEND = dict(dtype=runtime.BF16, nb_query_heads=4, causal=1, window=0, scale=0.125, q=BASE, out=BASE, q_stride=0, out_stride=0)


def split(over):
    parts = []
    for names in (CACHE, BATCH):
        parts.append(dict(names, **{k: v for k, v in over.items() if k in names}))
    return parts, {k: v for k, v in over.items() if k not in CACHE and k not in BATCH}


def append(**over):
    (cache, batch), rest = split(over)
    d = dict(new_k=BASE, new_v=BASE, dtype=runtime.BF16, stride=0)
    d.update(rest)
    return runtime.load().n2d2b_kv_append(0, C.byref(runtime.KvCacheDesc(**cache)), C.byref(runtime.KvBatchDesc(**batch)), d['new_k'], d['new_v'],
                                          d['dtype'], d['stride'], None)


def attention(**over):
    (cache, batch), rest = split(over)
    return runtime.load().n2d2b_kv_attention(0, C.byref(runtime.KvCacheDesc(**cache)), C.byref(runtime.KvBatchDesc(**batch)),
                                             C.byref(runtime.Attention(**dict(ATTEND, **rest))), None)


def refused(rc, words, code=INVALID):
    assert rc == code, (rc, runtime.load().n2d2b_last_error())
    assert words in runtime.load().n2d2b_last_error().decode()


@pytest.mark.parametrize('over, words', [
    (dict(dtype=0), 'dtype'), (dict(dtype=5), 'dtype'), (dict(rows=-1), 'rows'), (dict(columns=0), 'columns'), (dict(eps=-1.0), 'eps'),
    (dict(eps=float('nan')), 'eps'), (dict(x=None), 'NULL'), (dict(codes=None), 'NULL'), (dict(scales=None), 'NULL'),
    (dict(residual=BASE), 'together'), (dict(total=BASE), 'together'), (dict(x=BASE + 1), 'whole element'), (dict(scales=BASE + 2), 'whole element'),
    (dict(weight=BASE + 1), 'whole element'), (dict(x_stride=63), 'strides'), (dict(codes_stride=8), 'strides'),
    (dict(residual=BASE, total=BASE, total_stride=-64), 'strides'), (dict(dtype=runtime.F32, x=BASE + 2), 'whole element')])
def test_norm_refuses(over, words):
    refused(norm(**over), words)


@pytest.mark.parametrize('over, refuses', [
    (dict(x_stride=128, residual=BASE + 1024, total=BASE), True), (dict(residual=BASE + 1024, residual_stride=128, total=BASE + 1024), True),
    (dict(residual=BASE + 1024, total=BASE, total_stride=128), True), (dict(x_stride=128, residual=BASE + 1024, total=BASE, total_stride=128), False),
    (dict(x_stride=64, residual=BASE + 1024, total=BASE), False), (dict(x_stride=128, residual=BASE + 1024, total=BASE + 1024), False)])
def test_norm_refuses_a_sum_that_overwrites_other_rows(over, refuses):
    if refuses:
        refused(norm(**over), 'same stride')
    else:       # nothing to say about the strides: the next refusal answers
        refused(norm(codes_stride=8, **over), 'columns of a row')


@pytest.mark.parametrize('over, words, code', [
    (dict(dtype=1), 'dtype', INVALID), (dict(m=-1), 'size', INVALID), (dict(n=0), 'size', INVALID), (dict(k=0), 'size', INVALID),
    (dict(k=131072), '131071', TOO_LARGE), (dict(m=65535 * 64 + 1), 'exceeds', TOO_LARGE), (dict(n=65535 * 128 + 1, out_stride=2**24), 'exceeds', TOO_LARGE), (dict(a=None), 'NULL', INVALID),
    (dict(w_scales=None), 'NULL', INVALID), (dict(out=None), 'NULL', INVALID), (dict(out=BASE + 1), 'whole element', INVALID),
    (dict(bias=BASE + 2), 'whole element', INVALID), (dict(a_stride=15), 'strides', INVALID), (dict(out_stride=7), 'strides', INVALID)])
def test_matmul_refuses(over, words, code):
    refused(matmul(**over), words, code)


CACHE_REFUSALS = [
    (dict(nb_pages=0), 'page', INVALID), (dict(nb_heads=0), 'head', INVALID), (dict(page_tokens=8), 'page_tokens', INVALID),
    (dict(page_tokens=48), 'page_tokens', INVALID), (dict(head_size=96), 'head_size', INVALID),
    (dict(nb_pages=2**26, nb_heads=2), '2^31', TOO_LARGE), (dict(k=None), 'NULL', INVALID), (dict(v_scales=None), 'NULL', INVALID),
    (dict(v=BASE + 8), '16 bytes', INVALID), (dict(nb_sequences=-1), 'sequences', INVALID), (dict(pages_per_sequence=0), 'pages', INVALID),
    (dict(nb_sequences=32768), '32767', TOO_LARGE), (dict(pages_per_sequence=2**27), '2^31', TOO_LARGE), (dict(page_table=None), 'NULL', INVALID),
    (dict(lengths=BASE + 2), '4 bytes', INVALID), (dict(max_new=-1), 'new', INVALID)]


@pytest.mark.parametrize('over, words, code', CACHE_REFUSALS + [
    (dict(dtype=runtime.F32), 'dtype', INVALID), (dict(new_k=None), 'NULL', INVALID), (dict(new_v=BASE + 8), '16 bytes', INVALID),
    (dict(stride=127), 'stride', INVALID), (dict(stride=132), 'stride', INVALID), (dict(stride=-128), 'stride', INVALID)])
def test_append_refuses(over, words, code):
    refused(append(**over), words, code)


@pytest.mark.parametrize('over, words, code', CACHE_REFUSALS + [
    (dict(dtype=runtime.F32), 'dtype', INVALID), (dict(nb_query_heads=3), 'multiple', INVALID), (dict(nb_query_heads=0), 'multiple', INVALID),
    (dict(window=-1), 'window', INVALID), (dict(window=4, causal=0), 'window', INVALID), (dict(scale=float('nan')), 'scale', INVALID),
    (dict(scale=float('inf')), 'scale', INVALID), (dict(q=None), 'NULL', INVALID), (dict(out=BASE + 8), '16 bytes', INVALID),
    (dict(q_stride=255), 'strides', INVALID), (dict(out_stride=260), 'strides', INVALID),
    (dict(max_new=2**30, nb_tokens=2**30, starts=BASE), 'exceeds', TOO_LARGE)])
def test_attention_refuses(over, words, code):
    refused(attention(**over), words, code)


def test_missing_descriptions_are_refused():
    lib = runtime.load()
    refused(lib.n2d2b_rmsnorm_quantize(0, None, None), 'NULL')
    refused(lib.n2d2b_matmul_i8(0, None, None), 'NULL')
    refused(lib.n2d2b_kv_append(0, None, None, BASE, BASE, runtime.BF16, 0, None), 'NULL')
    refused(lib.n2d2b_kv_attention(0, C.byref(runtime.KvCacheDesc(**CACHE)), C.byref(runtime.KvBatchDesc(**BATCH)), None, None), 'NULL')


def test_nothing_to_do_is_done_without_a_device():
    assert norm(rows=0) == OK
    assert matmul(m=0) == OK
    for empty in (dict(nb_sequences=0), dict(nb_tokens=0), dict(max_new=0)):
        assert append(**empty) == OK
        assert attention(**empty) == OK


def test_types_are_named():
    with pytest.raises(ValueError, match='f32, f16, bf16'):
        runtime.rmsnorm_quantize(BASE, 0, 64, None, BASE, BASE, dtype='float')


def test_no_fallback_without_a_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip('a GPU is present')
    for rc in (norm(), matmul(), append(), attention(), runtime.load().n2d2b_token_check(0, None)):
        refused(rc, 'device 0 is not usable', CUDA)


def test_a_loose_bound_of_new_tokens_is_no_reason_to_refuse():
    """max_new only bounds: a call of few rows is as large as its rows."""
    import torch
    if torch.cuda.is_available():
        pytest.skip('a GPU is present')
    loose = dict(max_new=2**31 - 1, nb_tokens=7, starts=BASE, nb_sequences=32767, nb_heads=64, nb_query_heads=512)
    refused(attention(**loose), 'device 0 is not usable', CUDA)
    loose.pop('nb_query_heads')
    refused(append(**loose), 'device 0 is not usable', CUDA)


@pytest.mark.parametrize('page', [16, 32, 64, 128])
def test_positions_stay_in_32_bits(page):
    """The last step of 128 tokens of the longest row of pages, and the two that are looked ahead, end below 2^31."""
    most = (2**31 - 512) // page
    for call in (append, attention):
        refused(call(page_tokens=page, nb_pages=1, nb_heads=1, nb_query_heads=1, pages_per_sequence=most + 1) if call is attention else
                call(page_tokens=page, nb_pages=1, nb_heads=1, pages_per_sequence=most + 1), '2^31 - 512', TOO_LARGE)
    capacity = most * page
    assert (capacity + 127) // 128 * 128 + 2 * 128 <= 2**31
