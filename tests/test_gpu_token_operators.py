"""Token operators on the GPU against plain implementations in 64 bits, with bounds that follow from the arithmetic."""
import math

import pytest
import torch

from n2d2_b200 import runtime

pytestmark = pytest.mark.gpu
TYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
U = 2.0 ** -24          # half a step of 32 bits
TINY = 2.0 ** -100


def half_step(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def gen(seed=1):
    return torch.Generator(device='cuda').manual_seed(seed)


def normal(*shape, g):
    return torch.randn(shape, device='cuda', generator=g)


# ------------------------------------------------------------------------------------------------ norm
def check_norm(h, weight, codes, scales, dtype, eps):
    """codes, scales of rows h [rows][columns] (as stored) against u / step and step / sqrt(mean + eps) in 64 bits."""
    x = h.double()
    columns = x.shape[1]
    u = x * (1.0 if weight is None else weight.double())
    step = u.abs().amax(1) / 127
    none = step <= TINY
    # a code is round(u * (1 / (top * (1 / 127)))): the constant, three operations, and the product with the weight in 32-bit types
    want = torch.where(none[:, None], 0.0, u / torch.where(none, 1.0, step)[:, None])
    assert ((codes.double() - want).abs() <= 0.5 + 127 * 5 * U).all()
    assert (codes.double().abs() <= 127).all()
    expected = torch.where(none, 0.0, step) / torch.sqrt((x * x).mean(1) + eps)
    # the squares' sum: up to 32 values a thread (or its share of a long row), a tree of ten levels; half of it after the root; then the
    # root's own two steps and five more operations
    bound = ((42 + columns / 512) / 2 + 4 + 8) * U
    assert ((scales.double() - expected).abs() <= expected * bound).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, columns, residual, weight', [
    (1, 1, True, True), (3, 7, False, True), (2, 64, True, True), (5, 1000, True, True), (3, 1024, False, False), (8, 4096, True, True),
    (2, 5120, True, False), (1, 8191, True, True), (2, 16384, True, True), (3, 16400, True, True), (2, 20001, False, True), (300, 96, True, True)])
def test_norm(rows, columns, residual, weight, dtype):
    g, t = gen(rows + columns), TYPES[dtype]
    x = (normal(rows, columns, g=g) * 3).to(t)
    r = normal(rows, columns, g=g).to(t) if residual else None
    w = (1 + 0.3 * normal(columns, g=g)).to(t) if weight else None
    total = torch.full_like(x, 7) if residual else None
    codes = torch.full((rows + 1, columns), 55, dtype=torch.int8, device='cuda')
    scales = torch.full((rows + 1,), 9.0, device='cuda')
    runtime.rmsnorm_quantize(x.data_ptr(), rows, columns, w.data_ptr() if weight else None, codes.data_ptr(), scales.data_ptr(),
                             r.data_ptr() if residual else None, total.data_ptr() if residual else None, dtype=dtype, eps=1e-5)
    h = (x.float() + r.float()).to(t) if residual else x
    if residual:
        assert torch.equal(total, h)
    check_norm(h, w, codes[:rows], scales[:rows], dtype, 1e-5)
    assert (codes[rows] == 55).all() and scales[rows] == 9       # nothing behind the last row


@pytest.mark.parametrize('columns, strides, shift', [(64, (80, 72, 96, 64), 0), (64, (65, 64, 67, 70), 0), (63, (64, 64, 64, 64), 0), (64, (72, 72, 72, 72), 1)])
def test_norm_strides_and_addresses(columns, strides, shift):
    g = gen(5)
    rows = 6
    xs, rs, ts, cs = strides
    x = normal(rows * xs + 8, g=g).bfloat16()
    r = normal(rows * rs + 8, g=g).bfloat16()
    w = normal(columns + 8, g=g).bfloat16()
    total = torch.full((rows * ts + 8,), 3, dtype=torch.bfloat16, device='cuda')
    codes = torch.full((rows * cs + 8,), 55, dtype=torch.int8, device='cuda')
    scales = torch.zeros(rows, device='cuda')
    runtime.rmsnorm_quantize(x[shift:].data_ptr(), rows, columns, w[shift:].data_ptr(), codes[shift:].data_ptr(), scales.data_ptr(), r[shift:].data_ptr(),
                             total[shift:].data_ptr(), eps=0.0, x_stride=xs, residual_stride=rs, total_stride=ts, codes_stride=cs)

    def rows_of(a, stride):
        return a[shift:].as_strided((rows, columns), (stride, 1))
    h = (rows_of(x, xs).float() + rows_of(r, rs).float()).bfloat16()
    assert torch.equal(rows_of(total, ts), h)
    check_norm(h, w[shift:shift + columns], rows_of(codes, cs), scales, 'bf16', 0.0)
    for a, stride, left in ((total, ts, 3), (codes, cs, 55)):
        touched = torch.zeros(a.shape, dtype=torch.bool, device='cuda')
        rows_of(touched, stride).fill_(True)
        assert (a[~touched] == left).all()


@pytest.mark.parametrize('into', ['x', 'residual'])
@pytest.mark.parametrize('columns', [512, 1001, 17000])
def test_norm_sum_in_place(into, columns):
    g = gen(6)
    x, r = normal(3, columns, g=g).half(), normal(3, columns, g=g).half()
    h = (x.float() + r.float()).half()
    codes, scales = torch.zeros((3, columns), dtype=torch.int8, device='cuda'), torch.zeros(3, device='cuda')
    total = x if into == 'x' else r
    runtime.rmsnorm_quantize(x.data_ptr(), 3, columns, None, codes.data_ptr(), scales.data_ptr(), r.data_ptr(), total.data_ptr(), dtype='f16')
    assert torch.equal(total, h)
    check_norm(h, None, codes, scales, 'f16', 1e-6)


@pytest.mark.parametrize('columns', [512, 77])
def test_norm_rows_of_zeros_and_of_what_is_not_finite(columns):
    x = normal(6, columns, g=gen(7))
    x[1] = 0
    x[2, 3] = math.nan
    x[3, 4] = math.inf
    x[4] = 1e-38
    codes, scales = torch.full((6, columns), 5, dtype=torch.int8, device='cuda'), torch.zeros(6, device='cuda')
    runtime.rmsnorm_quantize(x.data_ptr(), 6, columns, None, codes.data_ptr(), scales.data_ptr(), dtype='f32', eps=1e-6)
    values = codes.float() * scales[:, None]
    assert (values[1] == 0).all() and (values[4] == 0).all()
    assert values[2].isnan().all() and values[3].isnan().all()
    keep = [0, 5]
    check_norm(x[keep], None, codes[keep], scales[keep], 'f32', 1e-6)


# ------------------------------------------------------------------------------------------------ matrix product
def check_matmul(a, w, sa, sw, bias, out, dtype):
    p = (a.double() @ w.double().T) * torch.outer(sa.double(), sw.double())
    y = p if bias is None else p + bias.double()
    # the sum is exact; its conversion, two products, the bias, and the rounding to the output's type (half a smallest step below its normal range)
    bound = 4 * U * p.abs() + 2 * U * y.abs() + half_step(dtype) * y.abs() * (1 + 8 * U) + torch.finfo(TYPES[dtype]).smallest_normal * half_step(dtype)
    off = (out.double() - y).abs()
    assert (off <= bound).all(), (off - bound).max()


def codes_of(m, k, g, low=-127):
    return torch.randint(low, 128, (m, k), device='cuda', generator=g).to(torch.int8)


@pytest.mark.parametrize('m, n, k, dtype, bias', [
    (1, 1, 1, 'f32', True), (3, 5, 7, 'bf16', False), (2, 64, 64, 'f16', True), (1, 4096, 4096, 'bf16', False), (17, 100, 33, 'bf16', True),
    (7, 129, 144, 'f32', False), (8, 256, 1024, 'f16', False), (9, 130, 272, 'bf16', True), (33, 1000, 2048, 'f32', True), (64, 200, 4096, 'bf16', False),
    (100, 520, 528, 'f16', True), (128, 128, 128, 'f32', False), (129, 1000, 640, 'bf16', True), (255, 260, 2064, 'f32', False),
    (257, 513, 1040, 'f16', False), (300, 520, 4096, 'bf16', True), (1000, 1001, 1024, 'f16', False), (513, 2050, 1003, 'bf16', False),
    (2500, 777, 160, 'f32', True), (1, 7, 16, 'f32', False), (5, 8192, 16, 'bf16', False), (2048, 2048, 2048, 'bf16', True)])
def test_matmul(m, n, k, dtype, bias):
    g = gen(m + n + k)
    a, w = codes_of(m, k, g, -128), codes_of(n, k, g, -128)
    sa, sw = torch.rand(m, device='cuda', generator=g) + 0.1, (torch.rand(n, device='cuda', generator=g) + 0.1) / (74 * math.sqrt(k))
    b = normal(n, g=g) if bias else None
    out = torch.full((m * n + 64,), 3.0, dtype=TYPES[dtype], device='cuda')
    runtime.matmul_i8(a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), out.data_ptr(), m, n, k, dtype=dtype, bias=b.data_ptr() if bias else None)
    runtime.token_check()
    assert (out[m * n:] == 3).all()
    check_matmul(a, w, sa, sw, b, out[:m * n].view(m, n), dtype)


@pytest.mark.parametrize('m, n, k', [(1, 40, 131056), (70, 300, 131071)])
def test_matmul_longest_sums(m, n, k):
    """Every product at its largest: the sums come near the end of 32 bits."""
    a = torch.full((m, k), -128, dtype=torch.int8, device='cuda')
    w = torch.full((n, k), -128, dtype=torch.int8, device='cuda')
    one_a, one_w = torch.ones(m, device='cuda'), torch.ones(n, device='cuda')
    out = torch.zeros((m, n), device='cuda')
    runtime.matmul_i8(a.data_ptr(), one_a.data_ptr(), w.data_ptr(), one_w.data_ptr(), out.data_ptr(), m, n, k, dtype='f32')
    runtime.token_check()
    assert (out.double() - 16384.0 * k).abs().max() <= 16384.0 * k * U


@pytest.mark.parametrize('m', [1, 5, 40, 300])
@pytest.mark.parametrize('a_stride, w_stride, out_stride, shift', [(96, 112, 104, 0), (81, 80, 101, 0), (96, 96, 99, 3), (96, 96, 104, 16)])
def test_matmul_strides_and_addresses(m, a_stride, w_stride, out_stride, shift):
    g = gen(m)
    n, k = 99, 80
    a, w = codes_of(1, m * a_stride + 32, g)[0], codes_of(1, n * w_stride + 32, g)[0]
    sa, sw = torch.rand(m, device='cuda', generator=g), torch.rand(n, device='cuda', generator=g)
    out = torch.full((m * out_stride + 8,), 3.0, device='cuda')
    runtime.matmul_i8(a[shift:].data_ptr(), sa.data_ptr(), w[shift:].data_ptr(), sw.data_ptr(), out[1:].data_ptr(), m, n, k, dtype='f32', a_stride=a_stride,
                      w_stride=w_stride, out_stride=out_stride)
    runtime.token_check()
    got = out[1:].as_strided((m, n), (out_stride, 1), 1)
    check_matmul(a[shift:].as_strided((m, k), (a_stride, 1), shift), w[shift:].as_strided((n, k), (w_stride, 1), shift), sa, sw, None, got, 'f32')
    touched = torch.zeros(out.shape, dtype=torch.bool, device='cuda')
    touched.as_strided((m, n), (out_stride, 1), 1).fill_(True)
    assert (out[~touched] == 3).all()


# ------------------------------------------------------------------------------------------------ cache
class Served:
    """A paged cache and the sequences of a step, every buffer with room behind it that has to keep its bytes."""

    def __init__(self, lengths, news, kv_heads, size, page, dtype, heads=None, seed=1, spare=2, one_each=False, extra_rows=3):
        g = self.g = gen(seed)
        self.lengths, self.news, self.page, self.size, self.kv_heads, self.dtype = lengths, news, page, size, kv_heads, dtype
        self.heads = heads or kv_heads
        need = [max(1, -(-n // page)) for n in lengths]
        self.row = max(need) + 1
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at:at + n] + [2 ** 31 - 1 - at] * (self.row - n))     # nothing may look behind a sequence's pages
            at += n
        self.starts = [0]
        for n in news:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1]
        shape = (self.pages, kv_heads, page, size)
        self.k, self.v = (torch.randint(-127, 128, shape, device='cuda', generator=g).to(torch.int8) for _ in range(2))
        self.k_scales, self.v_scales = (0.01 * (0.5 + torch.rand(shape[:2], device='cuda', generator=g)) for _ in range(2))
        width = (self.heads + 2 * kv_heads) * size
        self.joint = normal(self.tokens + extra_rows, width, g=g).to(TYPES[dtype])
        self.q = self.joint[:, :self.heads * size].unflatten(1, (self.heads, size))
        self.new_k = self.joint[:, self.heads * size:(self.heads + kv_heads) * size].unflatten(1, (kv_heads, size))
        self.new_v = self.joint[:, (self.heads + kv_heads) * size:].unflatten(1, (kv_heads, size))
        self.device_table = torch.tensor(self.table, dtype=torch.int32, device='cuda')
        self.device_lengths = torch.tensor(lengths, dtype=torch.int32, device='cuda')
        self.device_starts = None if one_each else torch.tensor(self.starts, dtype=torch.int32, device='cuda')
        self.cache = runtime.KvCache(self.k.data_ptr(), self.v.data_ptr(), self.k_scales.data_ptr(), self.v_scales.data_ptr(), self.pages, kv_heads, page,
                                     size)
        self.batch = runtime.KvBatch(len(lengths), self.device_table.data_ptr(), self.row, self.device_lengths.data_ptr(), self.tokens,
                                     max(news + [1]), None if one_each else self.device_starts.data_ptr())

    def append(self, **more):
        self.cache.append(self.batch, self.new_k.data_ptr(), self.new_v.data_ptr(), self.joint.stride(0), dtype=self.dtype, **more)

    def attention(self, out=None, scale=None, **more):
        if out is None:
            out = torch.full((self.tokens + 3, self.heads, self.size), 3.0, dtype=TYPES[self.dtype], device='cuda')
        self.cache.attention(self.batch, self.q.data_ptr(), out.data_ptr(), self.heads, scale or self.size ** -0.5, dtype=self.dtype,
                             q_stride=self.joint.stride(0), **more)
        return out


def check_append(s, before, after, scales_before, scales_after, new):
    """One of keys and values: codes and scales before and after against the definition in 64 bits."""
    want_codes, want_scales = before.clone().double(), scales_before.clone().double()
    loose = torch.zeros_like(want_codes)
    for b, (end, n) in enumerate(zip(s.lengths, s.news)):
        begin = end - n
        for p in range(max(begin, 0) // s.page, -(-end // s.page) if n else 0):
            number = s.table[b][p]
            if not 0 <= number < s.pages:
                continue
            lo, hi = max(begin, p * s.page), min(end, (p + 1) * s.page)
            x = new[s.starts[b] + lo - begin:s.starts[b] + hi - begin].double().transpose(0, 1)
            held = scales_before[number].double() if lo > p * s.page else torch.zeros(s.kv_heads, dtype=torch.float64, device='cuda')
            step = x.abs().amax((1, 2)) / 127
            grown = torch.maximum(held, torch.where(step <= TINY, 0.0, step))
            want_scales[number] = grown
            inside = torch.where(grown > 0, grown, 1.0)[:, None, None]
            old, fresh = slice(0, lo - p * s.page), slice(lo - p * s.page, hi - p * s.page)
            want_codes[number, :, old] = before[number, :, old].double() * (held[:, None, None] / inside)
            want_codes[number, :, fresh] = x / inside
            # rounded to whole numbers, behind a scale, its reciprocal or quotient and a product in 32 bits
            loose[number, :, :hi - p * s.page] = 0.5 + 127 * 5 * U
    assert ((scales_after.double() - want_scales).abs() <= want_scales.abs() * 2 * U).all()
    assert ((after.double() - want_codes).abs() <= loose).all()


CACHES = [(1, 64, 16, 'f16'), (2, 128, 16, 'bf16'), (3, 64, 32, 'bf16'), (2, 128, 64, 'f16'), (1, 128, 128, 'bf16'), (2, 64, 128, 'f16')]


@pytest.mark.parametrize('lengths, news', [([1], [1]), ([5, 0, 17, 64], [1, 1, 1, 1]), ([40, 200, 129], [40, 7, 128]), ([130, 0, 3, 257], [1, 0, 3, 200]),
                                           ([4, 33], [9, 2])])
@pytest.mark.parametrize('kv_heads, size, page, dtype', CACHES)
def test_append(lengths, news, kv_heads, size, page, dtype):
    s = Served(lengths, news, kv_heads, size, page, dtype, seed=len(lengths) + page)
    for big in (1.0, 30.0):       # the second time the new values are larger than what the pages hold: every scale grows
        s.joint.mul_(big)
        k, v, ks, vs = s.k.clone(), s.v.clone(), s.k_scales.clone(), s.v_scales.clone()
        s.append()
        check_append(s, k, s.k, ks, s.k_scales, s.new_k)
        check_append(s, v, s.v, vs, s.v_scales, s.new_v)


def test_append_one_token_each_without_starts():
    s = Served([5, 0, 17, 64], [1, 1, 1, 1], 2, 128, 32, 'bf16', one_each=True)
    k, ks = s.k.clone(), s.k_scales.clone()
    s.append()
    check_append(s, k, s.k, ks, s.k_scales, s.new_k)


def test_append_token_by_token_reads_as_what_went_in():
    """A page filled a token at a time: each growth of its scale costs at most half a step of the scale it grows to."""
    s = Served([0], [1], 1, 64, 64, 'bf16', one_each=True)
    s.device_table[0, 0] = s.table[0][0] = 0
    tokens = normal(64, 64, g=s.g).bfloat16() * torch.linspace(0.2, 3.0, 64, device='cuda')[:, None].bfloat16()
    growths, top = 0, 0.0
    for t in range(64):
        s.device_lengths[0] = t + 1
        s.new_k[0, 0], s.new_v[0, 0] = tokens[t], -tokens[t]
        s.append()
        growths += float(tokens[t].abs().max()) > top
        top = max(top, float(tokens[t].abs().max()))
    assert abs(float(s.k_scales[0, 0]) - top / 127) <= top * U
    off = (s.k[0, 0].double() * s.k_scales[0, 0].double() - tokens.double()).abs().max()
    assert off <= (growths + 1) * 0.5 * top / 127 * 1.001
    assert torch.equal(s.k[0, 0], -s.v[0, 0])


def test_append_values_that_are_not_finite_or_nothing():
    s = Served([20, 20, 20], [20, 20, 20], 1, 64, 16, 'bf16')
    s.new_k[3, 0, 5] = math.inf
    s.new_k[20 + 17, 0, 5] = math.nan
    s.new_k[40:56] = 0
    s.new_v[40:56] = 1e-38
    s.append()
    values = s.k.float() * s.k_scales[..., None, None]
    page = [[int(n) for n in row] for row in s.table]
    assert values[page[0][0]].isnan().all() and values[page[0][1], :, :4].isfinite().all()
    assert values[page[1][0]].isfinite().all() and values[page[1][1]].isnan().all()
    assert (s.k_scales[page[2][0]] == 0).all() and (s.k[page[2][0]] == 0).all()
    assert (s.v_scales[page[2][0]] == 0).all() and (s.v[page[2][0]] == 0).all()


# ------------------------------------------------------------------------------------------------ attention
def check_attention(s, out, causal=True, window=0, scale=None, poisoned=()):
    scale = scale or s.size ** -0.5
    group = s.heads // s.kv_heads
    for b, (end, n) in enumerate(zip(s.lengths, s.news)):
        got = out[s.starts[b]:s.starts[b] + n].double()
        if b in poisoned or not n:
            continue
        if not end:
            assert (got == 0).all()
            continue
        used = torch.tensor(s.table[b][:-(-end // s.page)], device='cuda')
        position = torch.arange(end - n, end, device='cuda')[:, None]
        j = torch.arange(end, device='cuda')[None]
        seen = torch.ones((n, end), dtype=torch.bool, device='cuda')
        if causal:
            seen = j <= position
            if window:
                seen &= j > position - window
        for h in range(s.heads):
            codes_v = s.v[used, h // group].double().flatten(0, 1)[:end]
            sv = s.v_scales[used, h // group].double().repeat_interleave(s.page)[:end]
            k = (s.k[used, h // group].double() * s.k_scales[used, h // group].double()[:, None, None]).flatten(0, 1)[:end]
            q = s.q[s.starts[b]:s.starts[b] + n, h].double()
            scores = (q @ k.T * scale).masked_fill(~seen, -math.inf)
            top = scores.amax(1, keepdim=True).clamp(min=-1e300)
            p = torch.exp(scores - top)
            total = p.sum(1, keepdim=True)
            share = torch.where(total > 0, p / total, 0.0)
            want = share @ (codes_v * sv[:, None])
            # scores: the products' sum in 32 bits, a rounding for each of its terms (tensor cores cut instead: a whole step), queries rounded to 11 bits
            # only below 2^-14 of their row's largest, three operations behind it
            reach = (q.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0).amax(1, keepdim=True)
            delta = reach * (s.size + 8) * 2 * U + scale * q.abs().amax(1, keepdim=True) * k.abs().sum(1).max() * 2.0 ** -25
            # a probability: the score's error twice (sum and product), 2^-22 of each exponential, 11 bits; sums over the tokens in steps
            # of 16 and a rescaling for each 32 (as many exponentials), joined over warps and blocks
            relative = 2 * delta + 2.0 ** -11 + (end / 16 + 100) * 4 * U
            # below 2^-14 of the largest the 16-bit probabilities have steps of 2^-24
            weighted = share * sv
            floor = 2.0 ** -25 * weighted.amax(1, keepdim=True) * codes_v.abs().sum(0)[None]
            bound = relative * (share @ (codes_v.abs() * sv[:, None])) + floor + half_step(s.dtype) * want.abs() * 1.01 + 2.0 ** -25
            off = (got[:, h] - want).abs()
            assert (off <= bound).all(), f'sequence {b} head {h}: {float((off - bound).max())} over, off {float(off.max())}'
    assert (out[s.tokens:] == 3).all()           # rows behind the last sequence


@pytest.mark.parametrize('kv_heads, size, page, dtype', CACHES)
@pytest.mark.parametrize('group', [1, 4, 5, 16, 24])
def test_attention_single_tokens(group, kv_heads, size, page, dtype):
    s = Served([1, 0, 17, 31, 32, 33, 100, 515], [1] * 8, kv_heads, size, page, dtype, heads=kv_heads * group, one_each=True, seed=group)
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('lengths', [[4000], [2000, 1, 4097], [127], [128], [129, 511]])
@pytest.mark.parametrize('size, page, dtype', [(128, 64, 'bf16'), (64, 16, 'f16'), (128, 16, 'f16')])
def test_attention_long_contexts(lengths, size, page, dtype):
    s = Served(lengths, [1] * len(lengths), 2, size, page, dtype, heads=8, one_each=True)
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('lengths, news', [([1], [1]), ([40, 0, 130], [40, 0, 2]), ([300, 64, 257], [129, 64, 1]), ([700], [700]), ([1000, 33], [300, 33]),
                                           ([513, 128, 90], [128, 128, 5])])
@pytest.mark.parametrize('kv_heads, size, page, dtype', CACHES)
@pytest.mark.parametrize('mode', ['causal', 'window', 'all'])
def test_attention_prompts(lengths, news, kv_heads, size, page, dtype, mode):
    s = Served(lengths, news, kv_heads, size, page, dtype, heads=kv_heads * 4)
    more = dict(causal=mode != 'all', window=50 if mode == 'window' else 0)
    out = s.attention(**more)
    runtime.token_check()
    check_attention(s, out, **more)


@pytest.mark.parametrize('window', [1, 2, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize('news', [[1, 1], [3, 40]])
def test_attention_windows(window, news):
    s = Served([300, 71], news, 2, 128, 64, 'bf16', heads=6)
    out = s.attention(window=window)
    check_attention(s, out, window=window)


@pytest.mark.parametrize('size', [64, 128])
def test_attention_queries_before_the_first_token_give_zeros(size):
    """More new tokens than the sequence holds: the first ones stand before position 0 and see nothing."""
    s = Served([5, 64], [9, 70], 1, size, 16, 'bf16', heads=2)
    out = s.attention()
    assert (out[:4] == 0).all() and (out[9:15] == 0).all()
    check_attention(s, out)


@pytest.mark.parametrize('news', [[1, 1, 1], [5, 40, 33]])
@pytest.mark.parametrize('size', [64, 128])
def test_attention_scales_of_any_size(news, size):
    """Pages whose scales lie far apart, one of zeros, and what is no number where no query looks."""
    s = Served([200, 150, 100], news, 1, size, 32, 'bf16', heads=4)
    s.v_scales.mul_(10.0 ** torch.randint(-6, 7, s.v_scales.shape, device='cuda', generator=s.g))
    s.k_scales[s.table[0][1]] *= 40
    s.v_scales[s.table[0][2]] = 0
    s.v[s.table[0][2]] = 0
    free = [n for n in range(s.pages) if n not in [x for row in s.table for x in row]]
    s.k_scales[free] = math.nan
    s.v_scales[free] = math.inf
    out = s.attention()
    check_attention(s, out)


@pytest.mark.parametrize('order', ['rising', 'falling', 'jumping'])
@pytest.mark.parametrize('size, page, new', [(128, 64, 1), (128, 16, 3), (64, 32, 1), (128, 64, 130), (128, 16, 70), (64, 16, 200)])
def test_attention_maxima_that_move(size, page, new, order):
    """Keys along the query, of scales that rise (or fall, or jump) from page to page: the maximum moves again and again, inside a step and between steps."""
    s = Served([1500], [new], 1, size, page, 'bf16', heads=2)
    used = s.table[0][:-(-1500 // page)]
    s.k[used] = torch.where(s.q[0, 0] > 0, 1, -1).to(torch.int8) * torch.randint(1, 128, (len(used), 1, page, 1), device='cuda', generator=s.g).to(torch.int8)
    rise = torch.linspace(0.01, 6.0, len(used), device='cuda')
    if order == 'falling':
        rise = rise.flip(0)
    if order == 'jumping':
        rise = rise[torch.randperm(len(used), device='cuda', generator=s.g)]
    s.k_scales[used] = (rise / size ** 0.5)[:, None]
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


def test_attention_prompt_of_many_tiles():
    """More rows than the other kernel's grid holds."""
    s = Served([300], [300], 1, 64, 64, 'f16', heads=4)
    s.batch.desc.max_new = 2 ** 19       # as a caller that knows no better bound
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('kv_heads, new', [(8, 300), (1, 1)])
def test_attention_small_probabilities_beside_a_large_one_of_nothing(kv_heads, new):
    """What is left when the token that nearly has it all holds zeros: probabilities of e^-10 to e^-16."""
    s = Served([3], [new], kv_heads, 64, 16, 'f16', heads=4 * kv_heads)
    page, signs = s.table[0][0], torch.where(torch.arange(64, device='cuda') % 3 == 0, -1.0, 1.0)
    s.k_scales.fill_(1 / 127)
    s.k[page, :, 0] = (127 * signs).to(torch.int8)
    s.v_scales.fill_(5.0)
    s.v[page, :, 0] = 0
    s.q.copy_((1 + 0.5 * torch.rand(s.q.shape[:2] + (1,), device='cuda', generator=s.g)) * signs)
    out = s.attention(scale=1 / 6, causal=False)
    runtime.token_check()
    check_attention(s, out, causal=False, scale=1 / 6)


@pytest.mark.parametrize('new', [1, 40])
@pytest.mark.parametrize('size', [64, 128])
def test_attention_of_a_negative_scale(new, size):
    s = Served([300, 41], [new, new], 2, size, 32, 'bf16', heads=8)
    out = s.attention(scale=-0.1)
    s.q.neg_()
    check_attention(s, out, scale=0.1)


@pytest.mark.parametrize('power', [-120, -30, 30, 120])
@pytest.mark.parametrize('new', [1, 40])
def test_attention_queries_of_any_size(power, new):
    s = Served([200], [new], 1, 128, 64, 'bf16', heads=2)
    s.q.mul_(2.0 ** power)
    out = s.attention(scale=2.0 ** -power * 0.09)
    check_attention(s, out, scale=2.0 ** -power * 0.09)


@pytest.mark.parametrize('new', [1, 40])
def test_attention_what_is_no_number_stays_in_its_row(new):
    s = Served([200, 90], [new, 1], 2, 64, 16, 'f16', heads=4)
    clean = s.attention()
    s.q[0, 1, 3] = math.nan
    out = s.attention()
    assert out[0, 1].isnan().all()
    same = torch.ones(out.shape[:2], dtype=torch.bool, device='cuda')
    same[0, 1] = False
    assert torch.equal(out[same], clean[same])


@pytest.mark.parametrize('which', ['k_scales', 'v_scales'])
@pytest.mark.parametrize('page, new, heads', [(16, 40, 1), (16, 12, 1), (64, 100, 2), (32, 60, 8), (128, 200, 4)])
def test_attention_a_poisoned_page_reaches_those_who_see_it(page, new, heads, which):
    s = Served([300], [new], 1, 128, page, 'bf16', heads=heads)
    clean = s.attention()
    last = 299 // page              # the page of the last token
    getattr(s, which)[s.table[0][last]] = math.nan
    out = s.attention()
    unaware = max(0, min(new, last * page - (300 - new)))
    assert torch.equal(out[:unaware], clean[:unaware])
    assert out[unaware:new].isnan().all()
    assert (out[new:] == 3).all()


@pytest.mark.parametrize('bad', [-1, -2 ** 31, 2 ** 31 - 1, None])
@pytest.mark.parametrize('news', [[1, 1, 1], [40, 5, 7]])
@pytest.mark.parametrize('page', [16, 64])
def test_bad_pages_and_lengths_touch_nothing(bad, news, page):
    """A page number outside the cache, or a length behind the row of the table: the queries that see it become no numbers, the rest stays."""
    s = Served([200, 150, 90], news, 2, 128, page, 'bf16', heads=4)
    clean = s.attention()
    if bad is None:
        s.device_lengths[1] = s.row * page + 4000
    else:
        s.device_table[1, 0] = bad
    out = s.attention()
    runtime.token_check()
    one, two = s.starts[1], s.starts[2]
    assert out[one:two].isnan().all()
    assert torch.equal(out[:one], clean[:one]) and torch.equal(out[two:], clean[two:])
    if bad is not None:
        s.device_table[1] = bad
    k, ks = s.k.clone(), s.k_scales.clone()
    s.append()
    torch.cuda.synchronize()
    mine = [n for n in s.table[1] if 0 <= n < s.pages]
    assert torch.equal(s.k[mine], k[mine]) and torch.equal(s.k_scales[mine], ks[mine])


def test_starts_beyond_the_rows_are_cut():
    s = Served([64, 64], [4, 4], 1, 64, 16, 'bf16')
    s.device_starts.copy_(torch.tensor([0, 2 ** 31 - 1, -5], dtype=torch.int32))
    out = s.attention()
    s.append()
    runtime.token_check()
    assert (out[s.tokens:] == 3).all()


# ------------------------------------------------------------------------------------------------ together
def layer(s, x, residual, w_norm, w_joint, w_scales, w_out, w_out_scales, buffers, stream=0):
    """A layer's attention half as a server runs it: norm, joint projection, append, attention, norm of the result, projection back."""
    codes, scales, total, codes2, scales2, out, back = buffers
    rows, width = x.shape
    joint = s.joint.shape[1]
    inner = s.heads * s.size
    runtime.rmsnorm_quantize(x.data_ptr(), rows, width, w_norm.data_ptr(), codes.data_ptr(), scales.data_ptr(), residual.data_ptr(), total.data_ptr(),
                             dtype=s.dtype, stream=stream)
    runtime.matmul_i8(codes.data_ptr(), scales.data_ptr(), w_joint.data_ptr(), w_scales.data_ptr(), s.joint.data_ptr(), rows, joint, width, dtype=s.dtype,
                      stream=stream)
    s.append(stream=stream)
    s.attention(out, stream=stream)
    runtime.rmsnorm_quantize(out.data_ptr(), rows, inner, None, codes2.data_ptr(), scales2.data_ptr(), dtype=s.dtype, stream=stream)
    runtime.matmul_i8(codes2.data_ptr(), scales2.data_ptr(), w_out.data_ptr(), w_out_scales.data_ptr(), back.data_ptr(), rows, width, inner, dtype='f32',
                      stream=stream)


def make_layer(lengths, news, dtype='bf16', **more):
    s = Served(lengths, news, 2, 64, 32, dtype, heads=8, extra_rows=0, **more)
    g, rows, width = s.g, s.tokens, 512
    x, residual = normal(rows, width, g=g).to(TYPES[dtype]), normal(rows, width, g=g).to(TYPES[dtype])
    w_norm = (1 + 0.1 * normal(width, g=g)).to(TYPES[dtype])
    w_joint, w_out = codes_of(s.joint.shape[1], width, g), codes_of(width, 512, g)
    w_scales = torch.rand(s.joint.shape[1], device='cuda', generator=g) / (74 * math.sqrt(width))
    w_out_scales = torch.rand(width, device='cuda', generator=g) / (74 * math.sqrt(512))
    buffers = (torch.empty((rows, width), dtype=torch.int8, device='cuda'), torch.empty(rows, device='cuda'), torch.empty_like(x),
               torch.empty((rows, 512), dtype=torch.int8, device='cuda'), torch.empty(rows, device='cuda'),
               torch.empty((rows, 8, 64), dtype=TYPES[dtype], device='cuda'), torch.empty((rows, width), device='cuda'))
    return s, (x, residual, w_norm, w_joint, w_scales, w_out, w_out_scales, buffers)


@pytest.mark.parametrize('lengths, news', [([70, 33, 1], [1, 1, 1]), ([70, 33], [70, 9])])
def test_a_layer(lengths, news):
    s, args = make_layer(lengths, news)
    x, residual, w_norm, w_joint, w_scales, w_out, w_out_scales, (codes, scales, total, codes2, scales2, out, back) = args
    k, ks = s.k.clone(), s.k_scales.clone()
    v, vs = s.v.clone(), s.v_scales.clone()
    layer(s, *args)
    runtime.token_check()
    # each step against 64 bits from what the step before it left
    check_norm(total, w_norm, codes, scales, s.dtype, 1e-6)
    check_matmul(codes, w_joint, scales, w_scales, None, s.joint, s.dtype)
    check_append(s, k, s.k, ks, s.k_scales, s.new_k)
    check_append(s, v, s.v, vs, s.v_scales, s.new_v)
    check_attention(s, torch.cat([out, torch.full_like(out[:1], 3)]))
    check_norm(out.flatten(1), None, codes2, scales2, s.dtype, 1e-6)
    check_matmul(codes2, w_out, scales2, w_out_scales, None, back, 'f32')


def test_a_layer_captured_and_replayed():
    """A step captured once and replayed with other contents gives what direct calls give, bit for bit; two graphs share nothing but the inputs."""
    s, args = make_layer([70, 33, 1], [1, 1, 1])
    layer(s, *args)                      # loads the kernels
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(s, *args, stream=torch.cuda.current_stream().cuda_stream)
    buffers = args[-1]
    for shift in (0, 3):
        s.device_lengths += shift
        args[0].normal_(generator=s.g)
        held = [t.clone() for t in (s.k, s.v, s.k_scales, s.v_scales)]
        layer(s, *args)
        torch.cuda.synchronize()
        want = [t.clone() for t in buffers + (s.k, s.v, s.k_scales, s.v_scales)]
        for t, old in zip((s.k, s.v, s.k_scales, s.v_scales), held):
            t.copy_(old)
        for t in buffers:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(buffers + (s.k, s.v, s.k_scales, s.v_scales), want))


def test_two_streams_at_once():
    layers = [make_layer([70, 33, 1], [1, 1, 1], seed=3), make_layer([400, 120], [200, 64], seed=4)]
    want = []
    for s, args in layers:
        layer(s, *args)
        torch.cuda.synchronize()
        want.append(args[-1][-1].clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (s, args), stream in zip(layers, streams):
            layer(s, *args, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for (s, args), w in zip(layers, want):
        assert torch.equal(args[-1][-1], w)       # appending the same tokens again changes nothing


def test_a_wait_that_runs_out_is_reported_once():
    runtime.token_check()
    runtime.token_selftest_wait_timeout(1000)
    with pytest.raises(runtime.N2D2BError, match='gave up'):
        runtime.token_check()
    runtime.token_check()


def test_long_cache_offsets_leave_32_bits():
    """A pool of more than 2^32 bytes of keys: the sequence's pages lie at its end."""
    pages, heads, page, size = 530000, 1, 64, 128
    k = torch.zeros((pages, heads, page, size), dtype=torch.int8, device='cuda')
    v = torch.zeros_like(k)
    ks, vs = torch.zeros((pages, heads), device='cuda'), torch.zeros((pages, heads), device='cuda')
    s = Served([130], [130], heads, size, page, 'bf16', heads=2)
    last = [pages - 1, pages - 3, pages - 2]
    s.k, s.v, s.k_scales, s.v_scales, s.pages = k, v, ks, vs, pages
    s.cache = runtime.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, page, size)
    s.table = [last]
    s.row = 3
    s.device_table = torch.tensor(s.table, dtype=torch.int32, device='cuda')
    s.batch = runtime.KvBatch(1, s.device_table.data_ptr(), 3, s.device_lengths.data_ptr(), s.tokens, 130, s.device_starts.data_ptr())
    s.append()
    out = s.attention()
    runtime.token_check()
    assert not k[:1000].any() and bool(k[last].any())
    check_attention(s, out)


def nothing(s, b, places):
    """Values of zero at places [lo, hi) of sequence b, as append leaves them: where a whole page has none its scale is 0."""
    for lo, hi in places:
        for t in range(lo, hi, s.page):
            assert lo % s.page == 0
            n = min(s.page, hi - t)
            s.v[s.table[b][t // s.page], :, :n] = 0
            if n == s.page or t + n >= s.lengths[b]:
                s.v_scales[s.table[b][t // s.page]] = 0


@pytest.mark.parametrize('new', [1, 3, 40, 300])
@pytest.mark.parametrize('size, page, length, places', [
    (128, 64, 256, [(0, 128)]), (64, 16, 512, [(0, 256)]), (128, 64, 512, [(256, 512)]), (64, 128, 1024, [(0, 512)]), (128, 64, 2000, [(0, 64), (128, 1984)]),
    (128, 64, 8000, [(0, 4032)]), (64, 64, 8192, [(0, 4608)]), (128, 128, 12000, [(256, 11904)]), (64, 32, 12000, [(0, 64), (96, 12000)]),
    (128, 16, 300, [(0, 300)])])
def test_attention_over_stretches_of_zeros(size, page, length, places, new):
    """Tokens whose values are zero have the scale 0 and take their share of the softmax all the same."""
    s = Served([length, 77], [new, new], 1, size, page, 'f16', heads=4)
    nothing(s, 0, places)
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('lengths', [[256] * 3, [600] * 40, [2047] * 80])
def test_attention_over_zeros_in_every_split(lengths):
    """Zeros over the first half of each of many sequences, so that the tokens are cut into few streams."""
    s = Served(lengths, [1] * len(lengths), 8, 64, 64, 'bf16', heads=8, one_each=True)
    for b, n in enumerate(lengths):
        nothing(s, b, [(0, n // 2 // 64 * 64)])
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('new', [1, 40, 300])
@pytest.mark.parametrize('power', [-90, -60, 60, 110, 120])
def test_attention_values_of_any_size(power, new):
    """Every scale of the values times a power of two: the outputs are times that power."""
    s = Served([700, 77], [new, min(new, 77)], 2, 128, 64, 'bf16', heads=8)
    s.v_scales.mul_(2.0 ** power)
    out = s.attention()
    runtime.token_check()
    s.v_scales.mul_(2.0 ** -power)
    real = out[:s.tokens].double() * 2.0 ** -power
    check_attention(s, torch.cat([real, out[s.tokens:].double()]))


@pytest.mark.parametrize('new', [1, 40])
def test_attention_values_of_nearly_nothing_beside_others(new):
    """Scales of 2^-97 take their share of the softmax as scales of zero do."""
    s = Served([3000, 77], [new, new], 1, 128, 64, 'f16', heads=4)
    s.v_scales[s.table[0][:40]] = 2.0 ** -97
    out = s.attention()
    runtime.token_check()
    check_attention(s, out)


@pytest.mark.parametrize('share', [0.9, 0.99, 0.999])
@pytest.mark.parametrize('size, length, new, batch', [(64, 3000, 1, 1), (128, 3000, 2, 1), (64, 500, 4, 40), (128, 1800, 1, 160), (64, 4000, 2, 160)])
def test_attention_of_single_tokens_beside_one_of_nothing(size, length, new, batch, share):
    """A first token that takes nearly all of a row and holds zeros: what the others give is as exact as without it."""
    s = Served([length] * batch, [new] * batch, 1, size, 64, 'f16', heads=4)
    # the first key stands along the queries, the others across them: equal scores but for a little
    s.q.copy_(torch.where(torch.arange(size, device='cuda') < size // 2, 1.0, 0.01 * normal(size, g=s.g)).half())
    first = [row[0] for row in s.table]
    s.k[:, :, :, :size // 2] = 0
    s.k_scales.fill_(0.02)
    s.k[first, :, 0, :size // 2], s.k[first, :, 0, size // 2:] = 100, 0
    s.v[first, :, 0] = 0
    s.v_scales.fill_(13.0)
    scale = math.log(share / (1 - share) * length) / (100 * 0.02 * (size // 2))
    out = s.attention(scale=scale, causal=False)
    runtime.token_check()
    for b in {0, batch // 2, batch - 1}:
        used = s.table[b][:-(-length // 64)]
        q, got = s.q[b * new:(b + 1) * new].double(), out[b * new:(b + 1) * new].double()
        k = (s.k[used, 0].double() * s.k_scales[used, 0].double()[:, None, None]).flatten(0, 1)[:length]
        v = (s.v[used, 0].double() * s.v_scales[used, 0].double()[:, None, None]).flatten(0, 1)[:length]
        p = torch.softmax(q @ k.T * scale, 2)
        want = p @ v
        # scores as in check_attention (queries of 22 bits are exact here); 2^-22 of each exponential and of the scale's logarithm, sums in 32 bits; a
        # probability is off by 2^-29 of the largest, half the step of a whole number of which the largest has 2^28
        delta = (q.abs() @ k.abs().T * scale).amax(2, keepdim=True) * (size + 8) * 2 * U
        relative = 2 * delta + 4 * 2.0 ** -21 + (length / 128 + 100) * U
        bound = relative * (p @ v.abs()) + 2.0 ** -29 * p.amax(2, keepdim=True) * v.abs().sum(0) + half_step('f16') * want.abs() * 1.01 + 2.0 ** -25
        off = (got - want).abs()
        assert (off <= bound).all(), (b, float((off - bound).max()), float((off / want.abs().mean()).max()))


@pytest.mark.parametrize('order', ['rising', 'falling', 'jumping', 'rising by little'])
@pytest.mark.parametrize('size, page, heads, new, batch', [(128, 16, 16, 400, 1), (64, 32, 16, 1000, 1), (128, 16, 8, 300, 20), (64, 16, 4, 600, 40)])
def test_attention_of_many_rows_whose_maxima_move_within_a_step(size, page, heads, new, batch, order):
    """Scores that change every 16 or 32 tokens of a step of 128, by far more (or by about as much) as leaves the maximum where it is: what the tokens before gave
    is rescaled again and again, inside the step and in the output so far.  Tokens over clusters of 4 and of 2 blocks, and undivided."""
    length = 1000
    s = Served([length] * batch, [new] * batch, 1, size, page, 'bf16', heads=heads)
    s.q.copy_(s.q[:1, :1].sign())
    s.k.copy_((s.q[0, 0] * 100).to(torch.int8))
    steps = -(-length // page)
    rise = torch.arange(steps, device='cuda') * (3.0 if order == 'rising by little' else 14.0)
    if order == 'falling':
        rise = rise.flip(0)
    if order == 'jumping':
        rise = rise[torch.randperm(steps, device='cuda', generator=s.g)]
    for row in s.table:
        s.k_scales[row[:steps]] = (rise / (100 * size ** 0.5))[:, None]
    out = s.attention(causal=False)
    runtime.token_check()
    check_attention(s, out, causal=False)


@pytest.mark.parametrize('window', [1, 2, 3, 15, 16, 17, 40])
@pytest.mark.parametrize('size, page', [(64, 16), (128, 16), (128, 64)])
@pytest.mark.parametrize('which', ['k_scales', 'v_scales', 'table'])
def test_attention_a_window_that_ends_in_a_poisoned_page(which, size, page, window):
    """Every place of a page at a window's lower edge: no number for those who see the page, the same bits for all others."""
    new = 1000 if window < 40 else 40
    s = Served([1100], [new], 2, size, page, 'bf16', heads=8)
    clean = s.attention(window=window)
    bad = 1 + 1080 // page // 2 * 2 - 2
    bad = min(bad, 1099 // page)
    if which == 'table':
        s.device_table[0, bad] = s.pages
    else:
        getattr(s, which)[s.table[0][bad]] = math.nan
    out = s.attention(window=window)
    runtime.token_check()
    position = torch.arange(1100 - new, 1100, device='cuda')
    sees = (position >= bad * page) & (position - window < (bad + 1) * page - 1)
    assert sees.any()
    assert out[:new][sees].isnan().all()
    assert torch.equal(out[:new][~sees], clean[:new][~sees])


@pytest.mark.parametrize('window', [1, 2, 5])
@pytest.mark.parametrize('new', [16, 1000])
def test_attention_queries_that_are_no_number_in_narrow_windows(new, window):
    s = Served([1000], [new], 2, 128, 64, 'bf16', heads=8)
    clean = s.attention(window=window)
    s.q[:, [1, 6], 7] = math.nan
    out = s.attention(window=window)
    runtime.token_check()
    assert out[:new, [1, 6]].isnan().all()
    keep = [0, 2, 3, 4, 5, 7]
    assert torch.equal(out[:new, keep], clean[:new, keep])


@pytest.mark.parametrize('what', [math.inf, -math.inf])
@pytest.mark.parametrize('window', [1, 2, 5, 0])
@pytest.mark.parametrize('new', [16, 1000])
def test_attention_queries_that_are_infinite(new, window, what):
    """An infinite query gives no numbers, as the few rows have it, not what one that sees nothing gives where all its scores are -inf."""
    s = Served([1000], [new], 2, 128, 64, 'bf16', heads=8)
    clean = s.attention(window=window)
    s.q[:, 6, 7] = what
    out = s.attention(window=window)
    runtime.token_check()
    assert out[:new, 6].isnan().all()
    keep = [0, 1, 2, 3, 4, 5, 7]
    assert torch.equal(out[:new, keep], clean[:new, keep])


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('columns', [64, 77, 4096, 20000])
@pytest.mark.parametrize('residual', [False, True])
def test_norm_rows_of_zeros_without_eps(columns, residual, dtype):
    """A scale of nothing is 0, whatever 0 / 0 is: a padded row, and one whose weights are zero where it is not."""
    x = torch.zeros((3, columns), device='cuda', dtype=TYPES[dtype])
    x[1, :5] = 2
    w = torch.ones(columns, device='cuda', dtype=TYPES[dtype])
    w[:5] = 0
    codes, scales = torch.full((3, columns), 5, dtype=torch.int8, device='cuda'), torch.full((3,), 9.0, device='cuda')
    r, total = torch.zeros_like(x), torch.ones_like(x)
    runtime.rmsnorm_quantize(x.data_ptr(), 3, columns, w.data_ptr(), codes.data_ptr(), scales.data_ptr(), r.data_ptr() if residual else None,
                             total.data_ptr() if residual else None, dtype=dtype, eps=0.0)
    assert (scales == 0).all() and (codes == 0).all()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('columns', [1, 77, 512, 4096, 20000])
@pytest.mark.parametrize('power', [-90, -75, -62, 50, 61, 63, 64, 100, 120])
@pytest.mark.parametrize('form', ['plain', 'weight', 'residual', 'in place'])
def test_norm_of_rows_of_any_size(form, power, columns, dtype):
    """Rows whose squares leave 32 bits on either side, without eps; beside them one of ordinary size."""
    g, t = gen(columns + 200 + power), TYPES[dtype]
    x = normal(3, columns, g=g).abs().add_(0.1).mul_(torch.where(normal(3, columns, g=g) < 0, -1.0, 1.0)).to(t)
    x[0] *= 2.0 ** power
    x[1] *= 2.0 ** power
    x[1, columns // 2:] = 0
    if columns == 1:
        x[1] = 2.0 ** power
    w = (1 + 0.3 * normal(columns, g=g)).to(t) if form == 'weight' else None
    r = torch.zeros_like(x)
    total = x if form == 'in place' else torch.ones_like(x)
    more = form in ('residual', 'in place')
    h = x.clone()
    codes, scales = torch.zeros((3, columns), dtype=torch.int8, device='cuda'), torch.zeros(3, device='cuda')
    runtime.rmsnorm_quantize(x.data_ptr(), 3, columns, w.data_ptr() if w is not None else None, codes.data_ptr(), scales.data_ptr(),
                             r.data_ptr() if more else None, total.data_ptr() if more else None, dtype=dtype, eps=0.0)
    check_norm(h, w, codes, scales, dtype, 0.0)


@pytest.mark.parametrize('held', [1e-45, 1e-40, 2.0 ** -127, 2.0 ** -110, 2.0 ** -100])
@pytest.mark.parametrize('fresh', [0.0, 2.0 ** -96, 1.0])
def test_append_onto_a_page_of_nearly_nothing(held, fresh):
    """A scale up to 2^-100 is 0, the one a page holds too: its codes become 0, as those of new values that small."""
    s = Served([20], [3], 2, 64, 32, 'bf16')
    s.k_scales.fill_(held)
    s.new_k[:] = fresh * normal(s.joint.shape[0], 2, 64, g=s.g).clamp(-1, 1).bfloat16()
    k = s.k.clone()
    s.append()
    number = s.table[0][0]
    assert (s.k[number, :, :17] == 0).all()
    if fresh < 1:
        assert (s.k_scales[number] == 0).all() and (s.k[number, :, 17:20] == 0).all()
    else:
        x = s.new_k[:3].double().transpose(0, 1)
        assert ((s.k[number, :, 17:20] * s.k_scales[number].double()[:, None, None] - x).abs() <= s.k_scales[number].double()[:, None, None] * 0.501).all()
    assert torch.equal(s.k[number, :, 20:], k[number, :, 20:])


@pytest.mark.parametrize('lengths, news', [([70, 33, 200], [1, 9, 40]), ([64], [64])])
def test_a_loose_bound_of_new_tokens_changes_nothing(lengths, news):
    s = Served(lengths, news, 2, 64, 16, 'bf16', heads=8)
    tight = Served(lengths, news, 2, 64, 16, 'bf16', heads=8)
    s.batch.desc.max_new = 2 ** 31 - 1
    tight.batch.desc.max_new = s.tokens
    k, v, ks, vs = s.k.clone(), s.v.clone(), s.k_scales.clone(), s.v_scales.clone()
    s.append()
    tight.append()
    out, want = s.attention(), tight.attention()
    runtime.token_check()
    check_append(s, k, s.k, ks, s.k_scales, s.new_k)
    check_append(s, v, s.v, vs, s.v_scales, s.new_v)
    check_attention(s, out)
    assert torch.equal(out, want) and torch.equal(s.k, tight.k) and torch.equal(s.v_scales, tight.v_scales)


# ------------------------------------------------------------------------------------------------ codes without a norm
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('columns, form', [(1, 'plain'), (77, 'residual'), (512, 'plain'), (4096, 'weight'), (4096, 'residual'), (20000, 'weight')])
@pytest.mark.parametrize('power', [-60, 0, 70])
def test_codes_without_a_norm(power, columns, form, dtype):
    if dtype == 'f16' and power:
        pytest.skip('16 bits do not hold them')
    g, t = gen(columns), TYPES[dtype]
    x, r = (normal(4, columns, g=g) * 2.0 ** power).to(t), (normal(4, columns, g=g) * 2.0 ** power).to(t)
    x[2] = r[2] = 0
    w = (1 + 0.3 * normal(columns, g=g)).to(t) if form == 'weight' else None
    total = torch.ones_like(x)
    codes, scales = torch.full((4, columns), 9, dtype=torch.int8, device='cuda'), torch.full((4,), 9.0, device='cuda')
    more = form == 'residual'
    runtime.rmsnorm_quantize(x.data_ptr(), 4, columns, w.data_ptr() if w is not None else None, codes.data_ptr(), scales.data_ptr(),
                             r.data_ptr() if more else None, total.data_ptr() if more else None, dtype=dtype, eps=0.0, skip_norm=True)
    h = (x.float() + r.float()).to(t) if more else x
    if more:
        assert torch.equal(total, h)
    u = h.double() * (1.0 if w is None else w.double())
    step = u.abs().amax(1) / 127
    # a product and the constant in 32 bits; the codes as in check_norm
    assert ((scales.double() - step).abs() <= step * 3 * U).all()
    assert (scales[2] == 0) and (codes[2] == 0).all()
    assert ((codes.double() - u / torch.where(step > 0, step, 1.0)[:, None]).abs() <= 0.5 + 127 * 5 * U).all()


@pytest.mark.parametrize('lengths, news', [([70, 33, 1], [1, 1, 1]), ([200, 90], [70, 90])])
def test_a_layer_against_the_layer_in_64_bits(lengths, news):
    """Norm, joint projection, append, attention and the projection back, as a user chains them, against the same layer without any rounding.

    What 8 bits cost: a rounding to a step s is noise of s / sqrt(12).  The largest of some hundred normal values is about 3.2 of their widths (of a page's 64 x 32, 3.7), so a
    step is 3.2 / 127 = 2.5 % of the width and its noise 0.7 % (0.9 % of a page's values, and as much again where its scale grows under old codes).  A product
    hands the relative noise of its input on as it is, and attention averages that of the values.  Three roundings one after the other: the normed input, keys and
    values, attention's output: sqrt(0.7^2 + 2 * 0.9^2 + 0.7^2) = 1.6 %, 0.3 % of bf16 beside it.  Scores are of the order of 1, so that the keys' and queries' own noise moves them by
    1 to 2 %, and the outputs by as much at most: 2.6 % in all.  A layer that takes another scale anywhere is off by tens of percent."""
    s, args = make_layer(lengths, news)
    x, residual, w_norm, w_joint, w_scales, w_out, w_out_scales, (codes, scales, total, codes2, scales2, out, back) = args
    rows, width = x.shape
    # a cache whose earlier tokens are of the size that the projection gives
    s.k_scales.mul_(1.5)
    s.v_scales.mul_(1.5)
    held = [(s.k.double() * s.k_scales.double()[..., None, None]), (s.v.double() * s.v_scales.double()[..., None, None])]
    joint = s.joint.shape[1]
    runtime.rmsnorm_quantize(x.data_ptr(), rows, width, w_norm.data_ptr(), codes.data_ptr(), scales.data_ptr(), residual.data_ptr(), total.data_ptr(),
                             dtype=s.dtype)
    runtime.matmul_i8(codes.data_ptr(), scales.data_ptr(), w_joint.data_ptr(), w_scales.data_ptr(), s.joint.data_ptr(), rows, joint, width, dtype=s.dtype)
    s.append()
    s.attention(out)
    runtime.rmsnorm_quantize(out.data_ptr(), rows, s.heads * s.size, None, codes2.data_ptr(), scales2.data_ptr(), dtype=s.dtype, skip_norm=True)
    runtime.matmul_i8(codes2.data_ptr(), scales2.data_ptr(), w_out.data_ptr(), w_out_scales.data_ptr(), back.data_ptr(), rows, width, s.heads * s.size, dtype='f32')
    runtime.token_check()

    h = x.double() + residual.double()
    n = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * w_norm.double()
    j = n @ (w_joint.double() * w_scales.double()[:, None]).T
    q, k, v = j.split([s.heads * s.size, s.kv_heads * s.size, s.kv_heads * s.size], 1)
    attended = torch.zeros(rows, s.heads, s.size, dtype=torch.float64, device='cuda')
    for b, (end, new) in enumerate(zip(lengths, news)):
        used, at = s.table[b][:-(-end // s.page)], slice(s.starts[b], s.starts[b] + new)
        full = []
        for pool, fresh in zip(held, (k, v)):
            t = pool[used].transpose(1, 2).flatten(0, 1)[:end].clone()          # [token][head][size]
            t[end - new:] = fresh[at].unflatten(1, (s.kv_heads, s.size))
            full.append(t.repeat_interleave(s.heads // s.kv_heads, 1))
        scores = torch.einsum('thd,jhd->htj', q[at].unflatten(1, (s.heads, s.size)), full[0]) * s.size ** -0.5
        hidden = torch.arange(end, device='cuda')[None] > torch.arange(end - new, end, device='cuda')[:, None]
        attended[at] = torch.einsum('htj,jhd->thd', torch.softmax(scores.masked_fill(hidden, -math.inf), 2), full[1])
    want = attended.flatten(1) @ (w_out.double() * w_out_scales.double()[:, None]).T
    off = (back.double() - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert off <= 0.026, float(off)


@pytest.mark.parametrize('columns', [5, 512, 4095])
@pytest.mark.parametrize('power, lift', [(-120, 40), (-125, 60), (-100, 10), (-135, 100)])
def test_norm_of_the_smallest_rows_under_large_weights(power, lift, columns):
    g = gen(columns)
    x = (1 + normal(2, columns, g=g).abs()) * 2.0 ** power
    w = (1 + 0.3 * normal(columns, g=g)) * 2.0 ** lift
    codes, scales = torch.zeros((2, columns), dtype=torch.int8, device='cuda'), torch.zeros(2, device='cuda')
    runtime.rmsnorm_quantize(x.data_ptr(), 2, columns, w.data_ptr(), codes.data_ptr(), scales.data_ptr(), dtype='f32', eps=0.0)
    check_norm(x, w, codes, scales, 'f32', 0.0)


@pytest.mark.parametrize('levels', [(-26, -18, 0, -26), (-25.5, -17.5, -17, 0), (-30.5, -20, -17, 0), (-18, -18, 0, -18), (-30.5, -17, -30.5, 0), (-12, -16, -4, 0), (0, -18, -16, -17)])
@pytest.mark.parametrize('size', [64, 128])
def test_attention_of_many_rows_keeps_what_came_before_a_maximum(size, levels):
    """Tokens of 2^-12 to 2^-20 of a row's largest, in the quarters of a step before it: every probability by itself, as each token's values stand in an element of their own."""
    s = Served([128] * 2, [128] * 2, 8, size, 64, 'f16', heads=128)
    c = torch.tensor([4 * x for x in levels], device='cuda').repeat_interleave(32)       # quarters of log2, a token's score
    c = c - 4 * torch.rand(128, device='cuda', generator=s.g).mul(2).floor().where(c < 0, torch.zeros_like(c))     # and some of one less
    c[c == 0] = -120
    c[32 * levels.index(0) + 11] = 0
    s.q.copy_(s.q[:1, :1].sign())
    s.k_scales.fill_(0.01)
    s.v_scales.fill_(100.0)
    s.v.zero_()
    at = torch.arange(128, device='cuda')
    out = []
    for part in range(128 // size):                  # (heads of 64 have room for half of the tokens at a time)
        s.v.zero_()
        for row in s.table:
            pages = torch.tensor(row[:2], device='cuda')[at // 64]
            s.k[pages, :, at % 64] = (c[:, None] * s.q[0, 0].float()).to(torch.int8)[:, None]
            mine = at // size == part
            s.v[pages[mine], :, at[mine] % 64, at[mine] % size] = 127
        out.append(s.attention(scale=0.25 * math.log(2) / (size * 0.01), causal=False)[:s.tokens].double() / 12700)
    runtime.token_check()
    p = torch.cat(out, 2)
    want = 2.0 ** (c.double() / 4)
    want = want / want.sum()
    # scores are exact but for the 32-bit scale (2^-22 of up to 30); 2^-18 of the polynomial, 11 bits down to 2^-19, then 2^-29 of the largest; the output's rounding
    bound = want * (30 * 2.0 ** -21 + 2.0 ** -17 + 2.0 ** -11 + half_step('f16') * 1.01) + 2.0 ** -29 + 2.0 ** -25 / 12700
    off = (p - want).abs()
    assert (off <= bound).all(), (float((off - bound).max()), int((off - bound).amax((0, 1)).argmax()))


@pytest.mark.parametrize('window', [0, 70])
@pytest.mark.parametrize('size, page, kv_heads, group, length, new, batch', [
    (64, 16, 1, 4, 1000, 1, 1), (128, 64, 2, 2, 700, 4, 3), (128, 32, 2, 16, 600, 1, 12), (64, 128, 8, 8, 500, 60, 3), (128, 16, 8, 16, 400, 300, 2), (64, 64, 2, 16, 900, 300, 12)])
def test_attention_every_probability_by_itself(size, page, kv_heads, group, length, new, batch, window):
    """Each token's values stand in an element of their own, so that an output is its probability: to within 2^-11 of itself or 2^-29 of the row's largest, as the
    header has it, wherever maxima move."""
    s = Served([length] * batch, [new] * batch, kv_heads, size, page, 'f16', heads=kv_heads * group)
    s.k_scales.mul_(2.0 ** torch.randint(-2, 3, s.k_scales.shape, device='cuda', generator=s.g))
    s.v_scales.fill_(2.0 ** 14 / 127).mul_(2.0 ** -torch.randint(0, 4, s.v_scales.shape, device='cuda', generator=s.g))
    scale, at, parts = size ** -0.5, torch.arange(length, device='cuda'), []
    for lo in range(0, length, size):
        s.v.zero_()
        t = at[lo:lo + size]
        for row in s.table:
            s.v[torch.tensor(row, device='cuda')[t // page], :, t % page, t % size] = 127
        parts.append(s.attention(scale=scale, window=window)[:s.tokens].double()[..., :len(t)] / 127)
    runtime.token_check()
    got = torch.cat(parts, 2)
    position = torch.arange(length - new, length, device='cuda')[:, None]
    seen = (at <= position) & ((at > position - window) if window else True)
    for b in {0, batch - 1}:
        used = torch.tensor(s.table[b][:-(-length // page)], device='cuda')
        for h in range(0, s.heads, max(1, group - 1)):
            sv = s.v_scales[used, h // group].double().repeat_interleave(page)[:length]
            k = (s.k[used, h // group].double() * s.k_scales[used, h // group].double()[:, None, None]).flatten(0, 1)[:length]
            q = s.q[b * new:(b + 1) * new, h].double()
            p = torch.softmax((q @ k.T * scale).masked_fill(~seen, -math.inf), 1) * sv
            # scores as in check_attention, queries to within 2^-21 of the row's largest; the output's own rounding beside the two bounds
            delta = (q.abs() @ k.abs().T * scale).amax(1, keepdim=True) * (size + 8) * 2 * U + scale * q.abs().amax(1, keepdim=True) * k.abs().sum(1).max() * 2.0 ** -21
            bound = p * (2 * delta + 2.0 ** -11 + half_step('f16') * 1.01 + (length / 16 + 100) * 4 * U) + 2.0 ** -29 * p.amax(1, keepdim=True) + 2.0 ** -25 / 127
            off = (got[b * new:(b + 1) * new, h] - p).abs()
            assert (off <= bound).all(), (b, h, float((off / bound).max()))
