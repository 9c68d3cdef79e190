"""8-bit layers on the device (kaldi_amd.int8) against their formulas in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of a 32-bit result; HALF[type] is half a step of the output's type."""
import os
import re

import numpy as np
import pytest
import torch

from kaldi_amd import decoder, int8
from kaldi_amd._lib import KamdError
from kaldi_amd.nnet import Layer

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -9 * 1.0001 * 2, torch.float16: 2.0 ** -12 * 1.0001 * 2}      # bf16 2^-8, fp16 2^-11; fp32: in the u's
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}                        # a step among the denormals
EPS = 1e-6


def rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def norm64(x, gain, eps, residual=None):
    h = x.double() if residual is None else x.double() + residual.double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
    return h, y if gain is None else y * gain.double()


def check_norm(y, want, dtype):
    # h, 1/rms, h * r and * gain: one rounding each, and h's own in r: 5 u (6 with what is of second order), then the output's
    off = (y.double().cpu() - want).abs()
    assert bool((off <= want.abs() * (6 * U + HALF[dtype]) + TINY[dtype]).all()), float((off / (want.abs() + 1e-30)).max())


def check_codes(q, scale, want, err=0.0):
    """codes and scales of the 64-bit rows `want`: a code is the nearest one, up to the roundings of its product (5 of them, 127
    codes wide) and a scale has three or four"""
    q, scale = q.cpu(), scale.double().cpu()
    top = want.abs().amax(1)
    assert bool(((scale - top / 127).abs() <= top / 127 * 6 * U + 2.0 ** -149).all())
    assert int(q.abs().max() if q.numel() else 0) <= 127
    off = (q.double() * scale[:, None] - want).abs()
    assert bool((off <= (top / 127)[:, None] * (0.5 + 127 * 10 * U) + 127 * 2.0 ** -149).all())


DIMS = [1, 3, 7, 8, 33, 100, 511, 512, 513, 1023, 1025, 1536, 2047, 2049, 4096, 4097, 8191, 8195, 16384, 16390, 32768, 32771, 70001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_norm_and_codes_over_dims(dtype, dim):
    rows = 5 if dim > 4096 else 9
    x, r, gain = rand(rows, dim, seed=dim, dtype=dtype), rand(rows, dim, seed=dim + 1, dtype=dtype, scale=2.0), 1 + 0.2 * rand(dim, seed=dim + 2)
    xd, rd, gd = x.cuda(), r.cuda(), gain.cuda()
    h, want = norm64(x, gain, EPS, r)
    y, s = int8.rms_norm(xd, gd, EPS, residual=rd)
    check_norm(y, want, dtype)
    assert torch.equal(s.cpu(), (x.float() + r.float()).to(dtype))
    check_norm(int8.rms_norm(xd, None, EPS), norm64(x, None, EPS)[1], dtype)
    q, scale, s2 = int8.rms_norm_int8(xd, gd, EPS, residual=rd)
    check_codes(q, scale, want)
    assert torch.equal(s2, s)
    check_codes(*int8.rms_norm_int8(xd, gd, EPS), norm64(x, gain, EPS)[1])
    check_codes(*int8.quantize_rows(xd), x.double())


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 64, 65, 257, 1000])
@pytest.mark.parametrize("dim", [40, 1536, 5000])
def test_norm_over_row_counts_and_strides(rows, dim):
    """rows apart, beginning anywhere, and nothing written beside them"""
    for dtype in TYPES:
        for lead, pad in ((0, 0), (1, 3), (5, 8)):
            def window(seed, t=dtype, fill=None):
                b = rand(rows + 2, lead + dim + pad, seed=seed).to(t) if fill is None else torch.full((rows + 2, lead + dim + pad), fill, dtype=t)
                b = b.cuda()
                return b, b[1:1 + rows, lead:lead + dim]
            (_, x), (_, r) = window(1), window(2)
            (yb, y), (sb, s) = window(0, fill=3.0), window(0, fill=5.0)
            (qb, q) = window(0, torch.int8, fill=77)
            scale = torch.full((rows + 2,), 9.0, device="cuda")
            _, want = norm64(x.cpu(), None, EPS, r.cpu())
            got = int8.rms_norm(x, None, EPS, residual=r, sum_out=s, out=y)
            assert got[0].data_ptr() == y.data_ptr() and got[1].data_ptr() == s.data_ptr()
            check_norm(y, want, dtype)
            int8.rms_norm_int8(x, None, EPS, residual=r, out=(q, scale[1:-1]))
            check_codes(q, scale[1:-1], want)
            for buf, view, v in ((yb, y, 3.0), (sb, s, 5.0), (qb, q, 77)):
                kept = torch.ones_like(buf, dtype=torch.bool)
                kept[1:1 + rows, lead:lead + dim] = False
                assert bool((buf[kept] == v).all())
            assert float(scale[0]) == 9.0 and float(scale[-1]) == 9.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, offsets", [(250, (0,)), (700, (0,)), (1100, (0,)), (1536, (0,)), (1733, (0,)), (2050, (0,)), (2304, (0,)), (5000, (0,)), (130, (-1, 0, 1)),
                                          (768, (-3, 0, 3)), (509, (-2, -1, 0, 1, 2)), (1000, (0, 4)), (257, tuple(range(8))), (9, tuple(range(8)))])
def test_many_rows_take_waves_of_their_own(dtype, dim, offsets):
    """every way in which 1024 rows and more are laid over the threads"""
    x, r, gain = rand(1100, dim, seed=dim, dtype=dtype), rand(1100, dim, seed=dim + 1, dtype=dtype), 1 + 0.2 * rand(dim, seed=2)
    lo, n = min(offsets), 1100 - (max(offsets) - min(offsets))
    check_codes(*int8.quantize_rows(x.cuda(), offsets), torch.cat([x[o - lo:o - lo + n] for o in offsets], 1).double())
    h, want = norm64(x, gain, EPS, r)
    rd = r.cuda()
    y, s = int8.rms_norm(x.cuda(), gain.cuda(), EPS, residual=rd, sum_out=rd)
    check_norm(y, want, dtype)
    assert s is rd and torch.equal(s.cpu(), (x.float() + r.float()).to(dtype))
    rd = r.cuda()
    q, scale, s = int8.rms_norm_int8(x.cuda(), gain.cuda(), EPS, residual=rd, sum_out=rd)
    check_codes(q, scale, want)
    assert torch.equal(s.cpu(), (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [100, 1501, 2999, 9003, 20005, 40001])
def test_norm_in_place(dtype, dim):
    x, r = rand(7, dim, seed=3, dtype=dtype).cuda(), rand(7, dim, seed=4, dtype=dtype).cuda()
    y, s = int8.rms_norm(x, None, EPS, residual=r)
    a, b = x.clone(), r.clone()
    int8.rms_norm(a, None, EPS, residual=b, sum_out=b, out=a)           # the residual stream is updated, the input becomes the output
    assert torch.equal(a, y) and torch.equal(b, s)
    a, b = x.clone(), r.clone()
    int8.rms_norm(a, None, EPS, residual=b, sum_out=a, out=b)
    assert torch.equal(b, y) and torch.equal(a, s)
    a = x.clone()
    int8.rms_norm(a, None, EPS, out=a)
    assert torch.equal(a, int8.rms_norm(x, None, EPS))
    q, scale, s2 = int8.rms_norm_int8(x, None, EPS, residual=r)
    b = r.clone()
    q2, scale2, _ = int8.rms_norm_int8(x, None, EPS, residual=b, sum_out=b)
    assert torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(b, s2)


@pytest.mark.parametrize("dim", [33, 1536, 5000, 40000])
def test_rows_out_of_the_ordinary(dim):
    """zeros, the smallest and largest numbers, infinities and NaN: by the formula, row by row, and only in their row"""
    big, small = 3e38, 1e-42
    x = rand(10, dim, seed=8)
    x[1] = 0
    x[2] *= 1e-40
    x[3] = big
    x[4] *= 1e30
    x[5] = 0
    x[5, dim // 2] = small
    x[6, 0] = float("inf")
    x[7, dim - 1] = float("nan")
    x[8, dim // 3] = -float("inf")
    xd = x.cuda()
    y = int8.rms_norm(xd, None, EPS).cpu()
    q, scale = int8.rms_norm_int8(xd, None, EPS)
    pq, pscale = int8.quantize_rows(xd)
    fine = [0, 1, 2, 3, 4, 5, 9]
    want = norm64(x[fine], None, EPS)[1]
    check_norm(y[fine], want, torch.float32)
    check_codes(q[fine], scale[fine], want)
    check_codes(pq[fine], pscale[fine], x[fine].double())
    assert float(scale[1]) == 0.0 and int(q[1].abs().max()) == 0 and float(pscale[1]) == 0.0
    for row in (6, 7, 8):
        assert bool(torch.isnan(scale[row])) and int(q[row].abs().max()) == 0
        assert bool(torch.isnan(pscale[row])) and int(pq[row].abs().max()) == 0
    assert bool(torch.isnan(y[7]).all())
    for row, at in ((6, 0), (8, dim // 3)):                              # inf / inf at its place, 0 elsewhere
        assert bool(torch.isnan(y[row, at])) and int(torch.isnan(y[row]).sum()) == 1
        assert float(y[row].nan_to_num(0.0).abs().max()) == 0.0
    b = (rand(4, dim, seed=9) * 1e20).bfloat16()                         # no sum of squares in 32 bits
    check_norm(int8.rms_norm(b.cuda(), None, EPS), norm64(b, None, EPS)[1], torch.bfloat16)
    x = rand(4, dim, seed=10) * 1e-15                                    # squares far below eps, and an eps that small
    check_norm(int8.rms_norm(x.cuda(), None, 2.0 ** -66), norm64(x, None, 2.0 ** -66)[1], torch.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, offsets", [(40, (0,)), (40, (-1, 0, 1)), (43, (-3, 0, 3)), (768, (-3, 0, 3)), (768, (0, 3)), (5, (2,)), (7, (-1, 0, 1, 2, 5, -2, 3, 4)),
                                          (1500, (3, -3)), (33, (1, 1, 0)), (9001, (-1, 0, 1, 2)), (64, (5, 9))])
def test_quantize_splices(dtype, dim, offsets):
    x = rand(23, dim, seed=dim, dtype=dtype)
    q, scale = int8.quantize_rows(x.cuda(), offsets)
    lo, n = min(offsets), 23 - (max(offsets) - min(offsets))
    want = torch.cat([x[o - lo:o - lo + n] for o in offsets], 1).double()
    assert tuple(q.shape) == (n, dim * len(offsets))
    check_codes(q, scale, want)
    assert int8.quantize_rows(x[:max(offsets) - lo].cuda(), offsets)[0].shape[0] == 0


def test_codes_are_the_nearest_ones_on_a_grid():
    """rows that are codes times a power of two come back as these codes; half-way values go to the even one"""
    codes = torch.randint(-127, 128, (64, 300), generator=torch.Generator().manual_seed(1))
    codes[:, 17] = 127
    for e in (-140, -120, -3, 0, 90):
        x = (codes.double() * 2.0 ** e).float()
        q, scale = int8.quantize_rows(x.cuda())
        assert torch.equal(q.cpu().long(), codes) and bool((scale.cpu().double() == 2.0 ** e).all())
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5]])
    assert int8.quantize_rows(x.cuda())[0].cpu().tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, -126]]


# ---- the product -------------------------------------------------------------------------------------------------------

def codes(rows, cols, seed, spread=40.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, cols, generator=g) * spread).round().clamp(-127, 127).to(torch.int8)


def on_device(q, extra=0, fill=113):
    """codes as rows of a wider buffer, begun on multiples of 16 bytes; what lies behind a row is not zero"""
    b = torch.full((q.shape[0], (q.shape[1] + 15) // 16 * 16 + extra), fill, dtype=torch.int8)
    b[:, :q.shape[1]] = q
    return b.cuda()[:, :q.shape[1]]


def product64(q, scale, w, ws, bias, relu, mul, add):
    """(the result, the bound of its 32-bit roundings)"""
    p = (q.double() @ w.double().T) * scale.double()[:, None] * ws.double()
    z = p if bias is None else p + bias.double()
    bound = 3 * U * p.abs() + U * z.abs()                                # the integer, two products, the sum
    if relu:
        z = z.clamp_min(0)
    if mul is not None or add is not None:
        m = z if mul is None else z * mul.double()
        bound = bound * (1 if mul is None else mul.double().abs()) + U * m.abs()
        z = m if add is None else m + add.double()
        bound = bound + U * z.abs()
    return z, bound * 1.01


def check_product(y, want, bound, dtype):
    off = (y.double().cpu() - want).abs()
    assert bool((off <= bound + want.abs() * HALF[dtype] + TINY[dtype]).all()), float((off - bound).max())


def layer_of(k, n, seed, full):
    g = torch.Generator().manual_seed(seed)
    v = lambda s, o: (o + s * torch.randn(n, generator=g)) if full else None  # noqa: E731
    return codes(n, k, seed), 0.01 * (0.5 + torch.rand(n, generator=g)), v(1.0, 0.0), v(0.5, 1.0), v(1.0, 0.0)


def both(rows, k, n, dtype, full=True, extra=0, seed=1):
    w, ws, bias, mul, add = layer_of(k, n, seed, full)
    q, scale = codes(rows, k, seed + 1), 0.01 * (0.5 + torch.rand(rows, generator=torch.Generator().manual_seed(seed + 2)))
    d = lambda t: None if t is None else t.cuda()  # noqa: E731
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), d(bias), full, d(mul), d(add))
    y = layer.propagate(on_device(q, extra), scale.cuda(), dtype)
    check_product(y, *product64(q, scale, w, ws, bias, full, mul, add), dtype)
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 200, 257, 513, 700])
def test_product_over_rows(dtype, rows):
    both(rows, 200, 90, dtype, seed=rows)


@pytest.mark.parametrize("k", [1, 5, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 384, 700, 1536, 4100])
def test_product_over_inputs(k):
    for rows in (1, 40, 150, 300):
        both(rows, k, 70, torch.float32, seed=k, extra=(k % 3) * 16)


@pytest.mark.parametrize("n", [1, 3, 15, 16, 17, 100, 127, 128, 129, 255, 257, 515])
def test_product_over_outputs(n):
    for rows in (1, 50, 140, 600):
        for dtype in TYPES:
            both(rows, 96, n, dtype, full=n % 2 == 0, seed=n)


@pytest.mark.parametrize("rows, k, n", [(2100, 1000, 1100), (4097, 257, 2050), (1030, 3000, 520), (9000, 130, 300)])
def test_product_of_many_tiles(rows, k, n):
    both(rows, k, n, torch.bfloat16)
    both(rows, k, n, torch.float32, full=False)


@pytest.mark.parametrize("rows, k, n", [(17, 130, 300), (100, 1000, 100), (500, 4000, 1000), (1000, 1500, 2000), (2000, 1537, 2328), (7000, 500, 1500),
                                        (3900, 1030, 4000), (8100, 700, 8000)])
def test_product_in_each_of_its_kernels(rows, k, n):
    """sizes at which the cost rule takes the split kernel, the 64 x 64, 64 x 128, 128 x 192 (one and two to a CU) and 256 x 256
    tiles, with rows, channels and codes that end inside a tile; the exact sums come from 64-bit products on the device"""
    w, ws, bias, mul, add = layer_of(k, n, 51, True)
    q, scale = codes(rows, k, 52), torch.rand(rows)
    d = [t.cuda() for t in (q, scale, w, ws, bias, mul, add)]
    layer = int8.AffineInt8(d[2], d[3], d[4], True, d[5], d[6])
    for dtype in TYPES:
        y = layer.propagate(on_device(q, 16), d[1], dtype)
        want, bound = product64(d[0], d[1], d[2], d[3], d[4], True, d[5], d[6])
        check_product(y, want.cpu(), bound.cpu(), dtype)


def test_an_output_larger_than_the_caches():
    """over 128 MB: stored past the caches, with rows, channels and the leading dimension off every boundary"""
    for rows, n, dtype in ((9001, 7777, torch.bfloat16), (300, 120001, torch.float32)):
        w, ws, bias, _, _ = layer_of(40, n, 53, True)
        q, scale = codes(rows, 40, 54), torch.rand(rows)
        out = torch.full((rows + 1, n + 3), 7.0, dtype=dtype, device="cuda")
        y = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda()).propagate(on_device(q), scale.cuda(), dtype, out=out[:rows, 1:n + 1])
        at = torch.cat([torch.arange(0, rows, 97), torch.tensor([rows - 1])])
        check_product(y[at], *product64(q[at], scale[at], w, ws, bias, False, None, None), dtype)
        assert bool((out[rows] == 7.0).all()) and bool((out[:, 0] == 7.0).all()) and bool((out[:, n + 1:] == 7.0).all())


def test_product_at_the_limits_of_its_sum():
    """the longest row of the largest codes: a sum of 2^31 - 16384 and one of its negative"""
    k = 131071
    q = torch.full((2, k), -128, dtype=torch.int8)
    q[1] = 127
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    for rows in (2, 80):
        y = int8.AffineInt8(w.cuda(), torch.ones(3).cuda()).propagate(on_device(q.repeat(rows // 2, 1)), torch.ones(rows).cuda())
        want = (q.double() @ w.double().T).float().repeat(rows // 2, 1)
        assert torch.equal(y.cpu(), want)
    assert float(want[0, 0]) == float(np.float32(128 * 128 * k))


def test_product_writes_its_matrix_only():
    for rows, n in ((3, 37), (150, 200), (1000, 300)):
        w, ws, bias, mul, add = layer_of(64, n, 5, True)
        layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda())
        q, scale = codes(rows, 64, 6), torch.rand(rows)
        for dtype in TYPES:
            for lead, pad in ((0, 0), (1, 2), (3, 8)):
                b = torch.full((rows + 2, lead + n + pad), 7.0, dtype=dtype, device="cuda")
                view = b[1:1 + rows, lead:lead + n]
                layer.propagate(on_device(q, 32), scale.cuda(), dtype, out=view)
                check_product(view, *product64(q, scale, w, ws, bias, False, None, None), dtype)
                kept = torch.ones_like(b, dtype=torch.bool)
                kept[1:1 + rows, lead:lead + n] = False
                assert bool((b[kept] == 7.0).all())


def test_a_rows_result_does_not_depend_on_the_others():
    w, ws, bias, mul, add = layer_of(300, 210, 7, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda(), True, mul.cuda(), add.cuda())
    q, scale = on_device(codes(2000, 300, 8)), torch.rand(2000, device="cuda")
    whole = layer.propagate(q, scale, torch.bfloat16)
    for a, b in ((0, 1), (5, 20), (64, 128), (100, 400), (1999, 2000)):
        assert torch.equal(layer.propagate(q[a:b], scale[a:b], torch.bfloat16), whole[a:b])


def test_scales_that_are_not_numbers_stay_in_their_row_and_channel():
    w, ws, bias, _, _ = layer_of(64, 40, 9, True)
    for rows in (20, 300):
        q, scale = codes(rows, 64, 10), torch.rand(rows)
        scale[3] = float("nan")
        scale[7] = 0.0
        y = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda(), relu=True).propagate(on_device(q), scale.cuda()).cpu()
        assert bool(torch.isnan(y[3]).all()) and int(torch.isnan(y).any(1).sum()) == 1
        assert torch.equal(y[7], bias.clamp_min(0))


def test_offsets_past_32_bits():
    """rows 2^23 codes apart, 300 of them; rows of a matrix of over 2^32 values"""
    ld, rows = 1 << 23, 300
    w, ws, bias, _, _ = layer_of(80, 50, 11, True)
    q, scale = codes(rows, 80, 12), torch.rand(rows)
    far = torch.empty(rows * ld, dtype=torch.int8, device="cuda").view(rows, ld)[:, :80]
    far.copy_(q.cuda())
    y = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda()).propagate(far, scale.cuda())
    check_product(y, *product64(q, scale, w, ws, bias, False, None, None), torch.float32)
    del far
    rows, ld = 1100, 1 << 22
    x = rand(rows, 100, dtype=torch.float16)
    far = torch.empty(rows * ld, dtype=torch.float16, device="cuda").view(rows, ld)[:, 7:107]
    far.copy_(x.cuda())
    check_norm(int8.rms_norm(far, None, EPS), norm64(x, None, EPS)[1], torch.float16)
    check_codes(*int8.quantize_rows(far, (0, 1)), torch.cat([x[:-1], x[1:]], 1).double())


# ---- as they are used ------------------------------------------------------------------------------------------------------

def test_layers_in_a_row_against_64_bits():
    """two pre-norm layers with a residual stream, every step checked from the codes that the step before handed over"""
    rows, d, f = 333, 200, 520
    w1, s1, b1, _, _ = layer_of(d, f, 21, True)
    w2, s2, b2, _, _ = layer_of(f, d, 22, True)
    up, down = int8.AffineInt8(w1.cuda(), s1.cuda(), b1.cuda(), relu=True), int8.AffineInt8(w2.cuda(), s2.cuda(), b2.cuda())
    x, h = rand(rows, d, seed=23, dtype=torch.bfloat16), rand(rows, d, seed=24, dtype=torch.bfloat16)
    xd, hd, gain = x.cuda(), h.cuda(), 1 + 0.1 * rand(d, seed=25)
    for _ in range(2):
        want = norm64(xd.cpu(), gain, EPS, hd.cpu())[1]
        q, scale, hd = int8.rms_norm_int8(xd, gain.cuda(), EPS, residual=hd)
        check_codes(q, scale, want)
        y = up.propagate(q, scale, torch.bfloat16)
        check_product(y, *product64(q.cpu(), scale.cpu(), w1, s1, b1, True, None, None), torch.bfloat16)
        q2, scale2 = int8.quantize_rows(y)
        check_codes(q2, scale2, y.double().cpu())
        xd = down.propagate(q2, scale2, torch.bfloat16)
        check_product(xd, *product64(q2.cpu(), scale2.cpu(), w2, s2, b2, False, None, None), torch.bfloat16)


@pytest.mark.parametrize("offsets", [[0], [-1, 0, 2], [-3, 0]])
def test_a_layer_in_8_bits_against_the_component(offsets):
    """AffineInt8.from_layer beside decoder.Component on the same `kaldi_amd.nnet.Layer`: the difference is that of the codes,
    at most half a scale on each side of every product"""
    rng = np.random.default_rng(3)
    k, n, T = 96, 150, 200
    W = (rng.standard_normal((n, k * len(offsets))) / np.sqrt(k * len(offsets))).astype(np.float32)
    v = lambda lo, hi: rng.uniform(lo, hi, n).astype(np.float32)  # noqa: E731
    layer = Layer("c", k, n, offsets, -1, W, v(-.1, .1), True, v(.5, 1.5), v(-.1, .1), post_offset=v(0, 2), post_scale=0.7)
    x = rng.standard_normal((T, k)).astype(np.float32)
    plain = decoder.Component(layer).Propagate(x).astype(np.float64)
    c = int8.AffineInt8.from_layer(layer)
    assert (c.in_dim, c.out_dim) == (k * len(offsets), n)
    y = c.Propagate(torch.from_numpy(x).cuda())
    assert y.dtype == torch.float32 and tuple(y.shape) == plain.shape
    q, scale = c.quantize_input(torch.from_numpy(x).cuda())
    xs = (q.double() * scale.double()[:, None]).cpu().numpy()
    ws = np.abs(W).max(1) / 127.0
    half_x = scale.double().cpu().numpy()[:, None] / 2 * 1.001
    # |x w - x' w'| <= |w| |x - x'| + |x'| |w - w'|, summed over k
    bound = half_x * np.abs(W).sum(1)[None] + np.abs(xs).sum(1)[:, None] * (ws / 2 * 1.001)[None]
    bound = bound * np.abs(layer.bn_scale * layer.post_scale)[None] + 2e-5 * max(1.0, np.abs(plain).max())
    off = np.abs(y.cpu().numpy() - plain)
    assert (off <= bound).all()
    assert np.sqrt((off ** 2).mean()) < 0.03 * np.sqrt((plain ** 2).mean())


def test_captured_and_replayed_beside_eager_calls():
    """a layer in a graph: replays on new inputs, with eager calls of other sizes between them, equal the eager results"""
    w, ws, bias, _, _ = layer_of(512, 320, 31, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda(), relu=True)
    for rows in (1, 48, 500):
        x, h = torch.zeros(rows, 512, device="cuda", dtype=torch.bfloat16), torch.zeros(rows, 512, device="cuda", dtype=torch.bfloat16)

        def step():
            q, scale, s = int8.rms_norm_int8(x, None, EPS, residual=h)
            return layer.propagate(q, scale, torch.bfloat16), s, int8.rms_norm(x, None, EPS)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for seed in range(3):
            x.copy_(rand(rows, 512, seed=seed, dtype=torch.bfloat16))
            h.copy_(rand(rows, 512, seed=seed + 50, dtype=torch.bfloat16))
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            for t, e in zip(got, step()):
                assert torch.equal(t, e)
            int8.rms_norm(rand(5, 40, seed=seed).cuda())


def test_captured_without_having_run():
    """kernels whose first launch is in a capture"""
    w, ws, bias, _, _ = layer_of(272, 1000, 61, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda())
    x = torch.zeros(610, 272, device="cuda", dtype=torch.float16)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, scale = int8.quantize_rows(x)
        y = layer.propagate(q, scale, torch.float16)
        n = int8.rms_norm(y)
    for seed in range(3):
        x.copy_(rand(610, 272, seed=seed, dtype=torch.float16))
        g.replay()
        torch.cuda.synchronize()
        q2, scale2 = int8.quantize_rows(x)
        y2 = layer.propagate(q2, scale2, torch.float16)
        assert torch.equal(q, q2) and torch.equal(scale, scale2) and torch.equal(y, y2) and torch.equal(n, int8.rms_norm(y2))


def test_more_rows_than_a_launch_takes():
    rows = (1 << 22) + 77
    w, ws, bias, _, _ = layer_of(16, 8, 62, True)
    q = torch.randint(-127, 128, (rows, 16), dtype=torch.int8, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    scale = torch.rand(rows, device="cuda")
    y = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda()).propagate(q, scale)
    want, bound = product64(q, scale, w.cuda(), ws.cuda(), bias.cuda(), False, None, None)
    check_product(y, want.cpu(), bound.cpu(), torch.float32)
    rows = (1 << 24) + 5                                                 # 4 rows to a workgroup of the row kernels
    x = torch.randn(rows, 8, device="cuda")
    y = int8.rms_norm(x, None, EPS)
    h = x.double()
    want = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    assert bool(((y.double() - want).abs() <= want.abs() * 6 * U).all())
    q, scale = int8.quantize_rows(x)
    top = h.abs().amax(1)
    assert bool(((scale.double() - top / 127).abs() <= top / 127 * 6 * U).all())
    assert bool(((q.double() * scale.double()[:, None] - h).abs() <= (top / 127)[:, None] * (0.5 + 127 * 10 * U)).all())


def test_two_streams_use_one_layer_at_once():
    w, ws, bias, _, _ = layer_of(768, 640, 41, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda())
    inputs = [(on_device(codes(r, 768, r)), torch.rand(r, generator=torch.Generator().manual_seed(r)).cuda()) for r in (40, 300, 900, 17)]
    want = [layer.propagate(q, s) for q, s in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = []
    for _ in range(5):
        for st, (q, s) in zip(streams, inputs):
            with torch.cuda.stream(st):
                got.append(layer.propagate(q, s))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % len(want)])


def test_empty_matrices():
    e = torch.empty(0, 64, device="cuda")
    assert int8.rms_norm(e).shape == (0, 64) and int8.quantize_rows(e)[0].shape == (0, 64)
    q, scale = int8.rms_norm_int8(e)
    w, ws, _, _, _ = layer_of(64, 20, 1, False)
    assert int8.AffineInt8(w.cuda(), ws.cuda()).propagate(q, scale).shape == (0, 20)


def test_refusals_on_the_device():
    x = torch.zeros(6, 40, device="cuda")
    w, ws, _, _, _ = layer_of(40, 20, 1, False)
    layer = int8.AffineInt8(w.cuda(), ws.cuda())
    q, scale = int8.quantize_rows(x)
    bad = [
        (lambda: int8.rms_norm(x.double()), "float32, bfloat16 or float16"), (lambda: int8.rms_norm(x[0]), "matrix"), (lambda: int8.rms_norm(x.t()), "contiguous"),
        (lambda: int8.rms_norm(x, gain=torch.ones(39, device="cuda")), "vector of 40"), (lambda: int8.rms_norm(x, gain=torch.ones(40)), "vector of 40"),
        (lambda: int8.rms_norm(x, residual=x[:5]), "shape"), (lambda: int8.rms_norm(x, residual=x.half()), "float32 expected"),
        (lambda: int8.rms_norm(x, eps=0.0), "eps"), (lambda: int8.rms_norm(x[:1].expand(6, 40)), "leading"),
        (lambda: int8.rms_norm(x, out=torch.empty(6, 41, device="cuda")), "shape"), (lambda: int8.rms_norm(x.cpu()), "on the GPU"),
        (lambda: int8.rms_norm(x.clone().requires_grad_()), "gradient"), (lambda: layer.propagate(q, scale, torch.int8), "float32, bfloat16 or float16"),
        (lambda: int8.quantize_rows(x, ()), "offsets"), (lambda: int8.quantize_rows(x, range(9)), "offsets"),
        (lambda: int8.quantize_rows(x, out=(q[:, :39], scale)), "shape"), (lambda: int8.quantize_rows(x, out=(q, scale[:5])), "vector of 6"),
        (lambda: layer.propagate(q[:, :32], scale), "codes"), (lambda: layer.propagate(q, scale[:5]), "vector of 6"), (lambda: layer.propagate(q, scale.half()), "vector"),
        (lambda: layer.propagate(torch.zeros(6, 40, dtype=torch.int8, device="cuda"), scale), "multiples of 16"),
        (lambda: layer.propagate(torch.zeros(6, 56, dtype=torch.int8, device="cuda")[:, 8:48], scale), "multiples of 16"),
        (lambda: layer.propagate(torch.zeros(5 * 48 + 40, dtype=torch.int8, device="cuda").as_strided((6, 40), (48, 1)), scale), "last row"),
        (lambda: layer.propagate(q, scale, torch.float64), "float32, bfloat16 or float16"), (lambda: layer.propagate(q, scale, out=torch.empty(6, 21, device="cuda")), "shape"),
        (lambda: layer.propagate(q, scale, torch.float16, out=torch.empty(6, 20, device="cuda")), "float16 expected"),
        (lambda: int8.AffineInt8(w.cuda().float(), ws.cuda()), "int8 expected"), (lambda: int8.rms_norm(x, gain=torch.ones(40, device="cuda", requires_grad=True)), "gradient"),
        (lambda: int8.rms_norm_int8(x, out=q), "pair"), (lambda: layer.propagate(q, scale, "float"), "torch.dtype"), (lambda: int8.quantize_rows(x, (0, 2 ** 40)), "out of range"), (lambda: int8.AffineInt8(w.cuda(), ws.cuda()[:19]), "vector of 20"),
        (lambda: int8.AffineInt8(torch.zeros(2, 131072, dtype=torch.int8, device="cuda"), ws.cuda()[:2]), "131071"),
    ]
    for call, says in bad:
        with pytest.raises(KamdError, match=says):
            call()
    with torch.no_grad():
        int8.rms_norm(x.clone().requires_grad_())
    torch.cuda.synchronize()


def test_given_outputs_count_as_written():
    """what autograd saved of a tensor that a call writes into is stale, and has to be known as such"""
    x = torch.randn(3, 64, device="cuda")
    w = torch.randn(64, 64, device="cuda", requires_grad=True)
    loss = (x @ w).sum()                      # saves x
    h, codes, y = x.clone(), (int8.empty_codes(3, 64, "cuda"), torch.empty(3, device="cuda")), torch.empty(3, 64, device="cuda")
    before = [t._version for t in (h, *codes, y)]
    int8.rms_norm(x, sum_out=h, out=y)
    int8.quantize_rows(x, out=codes)
    assert [t._version - b for t, b in zip((h, *codes, y), before)] == [1, 1, 1, 1]
    assert x._version == 0
    int8.rms_norm(x, residual=x, sum_out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        z = torch.randn(3, 64, device="cuda")
    int8.rms_norm(z, out=z)                   # has no count to keep


def test_one_row_of_a_matrix_whose_rows_lie_far_apart():
    big = torch.zeros(2, 1 << 24, dtype=torch.int8, device="cuda")
    row = big[1:, :48]
    row.copy_(torch.arange(-24, 24, dtype=torch.int8, device="cuda")[None])
    layer = int8.AffineInt8(torch.eye(48, dtype=torch.int8, device="cuda"), torch.ones(48, device="cuda"))
    y = layer.propagate(row, torch.full((1,), 0.5, device="cuda"))
    assert torch.equal(y, row.float() * 0.5)


@pytest.mark.parametrize("k", [1, 64, 128, 129, 384, 1000])
def test_sums_that_start_in_the_middle(k):
    """128 x 192 tiles side by side begin at different places of the sum: every column of tiles, sums from one stage upwards"""
    rows, n = 2030, 192 * 31 + 187            # two tiles per CU
    g = torch.Generator().manual_seed(k)
    q = int8.empty_codes(rows, k, "cuda")
    q.copy_(torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8))
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    layer = int8.AffineInt8(w.cuda(), torch.ones(n, device="cuda"))
    y = layer.propagate(q, torch.full((rows,), 2.0 ** -20, device="cuda"))
    # |sum| <= 1000 * 127^2 < 2^24: exact in 32-bit floats, and so is the power of two
    assert torch.equal(y.cpu().double(), (q.cpu().double() @ w.double().T) * 2.0 ** -20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, k, n", [(1, 4200, 8193), (16, 8000, 4500), (17, 4200, 8193), (3, 1000, 40000)])
def test_few_rows_of_large_weights(rows, k, n, dtype):
    """weights beyond the L2s, which up to 16 rows read past them"""
    g = torch.Generator().manual_seed(rows)
    q = int8.empty_codes(rows, k, "cuda")
    q.copy_(torch.randint(-15, 16, (rows, k), generator=g, dtype=torch.int8))
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    layer = int8.AffineInt8(w.cuda(), torch.ones(n, device="cuda"))
    scale = torch.full((rows,), 2.0 ** -20, device="cuda")
    # |sum| <= 8000 * 15 * 127 < 2^24: exact in 32-bit floats, so that the output's type rounds an exact value once
    want = ((q.cpu().float() @ w.float().T).double() * 2.0 ** -20).to(dtype)
    for _ in range(3):
        assert torch.equal(layer.propagate(q, scale, dtype).cpu(), want)


def test_outputs_over_other_arguments_are_refused():
    """views of one buffer: outputs beside the inputs are written there, over them they are refused"""
    w, ws, _, _, _ = layer_of(48, 24, 71, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda())
    b = rand(9, 100, seed=72).cuda()
    x, gain = b[:, :40], torch.ones(40, device="cuda")
    want = int8.rms_norm(x.clone(), gain, EPS)
    y = int8.rms_norm(x, gain, EPS, out=b[:, 40:80])                     # the columns beside x
    assert torch.equal(y, want) and torch.equal(b[:, 40:80], want)
    mem = torch.zeros(9 * 48, dtype=torch.int8, device="cuda")
    q, scale = int8.quantize_rows(rand(9, 48, seed=73).cuda(), out=(mem.view(9, 48), torch.empty(9, device="cuda")))
    bad = [
        lambda: int8.rms_norm(x, gain, EPS, out=b[:, 39:79]), lambda: int8.rms_norm(x[1:], gain, EPS, out=x[:-1]), lambda: int8.rms_norm(x, gain, EPS, out=b.as_strided((9, 40), (99, 1), 62)),
        lambda: int8.rms_norm(x, gain, EPS, residual=b[:, 1:41], sum_out=x), lambda: int8.rms_norm(x, b[0, 50:90], EPS, sum_out=b[:, 45:85]),
        lambda: int8.rms_norm_int8(x, gain, EPS, out=(b.view(torch.int8)[:, 100:140], torch.empty(9, device="cuda"))),
        lambda: int8.quantize_rows(x, out=(b.view(torch.int8)[:, 159:199], torch.empty(9, device="cuda"))),
        lambda: int8.quantize_rows(x, out=(torch.empty(9, 40, dtype=torch.int8, device="cuda"), b[0, 20:29])),
        lambda: layer.propagate(q[:1], scale[:1], out=mem.view(torch.float32)[:24].view(1, 24)),
        lambda: layer.propagate(q[:1], scale[:1], torch.float16, out=mem[46:94].view(torch.float16).view(1, 24)),
        lambda: layer.propagate(q[:1], b[0, 20:21], out=b[0, :24].view(1, 24)),
    ]
    before = b.clone(), mem.clone()
    for call in bad:
        with pytest.raises(KamdError, match="overlaps"):
            call()
    assert torch.equal(b, before[0]) and torch.equal(mem, before[1])
    # a spliced matrix and its codes in one buffer, the codes in the columns beside it
    s = torch.zeros(9, 256, dtype=torch.float32, device="cuda")
    s[:, :40] = x
    q2, scale2 = int8.quantize_rows(s[:, :40], (-1, 0, 1), out=(s.view(torch.int8)[1:8, 160:280], torch.empty(7, device="cuda")))
    q3, scale3 = int8.quantize_rows(x, (-1, 0, 1))
    assert torch.equal(q2, q3) and torch.equal(scale2, scale3)


# ---- each kernel of the product at the limits of what it addresses ---------------------------------------------------------

def kernel_of(rows, k, n):
    """The kernel that the cost rule of csrc/affine_i8.hip takes, (rows, channels, one to a CU) of its tile: the rule evaluated
    with the constants that the source holds, so that a size that a new constant moves to another kernel is noticed."""
    source = open(os.path.join(os.path.dirname(int8.__file__), "csrc", "affine_i8.hip")).read()
    table = re.search(r"static const Kernel kernels\[\] = \{(.*?)\};", source, re.S).group(1)
    kernels = re.findall(r"\{(\d+), (\d+), ([\d.]+), ([\d.]+), (true|false), Launch", table)
    assert len(kernels) == 7
    ceil = lambda a, b: -(-a // b)  # noqa: E731
    best = None
    for bm, bn, step, fixed, alone in kernels:
        per_cu = ceil(ceil(rows, int(bm)) * ceil(n, int(bn)), 256)
        cost = per_cu * (ceil(k, 128) * float(step) + float(fixed))
        if not (alone == "true" and per_cu > 1) and (best is None or cost < best[0]):
            best = cost, (int(bm), int(bn), alone == "true")
    return best[1]


def check_on_device(q, scale, w, ws, dtype, layer=None):
    y = (layer or int8.AffineInt8(w, ws)).propagate(q, scale, dtype)
    p = (q.double() @ w.double().T) * scale.double()[:, None] * ws.double()
    off = (y.double() - p).abs() - p.abs() * (4 * U + HALF[dtype])               # the integer, two products, (and a bias of 0)
    assert float(off.max()) <= TINY[dtype]


def random_codes(rows, cols, seed, out=None):
    g = torch.Generator("cuda").manual_seed(seed)
    q = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8, device="cuda")
    return q if out is None else out.copy_(q)


@pytest.mark.parametrize("rows, n, kernel", [(40, 50, (16, 16, False)), (300, 301, (32, 32, False)), (700, 701, (64, 64, False)), (1000, 1501, (64, 128, False)),
                                             (2000, 2301, (128, 192, True)), (3000, 3501, (128, 192, False)), (4000, 4001, (256, 256, False))])
def test_the_longest_sums_in_each_kernel(rows, n, kernel):
    """131071 codes, the largest of them in some rows and channels: sums up to 2^31 - 16384, weights to the end of a descriptor"""
    k = 131071
    assert kernel_of(rows, k, n) == kernel
    q, w = random_codes(rows, k, 81, int8.empty_codes(rows, k, "cuda")), random_codes(n, k, 82)
    for t in (q, w):
        t[0], t[1], t[-1], t[-2] = -128, 127, -128, 127
    check_on_device(q, torch.rand(rows, device="cuda"), w, torch.rand(n, device="cuda"), torch.float32)


@pytest.mark.parametrize("rows, k, n, kernel", [(200, 90, 300, (16, 16, False)), (300, 1000, 400, (32, 32, False)), (300, 1000, 1000, (64, 64, False)), (300, 500, 5000, (64, 128, False)),
                                                (300, 1500, 16000, (128, 192, True)), (300, 100, 40001, (128, 192, False)), (512, 2000, 32767, (256, 256, False))])
def test_rows_at_the_largest_distance_in_each_kernel(rows, k, n, kernel):
    """rows of codes 2^23 bytes apart: a tile's rows end just below 2^31 from its first, the call's beyond 2^32"""
    assert kernel_of(rows, k, n) == kernel
    far = torch.empty(rows * (1 << 23), dtype=torch.int8, device="cuda").view(rows, 1 << 23)[:, :k]
    random_codes(rows, k, 83, far)
    check_on_device(far, torch.rand(rows, device="cuda"), random_codes(n, k, 84), torch.rand(n, device="cuda"), torch.bfloat16)
    layer = int8.AffineInt8(random_codes(16, k, 85), torch.rand(16, device="cuda"))
    with pytest.raises(KamdError, match="at most 8388608 apart"):
        layer.propagate(torch.empty(2, (1 << 23) + 16, dtype=torch.int8, device="cuda")[:, :k], torch.rand(2, device="cuda"))


@pytest.mark.parametrize("rows, k, n, kernel", [(9800, 700, 8190, (256, 256, False)), (8300, 700, 8200, (128, 192, False)), (600, 100, 120001, (128, 192, False))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_16_bit_outputs_larger_than_the_caches(rows, k, n, kernel, dtype):
    assert kernel_of(rows, k, n) == kernel and rows * n * 2 > 128 << 20
    q, w = random_codes(rows, k, 86, int8.empty_codes(rows, k, "cuda")), random_codes(n, k, 87)
    check_on_device(q, torch.rand(rows, device="cuda"), w, torch.rand(n, device="cuda") * 2.0 ** -12, dtype)


@pytest.mark.parametrize("target", [1.0, 0.5, 3.0])
def test_normalize_component_and_its_floor(target):
    """NormalizeComponent's formula, x / sqrt(max(mean(x^2) / t^2, 2^-66)), in 64 bits (parity unpinned: there are no outputs of the
    reference for it): equal far from the floor, at most sqrt(2) apart at it"""
    dim, eps = 300, 2.0 ** -66 * target ** 2
    level = torch.tensor([0.0, 2.0 ** -60, 2.0 ** -34, 2.0 ** -33, 2.0 ** -32, 2.0 ** -18, 1.0, 2.0 ** 40])[:, None]
    x = rand(8, dim, seed=90)
    x = x / x.double().square().mean(1, keepdim=True).sqrt().float() * level * target
    want = x.double() / (x.double().square().mean(1, keepdim=True) / target ** 2).clamp_min(2.0 ** -66).sqrt()
    y = int8.rms_norm(x.cuda(), torch.full((dim,), target, device="cuda"), eps).double().cpu()
    # away from the floor: 1 / sqrt(1 + a), a <= 2^-30, beside the roundings of check_norm
    far = [0, 1, 5, 6, 7]
    assert bool(((y - want).abs()[far] <= want.abs()[far] * (6 * U + 2.0 ** -30)).all())
    ratio = (want / y)[2:5][:, x[2].abs() > 0]
    assert float(ratio.min()) >= 1 - 7 * U and float(ratio.max()) <= 2 ** 0.5 * (1 + 7 * U)
    assert float(ratio[1].min()) > 1.41


def test_a_gain_that_leaves_the_range_is_told():
    """finite rows whose h * gain is none: codes of nothing under a NaN scale, in their row only"""
    x = rand(3, 64, seed=91)
    x[1, 5] = 2e38
    gain = torch.full((64,), 4.0, device="cuda")
    q, scale = int8.rms_norm_int8(x.cuda(), gain, EPS)
    assert bool(torch.isnan(scale[1])) and int(q[1].abs().max()) == 0
    check_codes(q[[0, 2]], scale[[0, 2]], norm64(x[[0, 2]], gain.cpu(), EPS)[1])
    check_norm(int8.rms_norm(x.cuda(), gain, EPS), norm64(x, gain.cpu(), EPS)[1], torch.float32)


def test_a_handle_is_destroyed_while_a_stream_is_captured():
    """by the capturing thread and by another one: the capture goes on, and the memory is given back"""
    import threading

    from kaldi_amd._lib import lib
    n, k = 4096, 65536
    w, ws, bias, _, _ = layer_of(64, 40, 92, True)
    layer = int8.AffineInt8(w.cuda(), ws.cuda(), bias.cuda())
    large = [int8.AffineInt8(torch.ones(1, 1, dtype=torch.int8, device="cuda").expand(n, k), torch.ones(n, device="cuda")) for _ in range(2)]
    torch.cuda.empty_cache()
    q, scale = on_device(codes(5, 64, 93)), torch.rand(5, device="cuda")
    want = layer.propagate(q, scale)
    torch.cuda.synchronize()

    def free():
        from ctypes import byref, c_size_t
        f, t = c_size_t(), c_size_t()
        assert lib().kamd_device_mem_info(byref(f), byref(t)) == 0
        return f.value
    before = free()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer.propagate(q, scale)
        large.pop()
        other = threading.Thread(target=large.clear)
        other.start()
        other.join()
        z = layer.propagate(q, scale, torch.bfloat16)
    for _ in range(3):
        y.zero_()
        z.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want.bfloat16())
    torch.cuda.empty_cache()
    assert free() - before > n * k                                       # (both of them: 2 n k bytes, beside what the graph takes)


def test_layers_are_not_made_while_the_stream_is_captured():
    """refused without breaking the capture"""
    w, ws, bias, _, _ = layer_of(64, 40, 94, True)
    w, ws, bias = w.cuda(), ws.cuda(), bias.cuda()
    layer = int8.AffineInt8(w, ws, bias)
    q, scale = on_device(codes(5, 64, 95)), torch.rand(5, device="cuda")
    want = layer.propagate(q, scale)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = layer.propagate(q, scale)
        for make in (lambda: int8.AffineInt8(w, ws, bias), lambda: int8.AffineInt8.from_layer(Layer("c", 8, 4, [0], -1, np.ones((4, 8), np.float32)))):
            with pytest.raises(KamdError, match="being captured"):
                make()
        z = layer.propagate(q, scale)
    for _ in range(3):
        y.zero_()
        z.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want)
    assert torch.equal(int8.AffineInt8(w, ws, bias).propagate(q, scale), want)
