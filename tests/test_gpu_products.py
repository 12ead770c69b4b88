"""The experts' products on the GPU against plain 64-bit products, expert by expert.

Most inputs are small whole numbers: every product and partial sum is then exact in fp32 (and in
int32) in any order, so the result has to equal the 64-bit one rounded once, bit for bit.
"""

from __future__ import annotations

import re
import sys

import pytest
import torch

from vibe_megakernel_amd import _lib, products
from vibe_megakernel_amd import cases as C
from vibe_megakernel_amd import submission

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _log(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def _whole(shape, dtype, seed, most=4):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV, dtype=torch.int8).to(dtype)


def _counts(values):
    return torch.tensor(values, dtype=torch.int64, device=DEV)


def _each(counts):
    first = 0
    for e, c in enumerate(counts):
        yield e, first, first + c
        first += c


def _product(x, w, counts, transposed=False):
    """64-bit products; rows of no expert are zero."""
    y = torch.zeros((x.shape[0], w.shape[2 if transposed else 1]), dtype=torch.float64, device=DEV)
    for e, a, b in _each(counts):
        if b > a:
            m = w[e].double() if transposed else w[e].double().T.contiguous()
            y[a:b] = x[a:b].double() @ m
    return y


def _wgrad(dy, x, counts):
    dw = torch.zeros((len(counts), dy.shape[1], x.shape[1]), dtype=torch.float64, device=DEV)
    for e, a, b in _each(counts):
        dw[e] = dy[a:b].double().T.contiguous() @ x[a:b].double()
    return dw


def _same(got, want, what=""):
    if not torch.equal(got, want.to(got.dtype)):
        off = (got.double() - want.to(got.dtype).double()).abs()
        at = [int(i) for i in (off.nan_to_num(nan=1e30) > 0).nonzero()[0]]
        raise AssertionError(f"{what}: {int((off != 0).sum())} of {off.numel()} differ, first at {at}: "
                             f"{got[tuple(at)]} for {want[tuple(at)]}")


# (counts, K, N, rows of no expert): empty experts first, last and all; one row; tiles that are
# just full, one short and one over; sizes that are no multiple of a tile, of 16 bytes, or odd.
SHAPES = [
    ([1], 64, 64, 0), ([0, 1, 0], 32, 16, 0), ([0, 0, 0, 0], 64, 128, 5), ([3, 0, 5], 1, 1, 2),
    ([2, 7, 1], 40, 24, 0), ([5, 0, 3, 0, 9], 128, 136, 4), ([64, 63, 65], 72, 200, 0),
    ([16, 17, 15, 33], 520, 264, 1), ([255, 256, 257], 64, 256, 0), ([300, 0, 12], 200, 512, 70),
    ([128, 129, 127], 1000, 264, 0), ([1, 600], 192, 520, 3), ([70, 0, 5], 33, 65, 6), ([9, 2], 1001, 7, 0),
    ([1] * 8 + [0] * 120, 2048, 192, 0), ([4, 2, 0, 3] * 20, 256, 96, 0), ([0] * 1023 + [2], 64, 16, 1),
    ([1] * 1024, 16, 8, 0), ([512, 512], 328, 1032, 0), ([2000], 136, 264, 0), ([8], 4096, 32, 0),
]
IDS = [f"e{len(s[0])}r{sum(s[0])}-k{s[1]}n{s[2]}+{s[3]}" for s in SHAPES]


@pytest.mark.parametrize("dtype", (BF16, FP16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("transposed", (False, True), ids=("nk", "kn"))
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_grouped_mm_is_exact_on_whole_numbers(shape, transposed, dtype):
    counts, K, N, tail = shape
    _log(f"grouped_mm {counts[:6]} K={K} N={N} tail={tail} {dtype} transposed={transposed}")
    x = _whole((sum(counts) + tail, K), dtype, 1)
    w = _whole((len(counts), K, N) if transposed else (len(counts), N, K), dtype, 2)
    want = _product(x, w, counts, transposed)
    _same(products.grouped_mm(x, w, _counts(counts), transposed=transposed), want, "y")


@pytest.mark.parametrize("dtype", (BF16, FP16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_weight_gradient_is_exact_on_whole_numbers(shape, dtype):
    counts, K, N, tail = shape
    _log(f"wgrad {counts[:6]} K={K} N={N} tail={tail} {dtype}")
    R = sum(counts) + tail
    x, dy = _whole((R, K), dtype, 3), _whole((R, N), dtype, 4, most=2)
    _same(products.grouped_mm_wgrad(dy, x, _counts(counts)), _wgrad(dy, x, counts), "dw")


@pytest.mark.parametrize("out_dtype", (BF16, FP16, FP32), ids=("bf16", "fp16", "fp32"))
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_grouped_int8_mm_is_exact(shape, out_dtype):
    """(fp32(sum) * x_scale) * w_scale, each step rounded to fp32 as PyTorch rounds it."""
    counts, K, N, tail = shape
    _log(f"grouped_int8 {counts[:6]} K={K} N={N} tail={tail} {out_dtype}")
    R, E = sum(counts) + tail, len(counts)
    x, w = _whole((R, K), torch.int8, 5, most=127), _whole((E, N, K), torch.int8, 6, most=127)
    g = torch.Generator(device=DEV).manual_seed(7)
    xs, ws = torch.rand(R, generator=g, device=DEV) * 0.01, torch.rand((E, N), generator=g, device=DEV) * 0.01
    total = _product(x, w, counts)
    scale = torch.zeros((R, N), device=DEV)
    for e, a, b in _each(counts):
        scale[a:b] = ws[e]
    want = total.float() * xs[:, None] * scale
    _same(products.grouped_int8_mm(x, xs, w, ws, _counts(counts), out_dtype=out_dtype), want, "y")


@pytest.mark.parametrize("M,K,N", [(1, 64, 16), (1, 7168, 512), (3, 1000, 33), (17, 272, 48), (256, 128, 256),
                                   (257, 2048, 520), (1, 1, 1), (64, 33, 65), (40, 4096, 1024)])
def test_int8_mm_is_exact(M, K, N):
    _log(f"int8_mm M={M} K={K} N={N}")
    x, w = _whole((M, K), torch.int8, 8, most=127), _whole((N, K), torch.int8, 9, most=127)
    g = torch.Generator(device=DEV).manual_seed(10)
    xs, ws = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    want = (x.double() @ w.double().T.contiguous()).float() * xs[:, None] * ws
    for out_dtype in (BF16, FP32):
        _same(products.int8_mm(x, xs, w, ws, out_dtype=out_dtype), want, f"y {out_dtype}")


def test_int8_extremes_do_not_overflow():
    """-128 * -128 at the largest K stays within int32; its fp32 value is exact (a power of two
    times less than 2^24)."""
    K = 131071
    x = torch.full((2, K), -128, dtype=torch.int8, device=DEV)
    one = torch.ones(2, device=DEV)
    y = products.int8_mm(x, one, x, one, out_dtype=FP32)
    assert torch.equal(y, torch.full((2, 2), float(K * 16384), device=DEV))


@pytest.mark.parametrize("dtype", (BF16, FP16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("transposed", (False, True), ids=("nk", "kn"))
@pytest.mark.parametrize("counts,K,N", [([40, 0, 300, 7], 1536, 384), ([2, 1, 3], 2048, 256)])
def test_normal_inputs_within_the_rounding(counts, K, N, transposed, dtype):
    """|error| <= half a step of the result's type (finfo.eps / 2 of the value, half the smallest
    subnormal near zero) plus one unit of fp32 (2^-23) for each of the K additions, of the
    partial sums' bound sum |x w|. dw: the same with the expert's rows for K."""
    g = torch.Generator(device=DEV).manual_seed(11)
    R, E = sum(counts), len(counts)
    x = torch.randn((R, K), generator=g, device=DEV).to(dtype)
    w = (torch.randn((E, K, N) if transposed else (E, N, K), generator=g, device=DEV) * 0.02).to(dtype)
    dy = (torch.randn((R, N), generator=g, device=DEV) * 0.1).to(dtype)
    c, info = _counts(counts), torch.finfo(dtype)

    def near(got, want, size, terms, what):
        allowed = info.eps / 2 * want.abs() + info.smallest_normal * info.eps / 2 + terms * 2.0**-23 * size
        assert bool(((got.double() - want).abs() <= allowed * (1 + 2.0**-20)).all()), what

    near(products.grouped_mm(x, w, c, transposed=transposed), _product(x, w, counts, transposed),
         _product(x.abs(), w.abs(), counts, transposed), K, "y")
    near(products.grouped_mm_wgrad(dy, x, c), _wgrad(dy, x, counts), _wgrad(dy.abs(), x.abs(), counts), max(counts), "dw")


@pytest.mark.parametrize("dtype", (BF16, FP16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("transposed", (False, True), ids=("nk", "kn"))
@pytest.mark.parametrize("counts,K,N,tail", [([5, 0, 33, 2], 96, 72, 7), ([260, 1, 0], 64, 264, 0), ([3, 4], 33, 21, 1)])
def test_gradients(counts, K, N, tail, transposed, dtype):
    """Both gradients against their formulas and against differences. x and w are whole numbers up
    to 2 and dy is sparse with entries 0 and +-1, so no result passes 256 and each is held exactly
    in either type. y is linear in x and in w: <dy, y(x + h) - y(x)> has to equal <dx, h>, and
    with w likewise, without any error."""
    E, R, c = len(counts), sum(counts) + tail, _counts(counts)
    x = _whole((R, K), dtype, 12, most=2).requires_grad_()
    w = _whole((E, K, N) if transposed else (E, N, K), dtype, 13, most=2).requires_grad_()
    dy = _whole((R, N), dtype, 14, most=1) * (_whole((R, N), dtype, 15, most=9).abs() > 8)
    y = products.grouped_mm(x, w, c, transposed=transposed)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    with torch.no_grad():
        kn = w if transposed else w.transpose(1, 2).contiguous()  # [E, K, N]
        want = [_product(x, kn, counts, True), _exact_dx(dy, kn, counts), _wgrad(dy, x, counts)]
        if transposed:
            want[2] = want[2].transpose(1, 2)
        for name, got, exactly in zip(("y", "dx", "dw"), (y, dx, dw), want):
            assert float(exactly.abs().max()) <= 256, "the inputs are to keep every result exact"
            _same(got, exactly, name)
        hx, hw = _whole(x.shape, dtype, 16, most=1), _whole(w.shape, dtype, 17, most=1)
        forward = lambda a, b: products.grouped_mm(a, b, c, transposed=transposed).double()  # noqa: E731
        inner = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731
        assert inner(dy, forward(hx, w)) == inner(dx, hx) != 0
        assert inner(dy, forward(x, hw)) == inner(dw, hw) != 0
        # The same with both ends of the difference, halved steps of x and w being whole again.
        assert inner(dy, forward(x + hx, w) - forward(x - hx, w)) == 2 * inner(dx, hx)
        assert inner(dy, forward(x, w + hw) - forward(x, w - hw)) == 2 * inner(dw, hw)


def _exact_dx(dy, wt, counts):
    return _product(dy, wt.transpose(1, 2).contiguous(), counts, True)


@pytest.mark.parametrize("transposed", (False, True), ids=("nk", "kn"))
def test_second_derivatives(transposed):
    """The gradients are bilinear like the product: of <dx, v> and <dw, u> the derivatives are again
    products of the same kind, on these whole numbers exact."""
    counts, c, K, N = [5, 0, 9], _counts([5, 0, 9]), 40, 24
    x, dy = _whole((14, K), BF16, 140, most=1).requires_grad_(), _whole((14, N), BF16, 141, most=1).requires_grad_()
    w = _whole((3, K, N) if transposed else (3, N, K), BF16, 142, most=1).requires_grad_()
    v, u = _whole((14, K), BF16, 143, most=1), _whole(w.shape, BF16, 144, most=1)
    y = products.grouped_mm(x, w, c, transposed=transposed)
    dx, dw = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    by_dy, by_w = torch.autograd.grad(dx, (dy, w), v, retain_graph=True)
    back_dy, by_x = torch.autograd.grad(dw, (dy, x), u)
    with torch.no_grad():
        turned = lambda t: t.transpose(1, 2) if transposed else t  # noqa: E731
        _same(by_dy, _product(v, w, counts, transposed), "<dx, v> by dy")
        _same(by_w, turned(_wgrad(dy, v, counts)), "<dx, v> by w")
        _same(back_dy, _product(x, u, counts, transposed), "<dw, u> by dy")
        _same(by_x, _product(dy, u, counts, not transposed), "<dw, u> by x")


def test_gradient_of_broadcast_rows_and_of_one_input():
    """A result summed to a number hands back a broadcast gradient; x itself may be a broadcast
    row; and only the gradient that is asked for is made."""
    counts, c = [3, 2], _counts([3, 2])
    w = _whole((2, 24, 16), BF16, 18).requires_grad_()
    row = _whole((1, 16), BF16, 19).requires_grad_()
    y = products.grouped_mm(row.expand(5, 16), w, c)
    drow, dw = torch.autograd.grad(y.sum(), (row, w))
    ones = torch.ones((5, 24), dtype=BF16, device=DEV)
    wt = w.detach().transpose(1, 2).contiguous()
    _same(drow, _exact_dx(ones, wt, counts).to(BF16).sum(0, keepdim=True), "row")
    _same(dw, _wgrad(ones, row.detach().expand(5, 16), counts), "dw")
    x = _whole((5, 16), BF16, 20)
    y = products.grouped_mm(x, w, c)
    assert torch.equal(torch.autograd.grad(y, w, ones)[0], products.grouped_mm_wgrad(ones, x, c))
    with torch.no_grad():
        assert not products.grouped_mm(x, w, c).requires_grad


@pytest.mark.parametrize("dtype", (BF16, FP16, torch.int8), ids=("bf16", "fp16", "int8"))
def test_strides_offsets_and_given_results(dtype):
    """Rows within wider buffers, at 16-byte aligned and at odd places; rows of no expert stay as
    they were in a given result."""
    counts, K, N, tail = [7, 0, 30], 128, 64, 4
    R, c = sum(counts) + tail, _counts([7, 0, 30])
    for pad, at in ((64, 0), (64, 32), (3, 1)):
        big = _whole((R, K + pad), dtype, 21)
        x = big[:, at:at + K]
        w = _whole((3, N, K), dtype, 22)
        want = _product(x, w, counts)
        keep = torch.full((R, N + pad), 77.0, dtype=BF16 if dtype == torch.int8 else dtype, device=DEV)
        out = keep[:, at:at + N]
        if dtype == torch.int8:
            one = torch.ones(R, device=DEV)
            got = products.grouped_int8_mm(x, one, w, torch.ones((3, N), device=DEV), c, out=out)
        else:
            got = products.grouped_mm(x, w, c, out=out)
        assert got is out
        _same(out[:R - tail], want[:R - tail], f"pad {pad}")
        keep[:R - tail, at:at + N] = 77.0
        assert bool((keep == 77.0).all()), "values outside the result, or rows of no expert, changed"


def test_wgrad_strides_and_given_result():
    counts, K, N = [9, 0, 40], 72, 48
    bx, bd = _whole((49, K + 24), BF16, 23), _whole((49, N + 8), BF16, 24)
    for x, dy in ((bx[:, 8:8 + K], bd[:, 8:8 + N]), (bx[:, 3:3 + K], bd[:, 1:1 + N])):
        out = torch.full((3, N, K), 5.0, dtype=BF16, device=DEV)
        assert products.grouped_mm_wgrad(dy, x, _counts(counts), out=out) is out
        _same(out, _wgrad(dy, x, counts), "dw")


BAD_COUNTS = ([-1, 4], [5, 6], [1 << 62, 1 << 62], [-(1 << 62), 3], [2**31, 0], [2**32 + 1, 0])


@pytest.mark.parametrize("counts", BAD_COUNTS, ids=str)
def test_bad_counts_make_every_element_nan(counts):
    """Counts that are negative or pass the rows (10) alone or together; sums are taken without
    wrapping around."""
    c = _counts(counts)
    for K, N in ((64, 64), (33, 21)):
        x, w = _whole((10, K), BF16, 25), _whole((2, N, K), BF16, 26)
        _log(f"bad counts {counts} K={K}")
        assert bool(products.grouped_mm(x, w, c).isnan().all())
        assert bool(products.grouped_mm(x, w.transpose(1, 2).contiguous(), c, transposed=True).isnan().all())
        assert bool(products.grouped_mm_wgrad(_whole((10, N), BF16, 27), x, c).isnan().all())
        y = products.grouped_int8_mm(x.char(), torch.ones(10, device=DEV), w.char(), torch.ones((2, N), device=DEV), c)
        assert bool(y.isnan().all())


def test_infinities_and_nan_stay_in_their_rows():
    """Rows of no expert, other experts' rows and the padding of a tile never reach a result; a
    row's own NaN does."""
    counts, K, N, tail = [5, 0, 70], 136, 72, 6
    x, w = _whole((81, K), BF16, 28), _whole((3, N, K), BF16, 29)
    dy = _whole((81, N), BF16, 30)
    x[75:] = float("nan")
    dy[75:] = float("inf")
    w[1] = float("nan")  # the expert without rows
    clean = x.clone()
    clean[75:] = 0
    wc = w.clone()
    wc[1] = 0
    _same(products.grouped_mm(x, w, _counts(counts)), _product(clean, wc, counts), "y")
    _same(products.grouped_mm_wgrad(dy, x, _counts(counts)), _wgrad(dy[:75], clean[:75], counts), "dw")
    x[2, 3] = float("nan")
    y = products.grouped_mm(x, w, _counts(counts))
    assert bool(y[2].isnan().all()) and not bool(y[torch.arange(81, device=DEV) != 2].isnan().any())


def test_zero_sized_products():
    c = _counts([0, 0])
    assert products.grouped_mm(torch.empty((0, 16), dtype=BF16, device=DEV), _whole((2, 8, 16), BF16, 1), c).shape == (0, 8)
    y = products.grouped_mm(torch.empty((3, 0), dtype=BF16, device=DEV), torch.empty((2, 8, 0), dtype=BF16, device=DEV),
                            _counts([1, 2]))
    assert torch.equal(y, torch.zeros((3, 8), dtype=BF16, device=DEV))
    dw = products.grouped_mm_wgrad(torch.empty((0, 8), dtype=BF16, device=DEV),
                                   torch.empty((0, 16), dtype=BF16, device=DEV), c)
    assert torch.equal(dw, torch.zeros((2, 8, 16), dtype=BF16, device=DEV))
    q, s = products.quantize_rows_int8(torch.empty((0, 16), dtype=BF16, device=DEV))
    assert q.shape == (0, 16) and s.shape == (0,)


def test_long_offsets():
    """Weights and rows past 2^31 elements: the last expert and the last rows."""
    E, N, K = 70, 4096, 8192  # 2.3e9 elements
    w = torch.zeros((E, N, K), dtype=BF16, device=DEV)
    w[-1] = _whole((N, K), BF16, 31, most=1)
    counts = [0] * (E - 1) + [3]
    x = _whole((3, K), BF16, 32, most=1)
    want = x.double() @ w[-1].double().T.contiguous()
    _same(products.grouped_mm(x, w, _counts(counts)), want, "weights")
    dy = _whole((3, N), BF16, 33, most=1)
    _same(products.grouped_mm(dy, w, _counts(counts), transposed=True), dy.double() @ w[-1].double(), "transposed weights")
    del w
    R = 70000
    big = torch.zeros((R, 32768), dtype=BF16, device=DEV)  # 2.3e9 elements, a row stride of 32768
    x = big[:, :64]
    x[-2:] = _whole((2, 64), BF16, 34)
    w = _whole((2, 16, 64), BF16, 35)
    y = products.grouped_mm(x, w, _counts([R - 2, 2]))
    _same(y[-2:], x[-2:].double() @ w[1].double().T.contiguous(), "rows")
    dy = torch.zeros((R, 16), dtype=BF16, device=DEV)
    dy[-2:] = _whole((2, 16), BF16, 36)
    _same(products.grouped_mm_wgrad(dy, x, _counts([R - 2, 2]))[1], dy[-2:].double().T.contiguous() @ x[-2:].double(),
          "wgrad rows")


# Calls that the rules send to each kernel: (counts, K, N), with each of them the tiles and whether
# the weights go past the caches, in the form y = x w^T and in y = x w.
SIZES = {
    (256, 256, True): ([90, 110, 0, 200] * 16, 256, 520), (256, 256, False): ([3900, 4100], 256, 1032),
    (256, 128, True): ([4, 12, 0, 16] * 2, 256, 6144), (256, 128, False): ([4100, 3900], 256, 520),
    (128, 128, True): ([2, 1, 5, 0] * 16, 256, 520), (128, 128, False): ([260, 340] * 4, 4096, 520),
}


def _kernels(call):
    """(kernel, its type, its numbers) of every products kernel that ``call`` launches, from the profiler's names,
    demangled or not."""
    call()
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        call()
        torch.cuda.synchronize()
    found = set()
    for e in prof.events():
        kernel = re.search(r"k_(tiles|strips|product_any|wgrad_any|quantize_int8_any|quantize_int8)", e.name)
        if kernel:
            kind = re.search(r"Bf16|Fp16|Int8", e.name)
            plain = e.name.replace("true", "1").replace("false", "0")
            numbers = re.findall(r"(?<=L[ib])\d+(?=E)|(?<=FormE)\d(?=E)|(?<=[ )])\d+(?=[,>])", plain)
            found.add((kernel.group(1), kind.group(0) if kind else "", tuple(int(n) for n in numbers)[-3:]))
    return found


def _reached(kernel, kind, numbers, call):
    """Asserts that ``call`` launches it. Demangled names can lose the first numbers, but not the last ones' order."""
    found = _kernels(call)
    assert any(name == kernel and k == kind and n == numbers[len(numbers) - len(n):] for name, k, n in found), found


@pytest.mark.parametrize("dtype", (BF16, FP16, torch.int8), ids=("bf16", "fp16", "int8"))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}x{s[1]}{'-once' if s[2] else ''}")
def test_every_tile_size_is_reached_and_exact(size, dtype):
    counts, K, N = SIZES[size]
    kind = {BF16: "Bf16", FP16: "Fp16", torch.int8: "Int8"}[dtype]
    _log(f"{size} {dtype}: {sum(counts)} rows of {len(counts)} experts, K={K} N={N}")
    x, c = _whole((sum(counts) + 3, K), dtype, 150, most=3), _counts(counts)
    if dtype == torch.int8:
        w, one = _whole((len(counts), N, K), dtype, 151, most=3), torch.ones(len(x), device=DEV)
        ws = torch.ones((len(counts), N), device=DEV)
        for out_dtype in (BF16, FP16, FP32):
            call = lambda: products.grouped_int8_mm(x, one, w, ws, c, out_dtype=out_dtype)  # noqa: E731
            _reached("tiles", kind, size, call)
            _same(call(), _product(x, w, counts).float(), f"y {out_dtype}")
        return
    for transposed in (False, True):
        w = _whole((len(counts), K, N) if transposed else (len(counts), N, K), dtype, 151, most=3)
        call = lambda: products.grouped_mm(x, w, c, transposed=transposed)  # noqa: E731
        _reached("tiles", kind, size, call)
        _same(call(), _product(x, w, counts, transposed), "y")


@pytest.mark.parametrize("dtype", (BF16, FP16, torch.int8), ids=("bf16", "fp16", "int8"))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}x{s[1]}{'-once' if s[2] else ''}")
def test_tiles_store_rows_that_are_not_aligned(size, dtype):
    """An odd N, and results whose rows start anywhere; what lies between them stays."""
    counts, K, N = SIZES[size]
    N, R = N + 3, sum(counts)
    _log(f"{size} {dtype}: {R} rows of {len(counts)} experts, K={K} N={N}")
    x, c = _whole((R, K), dtype, 160, most=3), _counts(counts)
    w = _whole((len(counts), N, K), dtype, 161, most=3)
    for out_dtype in (BF16, FP16, FP32) if dtype == torch.int8 else (dtype,):
        out = torch.full((R, N + 6), 7.0, dtype=out_dtype, device=DEV)
        if dtype == torch.int8:
            products.grouped_int8_mm(x, torch.ones(R, device=DEV), w, torch.ones((len(counts), N), device=DEV), c,
                                     out_dtype=out_dtype, out=out[:, 1:N + 1])
        else:
            products.grouped_mm(x, w, c, out=out[:, 1:N + 1])
        want = _product(x, w, counts)
        _same(out[:, 1:N + 1], want.float() if dtype == torch.int8 else want, f"y {out_dtype}")
        assert bool((out[:, 0] == 7).all()) and bool((out[:, N + 1:] == 7).all())


@pytest.mark.parametrize("dtype", (BF16, FP16), ids=("bf16", "fp16"))
@pytest.mark.parametrize("size", SIZES, ids=lambda s: f"{s[0]}x{s[1]}{'-once' if s[2] else ''}")
def test_tiles_read_strided_rows_and_nothing_between(size, dtype):
    """Rows in a wider tensor whose other columns, and rows behind the last expert's, are NaN."""
    counts, K, N = SIZES[size]
    S = sum(counts)
    _log(f"{size} {dtype}: {S} rows of {len(counts)} experts, K={K} N={N}")

    def within(values):
        wide = torch.full((S + 5, values.shape[1] + 24), float("nan"), dtype=dtype, device=DEV)
        wide[:S, 8:-16] = values
        return wide[:, 8:-16]

    x, dy, c = _whole((S, K), dtype, 164, most=3), _whole((S, N), dtype, 165, most=3), _counts(counts)
    w = _whole((len(counts), N, K), dtype, 166, most=3)
    y = products.grouped_mm(within(x), w, c)
    _same(y[:S], _product(x, w, counts), "y")
    assert bool((y[S:] == 0).all())
    dx = torch.full((S + 5, K), 7.0, dtype=dtype, device=DEV)
    products.grouped_mm(within(dy), w, c, transposed=True, out=dx)
    _same(dx[:S], _product(dy, w, counts, True), "dx")
    assert bool((dx[S:] == 7).all())
    _same(products.grouped_mm_wgrad(within(dy), within(x), c), _wgrad(dy, x, counts), "dw")
    c[-1] += 6  # one row more than there are
    assert bool(products.grouped_mm(within(x), w, c).isnan().all())
    assert bool(products.grouped_mm_wgrad(within(dy), within(x), c).isnan().all())


def test_weight_gradient_tiles_store_anywhere():
    for counts, K, N in (([30] * 20, 1024, 1000), ([30, 5], 512, 520), ([700, 0, 3] * 3, 2048, 776)):
        x, dy, c = _whole((sum(counts), K), BF16, 162), _whole((sum(counts), N), BF16, 163), _counts(counts)
        flat = torch.full((len(counts) * N * K + 2,), 7.0, dtype=BF16, device=DEV)
        dw = flat[1:-1].view(len(counts), N, K)
        products.grouped_mm_wgrad(dy, x, c, out=dw)
        _same(dw, _wgrad(dy, x, counts), "dw")
        assert flat[0] == 7 and flat[-1] == 7


def test_the_other_kernels_are_reached():
    """Strips of both sizes, both tile sizes of the weights' gradient, the kernels of any alignment."""
    for dtype, kind in ((BF16, "Bf16"), (FP16, "Fp16")):
        for counts, K, N, strip in (([1] * 8, 2048, 768, (1, 1)), ([256], 2048, 768, (2, 2))):
            x, w, c = _whole((sum(counts), K), dtype, 152), _whole((len(counts), N, K), dtype, 153), _counts(counts)
            _reached("strips", kind, strip, lambda: products.grouped_mm(x, w, c))
            _same(products.grouped_mm(x, w, c), _product(x, w, counts), "y")
        for counts, K, N, size in (([30] * 20, 1024, 1000, (256, 256)), ([30, 5], 512, 520, (128, 128))):
            x, dy, c = _whole((sum(counts), K), dtype, 154), _whole((sum(counts), N), dtype, 155), _counts(counts)
            _reached("tiles", kind, (*size, 0), lambda: products.grouped_mm_wgrad(dy, x, c))
            _same(products.grouped_mm_wgrad(dy, x, c), _wgrad(dy, x, counts), "dw")
        x, w, c = _whole((5, 33), dtype, 156), _whole((1, 9, 33), dtype, 157), _counts([5])
        names = _kernels(lambda: (products.grouped_mm(x, w, c), products.grouped_mm_wgrad(_whole((5, 9), dtype, 1), x, c)))
        assert {n[:2] for n in names} == {("product_any", kind), ("wgrad_any", kind)}
    one = torch.ones(256, device=DEV)
    for M, strip in ((1, (1, 1)), (256, (2, 2))):
        x, w = _whole((M, 2048), torch.int8, 158), _whole((768, 2048), torch.int8, 159)
        _reached("strips", "Int8", strip, lambda: products.int8_mm(x, one[:M], w, torch.ones(768, device=DEV)))
    for dtype in (BF16, FP16, FP32):
        wide = 16 // dtype.itemsize
        for chunks, kernel in ((64, (1, 1)), (128, (2, 1)), (256, (1, 0)), (512, (2, 0)), (1024, (4, 0)), (2048, (8, 0))):
            x = _whole((3, chunks * wide), dtype, 160)
            _reached("quantize_int8", "", kernel, lambda: products.quantize_rows_int8(x))
        _reached("quantize_int8_any", "", (), lambda: products.quantize_rows_int8(_whole((3, 33), dtype, 1)))


# ---------------------------------------------------------------------------------------
# Rows to int8
# ---------------------------------------------------------------------------------------

def _quantized(x):
    """The rule in fp32 on the CPU (127.0 / a would be a reciprocal and a product, rounded twice)."""
    v = x.float().cpu()
    a = v.abs().amax(dim=1).clamp_min(2.0**-100)
    q = torch.round(v * (torch.full_like(a, 127.0) / a)[:, None])
    return q.to(torch.int8), a / torch.full_like(a, 127.0)


@pytest.mark.parametrize("dtype", (BF16, FP16, FP32), ids=("bf16", "fp16", "fp32"))
@pytest.mark.parametrize("rows,cols", [(1, 7168), (1, 1), (5, 33), (64, 128), (7, 1000), (300, 2048), (3, 16384),
                                       (2, 16385), (2, 70001), (4099, 72)])
def test_quantize_rows_int8_equals_the_rule(rows, cols, dtype):
    g = torch.Generator(device=DEV).manual_seed(40)
    x = (torch.randn((rows, cols), generator=g, device=DEV) * torch.logspace(-3, 2, rows, device=DEV)[:, None]).to(dtype)
    q, s = products.quantize_rows_int8(x)
    wq, ws = _quantized(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    # Half a step of 1/127 of the row's largest, and the roundings of 127 / a, of the product and of
    # a / 127 (2^-24 each of at most 127 steps: 3 * 127 * 2^-24 < 2^-15 of a step).
    off = (q.double() * s.double()[:, None] - x.double()).abs()
    assert bool((off <= s.double()[:, None] * (0.5 + 2.0**-15)).all())


def test_quantize_rows_int8_edges():
    x = torch.zeros((9, 40), dtype=FP32, device=DEV)
    x[1, 7] = float("nan")
    x[2, 0] = float("inf")
    x[3, 39] = float("-inf")
    x[4] = 3.0e38
    x[5, 5] = -1e-40
    x[6, ::2], x[6, 1::2] = 127.0, 0.5  # ties go to the even value
    x[7, 0], x[7, 1], x[7, 2] = 127.0, 1.5, -2.5
    x[8, 3] = 2.0**-101
    q, s = products.quantize_rows_int8(x)
    keep = [0, 4, 5, 6, 7, 8]
    wq, ws = _quantized(x)
    assert torch.equal(q.cpu()[keep], wq[keep]) and torch.equal(s.cpu()[keep], ws[keep])
    assert bool(s[1:4].isnan().all()) and not bool(q[1:4].any())
    assert q[6, 1] == 0 and q[7, 1] == 2 and q[7, 2] == -2 and int(q[4].min()) == 127
    wide = torch.randn((6, 100), device=DEV).to(BF16)
    for view in (wide[:, 3:90], wide[:, 8:72], wide[::2], wide.t(), wide[:1].expand(4, 100)):
        q, s = products.quantize_rows_int8(view)
        wq, ws = _quantized(view)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


# ---------------------------------------------------------------------------------------
# Streams, graphs, refusals, and the products together
# ---------------------------------------------------------------------------------------

def test_refusals():
    x, w, c = _whole((6, 16), BF16, 50), _whole((2, 8, 16), BF16, 51), _counts([3, 3])
    xq, wq, one = x.char(), w.char(), torch.ones(6, device=DEV)
    ws = torch.ones((2, 8), device=DEV)
    calls = [
        lambda: products.grouped_mm(x.float(), w.float(), c), lambda: products.grouped_mm(x, w.half(), c),
        lambda: products.grouped_mm(x, w[0], c), lambda: products.grouped_mm(x, w, c.int()),
        lambda: products.grouped_mm(x, w, c[:1]), lambda: products.grouped_mm(x[0], w, c),
        lambda: products.grouped_mm(x[:, :8], w, c), lambda: products.grouped_mm(x, w, c, transposed=True),
        lambda: products.grouped_mm(x, w.transpose(1, 2), c, transposed=True), lambda: products.grouped_mm(x, w, c.cpu()),
        lambda: products.grouped_mm(x, w, None), lambda: products.grouped_mm(x, w, c, out=x),
        lambda: products.grouped_mm(x, w, c, out=torch.empty((6, 8), dtype=FP16, device=DEV)),
        lambda: products.grouped_mm(x, w, c, out=torch.empty((8, 6), dtype=BF16, device=DEV).t()),
        lambda: products.grouped_mm(x, w, c, out=w.view(16, 16)[:6, :8]),
        lambda: products.grouped_mm(x.clone().requires_grad_(), w, c, out=torch.empty((6, 8), dtype=BF16, device=DEV)),
        lambda: products.grouped_mm(x, w[:0], c[:0]),
        lambda: products.grouped_mm_wgrad(x, w[0], c), lambda: products.grouped_mm_wgrad(x.half(), x, c),
        lambda: products.grouped_mm_wgrad(x, x, c.view(1, 2)),
        lambda: products.int8_mm(x, one, wq[0], ws[0]), lambda: products.int8_mm(xq, one[:5], wq[0], ws[0]),
        lambda: products.int8_mm(xq, one, wq, ws), lambda: products.int8_mm(xq, one.half(), wq[0], ws[0]),
        lambda: products.int8_mm(xq, one, wq[0], ws[0], out_dtype=torch.float64),
        lambda: products.grouped_int8_mm(xq, one, wq[0], ws[0], c),
        lambda: products.grouped_int8_mm(xq, one, wq, ws[:, :4], c), lambda: products.grouped_int8_mm(xq, one, wq, ws, None),
        lambda: products.quantize_rows_int8(xq), lambda: products.quantize_rows_int8(x[0]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was accepted")
    with pytest.raises(_lib.MegaMoEError):  # more experts than the limit
        products.grouped_mm(x, torch.zeros((1025, 8, 16), dtype=BF16, device=DEV), torch.zeros(1025, dtype=torch.int64, device=DEV))


def test_other_streams():
    """Work is issued on torch's current stream: a product on a side stream follows what was
    issued there before it."""
    counts, side = [40, 30], torch.cuda.Stream(DEV)
    x, w = _whole((70, 256), BF16, 52), _whole((2, 512, 256), BF16, 53)
    want = _product(x, w, counts)
    late = torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        y = products.grouped_mm(late, w, _counts(counts))
    side.synchronize()
    _same(y, want, "y")


def test_captured_products_replay_on_new_inputs():
    """Two graphs of the forward and both gradients (and the int8 products), replayed in turn on
    new contents with eager calls between, equal eager calls. The counts change as well."""
    E, R, K, N = 6, 90, 256, 320
    stream = torch.cuda.Stream(DEV)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        cut = sorted(int(v) for v in torch.randint(0, R - 5, (E - 1,), generator=g))
        counts = [b - a for a, b in zip([0] + cut, cut + [R - 5])]
        return [_whole((R, K), BF16, seed), _whole((E, N, K), BF16, seed + 1), _counts(counts),
                _whole((R, N), BF16, seed + 2, most=1)]

    def step(x, w, c, dy):
        y = products.grouped_mm(x, w, c)
        dx, dw = products.grouped_mm(dy, w, c, transposed=True), products.grouped_mm_wgrad(dy, x, c)
        q, s = products.quantize_rows_int8(x)
        ones = torch.ones((E, N), device=DEV)
        return y, dx, dw, products.grouped_int8_mm(q, s, w.char(), ones, c), products.int8_mm(q, s, w[0].char(), ones[0])

    graphs = []
    for i in range(2):
        static = inputs(60 + 10 * i)
        with torch.cuda.stream(stream):
            step(*static)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(*static)
        graphs.append((graph, static, out))
    for turn in range(4):
        for i, (graph, static, out) in enumerate(graphs):
            fresh = inputs(100 + 20 * turn + 5 * i)
            for s, f in zip(static, fresh):
                s.copy_(f)
            want = step(*fresh)
            graph.replay()
            torch.cuda.synchronize()
            for k, (a, b) in enumerate(zip(out, want)):
                assert torch.equal(a, b), f"turn {turn} graph {i} output {k}"


def test_captured_training_step():
    """Forward and backward through autograd inside a graph, from leaves made inside it, while an
    eager graph of the weights lives."""
    counts = _counts([20, 0, 44])
    x, w = _whole((64, 128), BF16, 70), _whole((3, 192, 128), BF16, 71)
    dy = _whole((64, 192), BF16, 72, most=1)
    alive = products.grouped_mm(x.clone(), w.requires_grad_(), counts)
    stream = torch.cuda.Stream(DEV)

    def step():
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = products.grouped_mm(a, b, counts)
        return (y.detach(), *torch.autograd.grad(y, (a, b), dy))

    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for turn in range(3):
        x.copy_(_whole((64, 128), BF16, 80 + turn))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    _same(torch.autograd.grad(alive.sum(), w)[0],
          _wgrad(torch.ones_like(dy), _whole((64, 128), BF16, 70), [20, 0, 44]), "the eager graph's gradient")


def test_same_inputs_same_bits():
    g = torch.Generator(device=DEV).manual_seed(73)
    counts = _counts([200, 3, 0, 61])
    x, w = torch.randn((264, 1024), generator=g, device=DEV).to(BF16), torch.randn((4, 512, 1024), generator=g, device=DEV).to(BF16)
    dy = torch.randn((264, 512), generator=g, device=DEV).to(BF16)
    first = (products.grouped_mm(x, w, counts), products.grouped_mm_wgrad(dy, x, counts))
    for _ in range(5):
        assert torch.equal(first[0], products.grouped_mm(x, w, counts))
        assert torch.equal(first[1], products.grouped_mm_wgrad(dy, x, counts))


def _routed(T, E, K, seed):
    """The framework's own routing of T tokens, and the rows in expert order."""
    case = C.Case.from_dict({**C.case("moe-fp8-tiny-t4").to_dict(), "id": "products",
                             "params": dict(tokens=T, hidden=256, experts=E, topk=K, intermediate=256)})
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = torch.randn((T, E), generator=g, device=DEV)
    ids, weights = submission.route(case, logits, None)
    order = ids.flatten().argsort(stable=True)
    return ids, weights, order, torch.bincount(ids.flatten(), minlength=E)


def test_bf16_experts_step_by_step():
    """Route, gather, gate/up, SwiGLU, down and the weighted sum, forward and backward, against
    the same step in 64 bits. Rounding: every one of the chain's five bf16 results (gate/up, h,
    down and the two gradients on the way back) is off by half a step, 2^-9 of its value; h and
    the products mix at most four of them into one number, whose errors add like independent ones
    over the sums: 8 * 2^-9 of the norm holds for the chain."""
    T, E, K, H, I = 60, 8, 2, 256, 192
    ids, weights, order, counts = _routed(T, E, K, 90)
    g = torch.Generator(device=DEV).manual_seed(91)
    x = torch.randn((T, H), generator=g, device=DEV).to(BF16).requires_grad_()
    w1 = (torch.randn((E, 2 * I, H), generator=g, device=DEV) * 0.06).to(BF16).requires_grad_()
    w2 = (torch.randn((E, H, I), generator=g, device=DEV) * 0.07).to(BF16).requires_grad_()
    dy = torch.randn((T, H), generator=g, device=DEV)

    def step(x, w1, w2, product):
        gate, up = product(x[order // K], w1).chunk(2, dim=1)
        down = product((torch.nn.functional.silu(gate) * up).contiguous(), w2)
        slots = torch.zeros_like(down).index_copy(0, order, down)
        return (slots.view(T, K, H).to(weights.dtype if down.dtype == BF16 else down.dtype) * weights[..., None]).sum(1)

    def plain(a, b):
        rows, first = [], 0
        for e, c in enumerate(counts.tolist()):
            rows.append(a[first:first + c] @ b[e].T)
            first += c
        return torch.cat(rows)

    y = step(x, w1, w2, lambda a, b: products.grouped_mm(a, b, counts))
    grads = torch.autograd.grad(y, (x, w1, w2), dy)
    leaves = [t.detach().double().requires_grad_() for t in (x, w1, w2)]
    z = step(*leaves, plain)
    for name, a, b in zip(("y", "dx", "dw1", "dw2"), (y, *grads), (z, *torch.autograd.grad(z, leaves, dy.double()))):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        _log(f"{name}: {rel:.2e}")
        assert rel <= 8 * 2.0**-9, name


def test_int8_experts_step_by_step():
    """Quantize, gate/up, SwiGLU, quantize, down and GPT-OSS's combine by expert id, against the
    same step with exact integer sums in 64 bits on the CPU from the same int8 weights."""
    T, E, K, H, I = 33, 8, 2, 256, 384
    ids, weights, order, counts = _routed(T, E, K, 95)
    g = torch.Generator(device=DEV).manual_seed(96)
    x = torch.randn((T, H), generator=g, device=DEV).to(BF16)
    w1, s1 = zip(*(products.quantize_rows_int8(torch.randn((2 * I, H), generator=g, device=DEV) * 0.06) for _ in range(E)))
    w2, s2 = zip(*(products.quantize_rows_int8(torch.randn((H, I), generator=g, device=DEV) * 0.05) for _ in range(E)))
    w1, s1, w2, s2 = (torch.stack(t) for t in (w1, s1, w2, s2))
    q, s = products.quantize_rows_int8(x)
    gate, up = products.grouped_int8_mm(q[order // K], s[order // K], w1, s1, counts).chunk(2, dim=1)
    h = torch.nn.functional.silu(gate) * up
    hq, hs = products.quantize_rows_int8(h)
    down = products.grouped_int8_mm(hq, hs, w2, s2, counts)
    slots = torch.empty_like(down).index_copy_(0, order, down).view(T, K, H)
    y = submission.combine_by_expert_id(slots, ids, weights.to(BF16))

    def plain(a, sa, b, sb):
        rows, first = [], 0
        a, sa, b, sb = a.cpu().long(), sa.cpu(), b.cpu().long(), sb.cpu()
        for e, c in enumerate(counts.tolist()):
            rows.append((a[first:first + c] @ b[e].T).float() * sa[first:first + c, None] * sb[e])
            first += c
        return torch.cat(rows).to(BF16)

    xq, xs = _quantized(x)
    o = (order // K).cpu()
    want = plain(xq[o], xs[o], w1, s1)
    assert torch.equal(torch.cat((gate, up), 1).cpu(), want)
    wq, wsc = _quantized(h)
    assert torch.equal(hq.cpu(), wq) and torch.equal(hs.cpu(), wsc)
    assert torch.equal(down.cpu(), plain(wq, wsc, w2, s2))
    assert y.shape == (T, H) and bool(y.isfinite().all())
