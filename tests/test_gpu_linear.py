"""The 8-bit linear layer against its definition in 64 bits.

A token's codes and the sums are whole numbers and compared as such (the
quotients that are rounded to codes are 32-bit products by definition, which
64 bits hold exactly before they are rounded).  Tolerance of an output, derived
here: the sum is rounded to 32 bits, multiplied by two scales, each of which
was rounded once, and the bias added: five roundings of 2^-24 relative to the
product (the scale of the token, the conversion, two products, the sum, of
which the last is relative to the result), and one of the output's type:
|err| <= u |y| + 2^-24 (4 |s t sum| + |y|), with u 2^-8 (bf16), 2^-11 (f16) or
2^-24 (f32); an f16 result under 2^-14 is off by 2^-25 at most."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
DEV = "cuda:0"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, dtype=torch.float32).to(dtype).to(DEV)


def f32(x):
    """64-bit numbers rounded to 32 bits, as 64-bit numbers."""
    return x.to(torch.float32).double()


def quantised(x):
    """Codes (64-bit whole numbers) and scales of rows on the CPU."""
    x = x.detach().cpu().double()
    top = x.abs().amax(-1, keepdim=True)
    odd = ~torch.isfinite(top)
    t = torch.where(odd | (top == 0), 1.0, top)
    up = torch.where(t < 2.0 ** -100, 2.0 ** 100, 1.0)
    inverse = f32(127 / (t * up))
    codes = torch.round(f32(torch.where(odd, 0.0, x) * up * inverse))
    return codes, torch.where(odd, math.nan, f32(top / 127))[:, 0]


def expected(x, codes, scales, bias, dtype):
    c, s = quantised(x)
    product = (c @ codes.cpu().double().T) * s[:, None] * scales.cpu().double()
    y = product if bias is None else product + bias.cpu().double()
    tol = U[dtype] * y.abs() + 2.0 ** -24 * (4 * product.abs() + y.abs())
    return y, tol + (2.0 ** -25 if dtype == F16 else 2.0 ** -149)


def check(got, want, tol):
    got = got.detach().cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    err = (got - want).abs()[fine]
    assert bool((err <= tol[fine]).all()), float((err - tol[fine]).max())


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("tokens,inputs,outputs,bias", [
    (1, 1, 1, True), (1, 4096, 512, False), (3, 64, 33, True), (31, 100, 70, True),
    (32, 192, 64, False), (33, 96, 31, True), (64, 1000, 130, False), (65, 129, 257, True),
    (130, 320, 65, True), (200, 511, 1000, False), (1030, 256, 96, True), (1500, 72, 40, False),
    (257, 2048, 1026, True)])
def test_linear(ctx, dtype, tokens, inputs, outputs, bias):
    from vectorstorekit_amd import Int8Linear

    g = gen(tokens + inputs)
    w = normal(g, outputs, inputs, dtype=dtype)
    b = normal(g, outputs) if bias else None
    layer = Int8Linear(ctx, w, b)
    codes, scales = quantised(w)
    assert torch.equal(layer.codes().cpu().double(), codes)
    assert torch.equal(layer.scales.cpu().double(), scales)
    x = normal(g, tokens, inputs, dtype=dtype)
    check(layer(x), *expected(x, codes, scales, b, dtype))
    for out in (BF, F16, F32):
        if out != dtype and tokens < 100:
            check(layer(x, dtype=out), *expected(x, codes, scales, b, out))


@pytest.mark.parametrize("tokens,inputs,outputs", [(2048, 128, 8192), (2100, 200, 8200),
                                                   (4099, 64, 4001)])
def test_large_tiles(ctx, tokens, inputs, outputs):
    """Enough outputs that every size of tile is taken, edges among them."""
    from vectorstorekit_amd import Int8Linear

    g = gen(outputs)
    codes = torch.randint(-127, 128, (outputs, inputs), generator=g, dtype=torch.int8).to(DEV)
    scales, b = torch.rand(outputs, generator=g).to(DEV), normal(g, outputs)
    x = normal(g, tokens, inputs, dtype=BF)
    layer = Int8Linear.over(ctx, codes, scales, b)
    assert torch.equal(layer.codes(), codes)
    for out in (BF, F32):
        check(layer(x, dtype=out), *expected(x, codes, scales, b, out))
