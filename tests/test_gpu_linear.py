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
import ctypes
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


def layer_of(ctx, g, outputs, inputs, bias=True):
    """A layer of given codes, its codes, scales and bias."""
    from vectorstorekit_amd import Int8Linear

    codes = torch.randint(-127, 128, (outputs, inputs), generator=g, dtype=torch.int8).to(DEV)
    scales = torch.rand(outputs, generator=g).to(DEV)
    b = normal(g, outputs) if bias else None
    return Int8Linear.over(ctx, codes, scales, b), codes, scales, b


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens,inputs,outputs", [
    # few tokens, a workgroup for 32 channels; two blocks of tokens
    (32, 1000, 65), (17, 5000, 33), (63, 1000, 500),
    # tiles of 64, also where few tokens have many channels
    (40, 64, 8300), (100, 700, 1000),
    # tiles of 128 with many steps in flight and with few; of few tokens
    (1500, 72, 1501), (2100, 200, 2100), (100, 64, 44001),
    # tiles of 256
    (1000, 64, 11003)])
def test_every_tile(ctx, dtype, tokens, inputs, outputs):
    g = gen(tokens + outputs)
    layer, codes, scales, b = layer_of(ctx, g, outputs, inputs)
    x = normal(g, tokens, inputs, dtype=dtype)
    check(layer(x), *expected(x, codes, scales, b, dtype))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("tokens,inputs,outputs", [
    # rows longer than the registers of a wave or a workgroup hold
    (2050, 16400, 33), (5, 40000, 33), (1, 131072, 40), (3, 131071, 1), (40, 33000, 64),
    # a long row for one launch, a place more than it takes
    (1, 16384, 40), (1, 16385, 40)])
def test_long_rows(ctx, dtype, tokens, inputs, outputs):
    g = gen(inputs)
    layer, codes, scales, b = layer_of(ctx, g, outputs, inputs)
    x = normal(g, tokens, inputs, dtype=dtype)
    check(layer(x), *expected(x, codes, scales, b, dtype))


def test_largest_sums(ctx):
    """The largest sums that the inputs allow, of both signs, are exact."""
    from vectorstorekit_amd import Int8Linear

    codes = torch.full((2, 131072), -128, dtype=torch.int8, device=DEV)
    codes[1] = 127
    layer = Int8Linear.over(ctx, codes, torch.ones(2, device=DEV))
    x = torch.full((40, 131072), -127.0, device=DEV)
    x[1::2] = 127.0
    for n in (1, 2, 40):
        got = layer(x[:n])
        assert got[0].tolist() == [127.0 * 128 * 131072, -127.0 * 127 * 131072]
        if n > 1:
            assert got[1].tolist() == [-127.0 * 128 * 131072, 127.0 * 127 * 131072]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("tokens,inputs,outputs", [
    (4, 4096, 100), (5, 3000, 100), (8, 2048, 97), (8, 2049, 97), (9, 2048, 64), (12, 1000, 1000),
    (64, 300, 2048), (64, 300, 2049), (65, 300, 1000), (511, 100, 100), (2, 100, 20000)])
def test_few_tokens(ctx, dtype, tokens, inputs, outputs):
    """Groups of tokens that one launch quantises and multiplies, and the sizes
    from which on two do."""
    g = gen(inputs + tokens)
    layer, codes, scales, b = layer_of(ctx, g, outputs, inputs)
    x = normal(g, tokens, inputs, dtype=dtype)
    check(layer(x), *expected(x, codes, scales, b, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("tokens", [8, 40, 2100])
def test_extreme_rows(ctx, dtype, tokens):
    """Rows of zeros, infinities, NaN, the smallest and the largest numbers
    leave the other rows as they are; such channels as well."""
    from vectorstorekit_amd import Int8Linear

    g = gen(tokens)
    x = normal(g, tokens, 130, dtype=dtype)
    x[0], x[1, 7], x[2, 129], x[3, 0] = 0.0, math.inf, math.nan, -math.inf
    x[4] *= 2.0 ** -117
    x[5] = x[5].clamp(-3, 3) * 2.0 ** 126
    x[6] *= 2.0 ** -134
    w = normal(g, 70, 130) * 1e-3
    w[3], w[4, 5], w[5, 129] = 0.0, math.nan, math.inf
    layer = Int8Linear(ctx, w)
    codes, scales = quantised(w)
    assert torch.equal(layer.codes().cpu().double(), codes)
    assert torch.equal(layer.scales.cpu().double().nan_to_num(-1.0), scales.nan_to_num(-1.0))
    for out in (dtype, F32):
        y, tol = expected(x, codes, scales, None, out)
        assert torch.isnan(y[1:4]).all() and torch.isnan(y[:, 4:6]).all()
        got = layer(x, dtype=out)
        assert torch.isnan(got[1:4]).all() and torch.isnan(got[:, 4:6]).all()
        # (a bf16 result under 2^-126 is off by 2^-134 at most)
        check(got, y, tol + (2.0 ** -134 if out == BF else 0.0))
        assert (got[0, :4] == 0).all() and (got[6:, 3] == 0).all()


@pytest.mark.parametrize("tokens", [5, 50, 2200])
def test_layouts(ctx, tokens):
    """Views, strides and alignments give what dense rows give."""
    from vectorstorekit_amd import Int8Linear

    g = gen(tokens)
    w = normal(g, 64, 90, dtype=BF)
    bias = normal(g, 64, dtype=F16)
    layer = Int8Linear(ctx, w, bias)
    assert torch.equal(layer.codes(), Int8Linear(ctx, w.T.contiguous().T).codes())
    assert torch.equal(layer.codes(), Int8Linear(ctx, normal(gen(1), 64, 99, dtype=BF)[:, 3:93]
                                                 .copy_(w)).codes())
    codes = layer.codes()
    assert torch.equal(codes, Int8Linear.over(ctx, codes.T.contiguous().T,
                                              layer.scales.repeat(2)[::2]).codes())
    x = normal(g, tokens, 90, dtype=BF)
    want = layer(x)
    assert torch.equal(layer(x), want)
    check(want, *expected(x, codes, layer.scales, bias, BF))
    wide = normal(g, tokens, 107, dtype=BF)
    for at in (0, 1, 8):
        wide[:, at:at + 90] = x
        assert torch.equal(layer(wide[:, at:at + 90]), want)
    assert torch.equal(layer(x.T.contiguous().T), want)
    assert torch.equal(layer(x[:, None].expand(-1, 3, -1)), want[:, None].expand(-1, 3, -1))
    assert torch.equal(layer(x[:1].expand(tokens, -1)), layer(x[:1]).expand(tokens, -1))
    assert torch.equal(layer(x.view(1, tokens, 1, 90)), want.view(1, tokens, 1, 64))
    assert torch.equal(layer(x[3]), want[3])
    assert layer(x[:0]).shape == (0, 64) and layer(x[:0], dtype=F32).dtype == F32
    assert layer(x.view(tokens, 1, 90)[:, :0]).shape == (tokens, 0, 64)


def test_rows_behind_are_left(ctx):
    """The C call writes the tokens' outputs and nothing beside or behind."""
    from vectorstorekit_amd import _lib

    g = gen(5)
    for tokens, outputs in ((3, 33), (20, 33), (70, 100), (1500, 1501), (1000, 11003)):
        layer, *_ = layer_of(ctx, g, outputs, 64)
        x = normal(g, tokens, 64, dtype=BF)
        out = torch.full((tokens + 70, outputs + 9), 7.0, dtype=F32, device=DEV)
        need = ctx.lib.vsk_int8_linear_workspace(layer._ref, tokens)
        work = torch.empty(need + 256, dtype=torch.uint8, device=DEV).fill_(77)
        rows = _lib.vsk_int8_rows(x.data_ptr(), out.data_ptr(), 64, outputs + 9, tokens,
                                  work.data_ptr(), need, 2, 0)
        stream = torch.cuda.current_stream().cuda_stream
        assert ctx.lib.vsk_int8_linear(ctx.handle, stream, layer._ref,
                                       ctypes.byref(rows)) == 0
        assert torch.equal(out[:tokens, :outputs], layer(x, dtype=F32))
        assert (out[tokens:] == 7).all() and (out[:, outputs:] == 7).all()
        assert (work[need:] == 77).all()


@pytest.mark.parametrize("tokens,inputs", [(3, 300), (20, 3000), (300, 300), (2500, 300)])
def test_graph_and_stream(ctx, tokens, inputs):
    """Replays over changed inputs with other work between; two streams at once."""
    g = gen(tokens)
    layer, codes, scales, b = layer_of(ctx, g, 640, inputs)
    x = normal(g, tokens, inputs, dtype=BF)
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(layer(x)[:, :inputs] if inputs <= 640 else x)
    for step in range(4):
        x.copy_(normal(g, tokens, inputs, dtype=BF))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        want = layer(layer(x)[:, :inputs] if inputs <= 640 else x)
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [layer(x) for _ in range(3)]
    here = [layer(x) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, here[0]) for y in there + here)
    check(here[0], *expected(x, codes, scales, b, BF))


@pytest.mark.parametrize("tokens,inputs,outputs", [(70001, 64, 32768), (20001, 131072, 40)])
def test_past_32_bits(ctx, tokens, inputs, outputs):
    """More than 2^31 outputs, inputs and packed bytes: the last tokens' outputs
    are what they are by themselves."""
    g = gen(tokens)
    layer, codes, scales, b = layer_of(ctx, g, outputs, inputs)
    tail = normal(g, 50, inputs, dtype=BF)
    x = torch.zeros(tokens, inputs, dtype=BF, device=DEV)
    x[-50:] = tail
    got = layer(x)
    assert torch.equal(got[-50:], layer(tail))
    assert torch.equal(got[0], b.to(BF)) and torch.equal(got[-51], b.to(BF))
    check(got[-3:], *expected(tail[-3:], codes, scales, b, BF))


def test_refusals(ctx):
    from vectorstorekit_amd import Int8Linear, VSKError

    g = gen(6)
    w, x = normal(g, 20, 30, dtype=BF), normal(g, 4, 30, dtype=BF)
    layer = Int8Linear(ctx, w)
    codes, scales = layer.codes(), layer.scales
    bad = [
        lambda: layer(x.cpu()), lambda: layer(x.double()), lambda: layer(x[:, :29]),
        lambda: layer(x, dtype=torch.float64), lambda: layer(x[0, 0]), lambda: layer([1.0] * 30),
        lambda: layer(x.clone().requires_grad_()),
        lambda: Int8Linear(ctx, w.cpu()), lambda: Int8Linear(ctx, w.double()),
        lambda: Int8Linear(ctx, w[0]), lambda: Int8Linear(ctx, w[:0]),
        lambda: Int8Linear(ctx, w[:, :0]), lambda: Int8Linear(ctx, w, scales[:19]),
        lambda: Int8Linear(ctx, w, scales.cpu()), lambda: Int8Linear(ctx, w, scales.double()),
        lambda: Int8Linear(ctx, w, scales[:, None]),
        lambda: Int8Linear(ctx, torch.nn.Parameter(w)),
        lambda: Int8Linear(ctx, torch.zeros(1, 131073, dtype=BF, device=DEV)),
        lambda: Int8Linear.over(ctx, codes.float(), scales),
        lambda: Int8Linear.over(ctx, codes, scales[:19]),
        lambda: Int8Linear.over(ctx, codes, scales.half()),
        lambda: Int8Linear.over(ctx, codes, scales[:, None]),
        lambda: Int8Linear.over(ctx, codes.cpu(), scales),
        lambda: Int8Linear.over(ctx, codes, scales, scales[:5]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(VSKError):
            call()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        assert torch.equal(Int8Linear(ctx, torch.nn.Parameter(w))(x.requires_grad_()), layer(x))


def test_c_refusals(ctx):
    """The C calls' own checks (of what Python checks before)."""
    from vectorstorekit_amd import _lib

    g = gen(7)
    layer, *_ = layer_of(ctx, g, 5000, 64)
    x, out = normal(g, 100, 64, dtype=BF), torch.zeros(100, 5000, dtype=BF, device=DEV)
    lib, h = ctx.lib, ctx.handle
    need = lib.vsk_int8_linear_workspace(layer._ref, 100)
    work = torch.empty(need, dtype=torch.uint8, device=DEV)
    fine = _lib.vsk_int8_rows(x.data_ptr(), out.data_ptr(), 64, 5000, 100, work.data_ptr(), need,
                              2, 2)
    ref = lambda c: ctypes.byref(c) if isinstance(c, ctypes.Structure) else c
    call = lambda w, r: lib.vsk_int8_linear(h, None, ref(w), ref(r))
    changed = lambda c, **k: [setattr(c, *x) for x in k.items()] and c
    copy = lambda: _lib.vsk_int8_rows.from_buffer_copy(fine)
    weight = lambda: _lib.vsk_int8_weight.from_buffer_copy(layer._weight)
    there = torch.zeros(10)
    host = there.data_ptr()
    assert need > 0
    assert call(None, fine) == -2 and call(layer._ref, None) == -2
    for fields, status in (({"x_dtype": 3}, -8), ({"out_dtype": -1}, -8), ({"tokens": -1}, -2),
                           ({"tokens": 1 << 31}, -9), ({"x": 0}, -2), ({"out": 0}, -2),
                           ({"x": host}, -2), ({"out": host}, -2), ({"workspace": 0}, -9),
                           ({"workspace_bytes": need - 1}, -9), ({"workspace": host}, -9),
                           ({"workspace": work.data_ptr() + 8}, -9)):
        assert call(layer._ref, changed(copy(), **fields)) == status, fields
    for fields, status in (({"outputs": 0}, -3), ({"inputs": 0}, -3), ({"inputs": 131073}, -9),
                           ({"packed": 0}, -2), ({"scales": 0}, -2), ({"scales": host}, -2),
                           ({"bias": host}, -2), ({"packed": layer.packed.data_ptr() + 4}, -2)):
        assert call(changed(weight(), **fields), fine) == status, fields
    pack = lambda t, rows, w: lib.vsk_int8_pack(h, None, t, rows, 64, ref(w))
    assert pack(4, x.data_ptr(), layer._ref) == -8 and pack(2, None, layer._ref) == -2
    assert pack(2, host, layer._ref) == -2 and pack(2, x.data_ptr(), None) == -2
    assert call(layer._ref, changed(copy(), tokens=0, x=0, out=0)) == 0
    assert call(layer._ref, fine) == 0
    assert torch.equal(out, layer(x))
