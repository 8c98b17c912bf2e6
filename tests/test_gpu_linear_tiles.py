"""Every kernel of the 8-bit linear layers by name, as profiling reports it, so
that a change of the rule that chooses them cannot leave one without a test;
the tiles with more steps than they keep in flight.  Definition and tolerance:
test_gpu_linear.py."""
import pytest

from test_gpu_kvcache import kernels_of
from test_gpu_linear import BF, F16, F32, check, expected, gen, layer_of, normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("kernel,tokens,inputs,outputs", [
    ("int8_token", 1, 700, 300), ("int8_token", 12, 1000, 1001),
    ("int8_token", 9, 2048, 65), ("int8_few", 9, 2049, 65), ("int8_few", 32, 5000, 520),
    ("int8_few64", 33, 3000, 8192), ("int8_few64", 64, 1030, 8190),
    # eight steps in flight: fewer, as many, more, several times as many
    ("int8_tile64", 40, 64, 8300), ("int8_tile64", 600, 500, 704), ("int8_tile64", 600, 1000, 700),
    ("int8_tile64", 40, 2000, 8300), ("int8_tile64", 777, 1000, 1777),
    ("int8_tile128_ahead", 4000, 320, 1000), ("int8_tile128_ahead", 1500, 449, 1600),
    ("int8_tile128_ahead", 1500, 1100, 1501), ("int8_tile128_ahead", 1700, 1990, 1536),
    # four
    ("int8_tile128", 4099, 64, 4001), ("int8_tile128", 2100, 256, 2104),
    ("int8_tile128", 2100, 1000, 2100), ("int8_tile128", 100, 1500, 44001),
    # four; tiles of 256, wide and odd outputs, tokens at a tile's ends
    ("int8_tile256", 1000, 1100, 11003), ("int8_tile256", 2100, 2048, 5003),
    ("int8_tile256", 2049, 1025, 5120), ("int8_tile256", 129, 3000, 43521),
    ("int8_tile256", 256, 1088, 44032)])
def test_kernels(ctx, dtype, kernel, tokens, inputs, outputs):
    g = gen(tokens + outputs)
    layer, codes, scales, b = layer_of(ctx, g, outputs, inputs, bias=outputs % 2 == 1)
    x = normal(g, tokens, inputs, dtype=dtype)
    out, used = kernels_of(ctx, lambda: layer(x))
    assert used == ({kernel} if kernel == "int8_token" else {kernel, "int8_quantize"})
    check(out, *expected(x, codes, scales, b, dtype))
