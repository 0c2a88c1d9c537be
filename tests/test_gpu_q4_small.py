"""GPU: products with 4-bit weights of the smallest values, held to what f32 itself loses there, and
after a refused call."""
import numpy as np
import pytest

from m1moe_amd import M1MoEError

from cases import rel_l2, say
from draft_cases import q4_dense, q4_weights
from serving_cases import as_dtype, f64
from test_gpu_drafts import Product, dev, product  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 6, 12, 20, 50])
@pytest.mark.parametrize("x_dtype", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-90, -110, -113, -118, -120, -124])
def test_q4_of_the_smallest_values(dev, tokens, x_dtype, power):  # noqa: F811
    """Rows around 2^-112, below which a row is no longer brought to 2^14: held to what f32 itself
    loses there, a few steps of 2^-149 per sum, and in the 2-norm of each row."""
    rng = np.random.default_rng(tokens)
    w, s, b = q4_weights(rng, 70, 640, 64)
    x = as_dtype(rng.normal(0, 1, (tokens, 640)) * 2.0 ** power, x_dtype)
    say(f"q4 values of 2^{power} {x_dtype}, {tokens} tokens")
    y = product(dev, x, w, s, b, 64, x_dtype)
    dense, size = q4_dense(w, s, b, 64)
    x = f64(x)
    ref = x @ dense.T
    # (as q4_bound; f16 parts end at steps of 2^-24 of x times at most 2^126: half a step is 2^-151.
    # Units of columns, their sums over waves and workgroups and the result: 8 roundings of 2^-150)
    mag, top = np.abs(x) @ size.T, np.abs(x).max(1, keepdims=True)
    bound = mag * (2.0 ** -22 + (2 * 64 + 10 + 8) * 2.0 ** -23) + np.abs(ref) * 2.0 ** -22
    bound += np.maximum(top * 2.0 ** -39, 2.0 ** -151) * size.sum(1)[None] + 8 * 2.0 ** -150
    assert np.max(np.abs(y - ref) / bound) <= 1.0
    # (independent roundings, as test_q4 has it: 2e-6 of the products' size in the 2-norm; and the
    # steps above)
    for t in range(tokens):
        norm = np.linalg.norm(x[t]) * np.linalg.norm(dense)
        assert np.linalg.norm(y[t] - ref[t]) < 2e-6 * norm + np.sqrt(70) * (2.0 ** -151 * size.sum(1).max() + 8 * 2.0 ** -150)
        if power >= -120:
            assert rel_l2(y[t], ref[t]) < 1e-4


def test_q4_refuses_nothing_after_an_error(dev):  # noqa: F811
    """A refused call leaves the workspace usable."""
    ctx, ops = dev
    p = Product(dev, 40, 96, 512)
    p()
    want = p.result()
    with pytest.raises(M1MoEError):
        ops.matmul_q4(p.weights, p.held[3], "f32", 500, 40, p.held[4], "f32", 96)
    p()
    assert np.array_equal(p.result(), want)
    p.free()
