"""examples/decode_fp8.py: its 8-bit rounding on the CPU, and a small run of it on the GPU."""

import importlib.util
import os

import numpy as np
import pytest

import serving_plain as plain


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_fp8.py")
    spec = importlib.util.spec_from_file_location("decode_fp8", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_e4m3(example):
    """Every number, every halfway value and what lies around it, as the tests' own rounding has them."""
    numbers = plain.F8[:127]
    halfway = (numbers[:-1] + numbers[1:]) / 2
    x = np.concatenate([numbers, halfway, halfway * (1 + 2.0 ** -12), halfway * (1 - 2.0 ** -12), np.linspace(0, 448, 4001)]).astype(np.float32)
    x = np.concatenate([x, -x])
    assert np.array_equal(example.e4m3(x), plain.f8_bits(x))


@pytest.mark.parametrize("n,k", [(128, 128), (130, 300), (1, 1), (257, 64)])
def test_block_scaled(example, n, k):
    rng = np.random.default_rng(n)
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[:, :1] = 0 if k == 1 else w[:, :1]
    q, s = example.block_scaled(w)
    assert q.shape == (n, k) and s.shape == (-(-n // 128), -(-k // 128)) and (s > 0).all()
    step = np.repeat(np.repeat(s, 128, 0), 128, 1)[:n, :k].astype(np.float64)
    got = plain.F8[q] * step
    assert (np.abs(got - w) <= np.maximum(2.0 ** -4 * np.abs(w), 2.0 ** -10 * step) * (1 + 1e-6)).all()


def test_refuses_what_does_not_fit(example):
    with pytest.raises(SystemExit):
        example.main(["--prompt", "10", "--steps", "10", "--context", "19"])


@pytest.mark.gpu
@pytest.mark.parametrize("argv", [
    ["--layers", "2", "--hidden", "256", "--heads", "4", "--kv-heads", "2", "--head-dim", "64", "--ffn", "384", "--vocabulary", "320",
     "--batch", "3", "--prompt", "21", "--steps", "20", "--context", "64", "--page", "8"],
    ["--layers", "1", "--hidden", "320", "--heads", "6", "--kv-heads", "1", "--head-dim", "32", "--ffn", "200", "--vocabulary", "130",
     "--batch", "1", "--prompt", "1", "--steps", "4", "--context", "40", "--page", "16"],
])
def test_decodes(example, argv):
    """Steps replayed as a graph give the logits that the same tokens give as one prompt, to the noise of the roundings."""
    print("decode", argv, flush=True)
    result = example.main(argv)
    assert result["finite"] and result["difference"] < example.AGREES
