"""Scaled rotations, whole prompts and 4-bit pools on the CPU (tests/cpp/rotation_tests.cc): what
the entry points refuse and how tiles are listed; and the binding's own checks."""
import os
import subprocess

import numpy as np
import pytest
import torch

from chibillm_amd import ckv
from tests import fp4_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rotations_cpp():
    path = os.path.join(ROOT, "chibillm_amd", "bin", "rotation_tests")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built: run __graft_entry__.build()")
    proc = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(proc.stdout[-4000:])
    assert proc.returncode == 0, proc.stdout[-4000:] + proc.stderr[-2000:]
    assert " 0 failed checks" in proc.stdout


def test_binding_refuses_rotations_and_rows_it_cannot_pass():
    for width in (-1, 2 ** 32):
        with pytest.raises(ValueError):
            ckv.Rotation(1e4, width)
        with pytest.raises(ValueError):
            ckv.Rotation(1e4, 64, "halves", "yarn", 4.0, original=width)
    with pytest.raises(KeyError):
        ckv.Rotation(1e4, layout="thirds")
    with pytest.raises(KeyError):
        ckv.Rotation(1e4, scaling="cubic")
    pool, x = object.__new__(ckv.Pool), torch.zeros(4, 128)
    with pytest.raises(ValueError, match="GPU"):
        pool.prompt_attention(x, x, x, 1, 1.0, x)
    pool.handle = None


class OnDevice:
    """A tensor that says it is on a GPU; its memory is never read."""

    def __init__(self, x):
        self.x, self.is_cuda, self.shape = x, True, x.shape

    def dim(self):
        return self.x.dim()

    def stride(self, i):
        return self.x.stride(i)

    def data_ptr(self):
        return self.x.data_ptr()


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("make,said", [
    (lambda n: torch.zeros(1, n).expand(4, -1), "overlap"),            # one row, four times
    (lambda n: torch.zeros(4 * n).as_strided((4, n), (n - 1, 1)), "overlap"),
    (lambda n: torch.zeros(4, 2 * n)[:, :n - 8], "are needed"),        # part of a row
    (lambda n: torch.zeros(4, n + 8), "are needed"),
    (lambda n: torch.zeros(3, n), "are needed"),                       # a row too few
    (lambda n: torch.zeros(4, 1, n), "side by side"),
])
def test_prompt_rows_that_would_be_read_past_their_end(which, make, said):
    """Of a pool of 2 KV heads of 64 and 4 query heads, four rows."""
    pool = object.__new__(ckv.Pool)
    pool.geometry = (1, 1, 16, 2, 64)
    rows = [torch.zeros(4, 256), torch.zeros(4, 128), torch.zeros(4, 128)]
    rows[which] = make(rows[which].shape[1])
    with pytest.raises(ValueError, match=said):
        pool.prompt_attention(*map(OnDevice, rows), 4, 1.0, None, rows=4)
    pool.handle = None


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_the_reference_holds_what_the_levels_say(dtype):
    """The oracle of the device tests against a search through all 16 numbers."""
    levels = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    rng = np.random.RandomState(5)
    rows = np.concatenate([rng.randn(20, 32), np.exp(rng.randn(20, 32) * 8), np.full((1, 32), 5.0),
                           np.linspace(-7.9, 7.9, 32)[None], np.zeros((1, 32)), rng.randint(-28, 29, (200, 32)) / 4.0])
    rows[0, 3] = 7.0
    got = ref.held(torch.from_numpy(rows), dtype).numpy()
    for x, h in zip(rows, got):
        m = np.abs(x).max()
        if dtype == "f16" and m >= 2.0 ** 16:  # past the type: the block is lost
            assert np.isnan(h).all()
            continue
        scale = 2.0 ** max(np.floor(np.log2(m)) - 2 if m else -1000, ref.LEAST[dtype])
        for a, b in zip(np.abs(x) / scale, np.abs(h) / scale):
            assert b in levels
            away = np.abs(levels - min(a, 6.0))
            assert np.abs(b - min(a, 6.0)) == away.min()
            if (away == away.min()).sum() == 2:  # between two: the even code
                assert list(levels).index(b) % 2 == 0
        assert np.array_equal(np.signbit(h), np.signbit(x))
