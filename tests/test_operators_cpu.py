"""Windowed attention, rotation on several axes and compaction on the CPU
(tests/cpp/operator_tests.cc): the window's arithmetic, the fixed-point turns, the runs
moves are cut into and what the entry points refuse; and the binding's own checks."""
import os
import subprocess
import warnings

import numpy as np
import pytest

from chibillm_amd import ckv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_operators_cpp():
    path = os.path.join(ROOT, "chibillm_amd", "bin", "operator_tests")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built: run __graft_entry__.build()")
    proc = subprocess.run([path], capture_output=True, text=True, timeout=120)
    print(proc.stdout[-4000:])
    assert proc.returncode == 0, proc.stdout[-4000:] + proc.stderr[-2000:]
    assert " 0 failed checks" in proc.stdout


@pytest.mark.parametrize("sections", [[32], [8, 12, 12], [24, 20, 20], [11, 11, 10], [5, 3]])
def test_rope_pair_axes(sections):
    apart, mixed = ckv.rope_pair_axes(sections), ckv.rope_pair_axes(sections, interleaved=True)
    assert apart.dtype == mixed.dtype == np.uint8 and apart.size == mixed.size == sum(sections)
    assert apart.tolist() == sorted(apart.tolist())
    for axis, pairs in enumerate(sections):
        assert (apart == axis).sum() == pairs
        if axis:
            assert np.flatnonzero(mixed == axis).tolist() == [
                j for j in range(sum(sections)) if j % len(sections) == axis and j < pairs * len(sections)]


@pytest.mark.parametrize("sections,turned", [([8, 12, 12], [11, 11, 10]), ([4, 20], [12, 12]), ([20, 20, 4], [25, 15, 4])])
def test_interleaved_sections_that_do_not_fit_are_told(sections, turned):
    with pytest.warns(UserWarning, match=r"turn \[{}\] pairs".format(", ".join(map(str, turned)))):
        axes = ckv.rope_pair_axes(sections, interleaved=True)
    assert np.bincount(axes).tolist() == turned


@pytest.mark.parametrize("sections", [[32], [24, 20, 20], [11, 11, 10], [5, 3], [2, 1, 1, 1], [5, 0, 2]])
def test_interleaved_sections_turn_what_they_say(sections):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        axes = ckv.rope_pair_axes(sections, interleaved=True)
        ckv.rope_pair_axes([8, 12, 12])  # one after another any sections do
    assert np.bincount(axes, minlength=len(sections)).tolist() == sections


class _Stub:
    """A pool that never reaches the library."""
    geometry = (1, 4, 16, 2, 128)
    upload_axes, rope_axes, compact = ckv.Pool.upload_axes, ckv.Pool.rope_axes, ckv.Pool.compact
    _pair_axis = ckv.Pool._pair_axis


def test_binding_refuses_arrays_of_other_sizes():
    pool, rows = _Stub(), np.zeros((2, 256))
    with pytest.raises(ValueError):
        pool.upload_axes([1, 2, 3])
    with pytest.raises(ValueError):
        pool.rope_axes(rows, rows, 2, 1e4, [0] * 63)
    with pytest.raises(ValueError):
        pool.rope_axes(rows, rows, 2, 1e4, [0] * 64, rotary_dim=64)
    for moves in (([1, 2], [3], [2], None), ([1, 2], [3, 4], [1], None), ([1, 2], [3, 4], [2], [0])):
        with pytest.raises(ValueError):
            pool.compact(*moves)


def test_binding_refuses_numbers_that_wrap():
    """Slots, shifts, positions and axes that 32 or 8 bits do not hold, and negative windows and sinks
    (size_t to the library), would be other numbers there."""
    pool, rows = _Stub(), np.zeros((2, 256))
    with pytest.raises(ValueError):
        pool.upload_axes(np.array([[1, -1]]))
    with pytest.raises(ValueError):
        pool.upload_axes(np.array([[1, 2 ** 32]]))
    for axis in (-1, 256, 257):
        with pytest.raises(ValueError):
            pool.rope_axes(rows, rows, 2, 1e4, [axis] * 64)
    for moves in (([2 ** 32 + 5], [3], [1], None), ([5], [-3], [1], None), ([5], [3], [1], [2 ** 31]), ([5], [3], [1], [0.5])):
        with pytest.raises(ValueError):
            pool.compact(*moves)
    for window, sinks in ((-1, 0), (8, -1)):
        for call in (lambda: ckv.Pool.attention_window(pool, 0, rows, 2, 1.0, window, rows, sinks=sinks),
                     lambda: ckv.Pool.append_decode_window(pool, 0, rows, rows, rows, 2, 1.0, window, rows, sinks=sinks),
                     lambda: ckv.Pool.rope_append_decode_window(pool, 0, rows, rows, rows, 2, 1.0, 1e4, window, rows, sinks=sinks)):
            with pytest.raises(ValueError, match="counts of tokens"):
                call()
