"""Windowed decode of batches that fill the GPU, against its definition: rows halved between two
workgroups, whole rows at 4 and 8 waves, wide groups and heads, and pieces of a few pages (the plans
and waves at these sizes are in the CPU tests "window plan" and "window decode")."""
import numpy as np
import pytest

from tests.gpu_util import new_context
from tests.test_gpu_window import decode_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = new_context()
    yield c
    c.sync()
    c.close()


def lengths(rows, low, high):
    return [int(x) for x in np.random.RandomState(rows).randint(low, high, rows)]


@pytest.mark.parametrize("dtype,heads,group,d,window,rows,high", [
    ("bf16", 8, 2, 128, 1024, 33, 1700),  # halves, 4 waves
    ("bf16", 8, 2, 128, 1024, 48, 1500),
    ("f16", 8, 1, 128, 600, 40, 1300),
    ("bf16", 8, 4, 128, 530, 40, 900),
    ("bf16", 8, 8, 128, 530, 36, 800),    # halves at 8 waves
    ("bf16", 8, 2, 128, 400, 52, 900),    # whole rows at 8 waves
    ("bf16", 8, 2, 128, 300, 64, 700),    # at 4
    ("f16", 8, 4, 128, 256, 80, 600),
    ("bf16", 8, 8, 128, 200, 64, 500),
    ("bf16", 8, 8, 128, 200, 80, 400),
    ("bf16", 8, 4, 256, 272, 40, 600),    # 256-wide halves
    ("f16", 2, 2, 256, 300, 150, 500),
    ("f32", 8, 2, 128, 300, 40, 700),
    ("f32", 2, 4, 256, 200, 150, 400),
    ("bf16", 8, 2, 128, 512, 4, 1900),    # pieces of four pages
    ("bf16", 8, 2, 128, 256, 1, 1200)])
def test_window_decode_of_a_batch(ctx, dtype, heads, group, d, window, rows, high):
    print(f"window decode {dtype} {heads} x {group} d {d} window {window} rows {rows}", flush=True)
    decode_case(ctx, dtype, heads, group, d, window, 4, lengths=lengths(rows, window, high), gated=rows % 2 == 0, seed=rows)
