"""Sampled ids of rows up to the longest, where many ids lie close to each other: equal weights, and a few above them.

Bounds.  For cols ids a weight is a whole multiple of 2^-s of the largest, s the largest up to 50 with 2^(62 - s) >= cols: 45 for 131072
ids, 44 beyond.  Each is off by half a unit, so that a sum of n weights w is off by less than n 2^-45, 2^-45 / w of itself: below 1e-10 for
the weights here, e^-8 and above.  The place of a border, and of the chosen id, in a run of equals is then off by less than 1e-4 of a place,
and none of those here falls that near to a whole one."""
import numpy as np
import pytest
import torch

import kv8_cases as K

pytestmark = pytest.mark.gpu
# the last of them takes the last id that is kept
UNIFORM = torch.tensor([0.0, 0.3, 0.77, 1 - 2.0 ** -24])


def check(row, dtype=torch.float32, **knobs):
    from baranet_bdml_b200 import ops
    x = row.to(dtype)[None].repeat(len(UNIFORM), 1).cuda()
    got = ops.sample_rows(x, UNIFORM.cuda(), **knobs)
    exact = x[0].float().cpu().numpy()
    assert got.tolist() == [K.choose(exact, float(u), **knobs) for u in UNIFORM]


def one_above(cols, gap):
    row = torch.full((cols,), -float(gap))
    row[cols // 3] = 0.0
    return row


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top_p", [0.05, 0.5, 0.9, 0.999])
@pytest.mark.parametrize("cols,gap", [(65537, 6), (131072, 8), (131072, 7.25), (151936, 5), (262143, 0.5), (262144, 8)])
def test_one_above_equals(lib, cols, gap, top_p, dtype):
    """More than 65537 ids in one step of the histogram: the 16-bit parts of their weights add up to more than 32 bits"""
    check(one_above(cols, gap), dtype, top_p=top_p)


@pytest.mark.parametrize("knobs", [{"top_p": 0.3}, {"top_p": 0.9, "top_k": 200001}, {"top_k": 131073}, {"min_p": 0.5}, {}], ids=str)
def test_all_equal(lib, knobs):
    check(torch.zeros(262144), **knobs)


@pytest.mark.parametrize("knobs", [{"top_p": 0.9}, {"top_p": 0.4, "temperature": 0.7}, {"top_p": 0.97, "top_k": 250000}, {"top_p": 0.8, "min_p": 0.01}], ids=str)
@pytest.mark.parametrize("cols", [100003, 200000, 262144])
def test_few_values(lib, cols, knobs):
    """Seven values in no order, one of them far more often than the others"""
    g = torch.Generator().manual_seed(cols)
    value = torch.tensor([0.0, -0.7, -1.9, -2.0, -2.1, -4.0, -7.3])
    which = torch.multinomial(torch.tensor([0.001, 0.01, 0.04, 0.8, 0.1, 0.04, 0.009]), cols, replacement=True, generator=g)
    check(value[which], **knobs)


@pytest.mark.parametrize("share", [0.999, 0.9995, 0.9999999, 1.0005, 1.001])
@pytest.mark.parametrize("cols,depth,run,second", [(187324, 0.25, 26, 22), (251913, 0.5, 11, 10), (167815, 1.0, 4, 3), (229292, 0.25, 16, 11), (187712, 0.5, 13, 7)])
def test_a_border_before_a_long_run(lib, cols, depth, run, second, share):
    """Two ids, then all others (`second` and `run` steps of the histogram below, and one at its end), and a top-p whose share of the sum is about
    what the two weigh: fp32 sums that take in the run have lost what tells on which side of it the border lies"""
    row = torch.full((cols,), float(np.float32(-run * depth / 512)))
    row[5], row[100], row[200] = -depth, 0.0, float(np.float32(-second * depth / 512))
    w = np.exp(row.double().numpy())
    check(row, top_p=float(np.float32((w[100] + w[200]) / w.sum() * share)))
