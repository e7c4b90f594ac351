"""Attention over the 8-bit cache where the scales of a sequence's values lie as far apart as the format allows, 2^-100 (which zeros
have) to 2^118 (beyond it results leave fp32).  The softmax's denominator knows nothing of them.

Bounds are those of test_gpu_kv8.check_decode: fp16 roundings of q and of the weights, against the definition in 64 bits."""
import pytest
import torch

import kv8_cases as K
from test_gpu_kv8 import VALUES, check_decode, fill, make, queries

pytestmark = pytest.mark.gpu


def run(values, lens, exponents, zero=None, hkv=1, heads=8, std=1.0, key_exponents=-40, seed=50, **kw):
    """Value scales 2^exponents[b][t], keys so small that the weights are about the same (unless `key_exponents` says so), tokens with
    `zero` having zeros at the format's least scale"""
    cache, table, rng = make(lens, hkv, values, seed)
    fill(cache, values, rng)
    gk, gv, ks, vs = K.unpacked(cache.pool, values)
    for b, n in enumerate(lens):
        for t in range(n):
            page, slot = table[b, t // K.PAGE], t % K.PAGE
            vs[page, :, slot] = 2.0 ** float(exponents(b, t))
            ks[page, :, slot] = 2.0 ** float(key_exponents(b, t) if callable(key_exponents) else key_exponents)
            if zero is not None and zero(b, t):
                gv[page, :, slot], vs[page, :, slot] = 0.0, K.LEAST
    cache.pool.copy_(K.packed(gk, gv, ks, vs, values))
    return check_decode(cache, gk * ks[..., None], gv * vs[..., None], table, lens, queries(rng, len(lens), heads, std), **kw)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("high", [36, 37, 59, 60, 61, 90, 100, 118])
@pytest.mark.parametrize("zero", ["before", "behind", "between", "first"])
def test_zeros_beside_large_values(lib, values, high, zero):
    """Zeros weigh as much as other tokens do, in a warp's stages before, behind or beside those of large values"""
    which = {"before": lambda b, t: t < 600, "behind": lambda b, t: t >= 600, "between": lambda b, t: t // 5 % 2 == 0,
             "first": lambda b, t: t > 0}[zero]
    run(values, [1200, 130], lambda b, t: high, which)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("spread", [62, 80, 100])
def test_any_scales(lib, values, spread):
    e = torch.randint(-spread, spread + 1, (3, 3000), generator=torch.Generator().manual_seed(spread))
    run(values, [600, 3000, 17], lambda b, t: e[b, t], hkv=2, heads=12)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("first,second", [(-100, 100), (100, -100), (118, 20), (20, 118), (-100, 37), (-34, 32), (-40, 34), (-100, -34)])
def test_parts_of_a_sequence_far_apart(lib, values, first, second):
    """Either half in other warps' and other CTAs' hands, which join what they have"""
    run(values, [9000], lambda b, t: first if t < 4500 else second)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("high", [0, 59, 60, 61, 118])
def test_many_small_weights_under_a_large_scale(lib, values, high):
    """One token's score stands some 12.5 above those of 16000 others, which together still count: with scales of 2^118 the weights over the
    scale lie below fp32's range"""
    lens, at = [16000], 9000
    cache, table, rng = make(lens, 1, values, 51)
    fill(cache, values, rng)
    gk, gv, ks, vs = K.unpacked(cache.pool, values)
    ks[:], vs[:] = 2.0 ** -40, 2.0 ** high
    page, slot = table[0, at // K.PAGE], at % K.PAGE
    gk[page, 0, slot], ks[page, 0, slot] = 64.0, 2.0 ** -5           # (1/8 * 64 / 32 * sum |q|, which is about 51)
    cache.pool.copy_(K.packed(gk, gv, ks, vs, values))
    check_decode(cache, gk * ks[..., None], gv * vs[..., None], table, lens, queries(rng, 1, 8).abs(), rope=False)


@pytest.mark.parametrize("values", VALUES)
def test_scores_rise_while_scales_fall(lib, values):
    """From stage to stage scores rise by more than scales fall and the other way round"""
    run(values, [5000, 5000], lambda b, t: 100 - t // 25 if b == 0 else -100 + t // 25, std=0.5,
        key_exponents=lambda b, t: -12 + t // 600)
