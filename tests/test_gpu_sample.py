"""Sampled ids, against the definition in extended precision: they are whole numbers, so they are equal.

Weights are whole multiples of 2^-46 of the largest (32000 ids) or finer, so that the sums at a border are off by less than 1e-9 of a row's
sum: of the some 1e4 random rows here none falls that near to one.  Borders that fall on a sum by construction are those of equal
weights, whose sums are exact."""
import numpy as np
import pytest
import torch

import kv8_cases as K

pytestmark = pytest.mark.gpu


def want(x, u, **knobs):
    rows = x.shape[0]
    one = lambda v, r: v[r].item() if isinstance(v, torch.Tensor) else v      # noqa: E731
    x = x.float().cpu().numpy()
    return [K.choose(x[r], float(u[r]), **{k: one(v, r) for k, v in knobs.items()}) for r in range(rows)]


def check(x, u, **knobs):
    from baranet_bdml_b200 import ops
    got = ops.sample_rows(x, u, **knobs)
    assert got.dtype == torch.int32 and got.shape == (x.shape[0],)
    assert got.tolist() == want(x, u, **knobs)


def logits(rows, vocab, seed, std=2.5, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * std).to(dtype), torch.rand((rows,), generator=g, device="cuda")


KNOBS = [{}, {"temperature": 0.3}, {"temperature": 5.0}, {"top_k": 1}, {"top_k": 50}, {"top_k": 700, "temperature": 2.0}, {"top_p": 0.9},
         {"top_p": 0.999, "temperature": 3.0}, {"top_p": 0.0}, {"min_p": 0.05}, {"min_p": 1.0}, {"top_k": 40, "top_p": 0.8, "min_p": 0.02, "temperature": 1.3},
         {"top_k": 5000, "top_p": 0.97, "temperature": 4.0}, {"temperature": 0.0}, {"temperature": 1e-30}, {"temperature": 1e30, "top_p": 0.5}]


@pytest.mark.parametrize("knobs", KNOBS, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (5, 10007), (33, 1000), (3, 131072), (200, 77)])
def test_sample(lib, rows, vocab, knobs):
    check(*logits(rows, vocab, vocab + rows), **knobs)


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 32, 33, 1023, 1024, 1025, 4099, 70001, 262143])
def test_sizes(lib, vocab):
    x, u = logits(4, vocab, vocab)
    for knobs in ({}, {"top_k": 2}, {"top_p": 0.7}, {"top_k": max(1, vocab // 2), "top_p": 0.9, "min_p": 0.01}):
        check(x, u, **knobs)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 75, 150, 700])
def test_rows(lib, rows):
    x, u = logits(rows, 3001, rows)
    check(x, u, top_p=0.8, temperature=1.5)
    check(x, u, top_k=20, min_p=0.1)


@pytest.mark.parametrize("levels", [1, 2, 7, 100])
def test_equals_go_by_their_ids(lib, levels):
    """Logits of few values: the last that are kept are cut out of a run of equals"""
    g = torch.Generator(device="cuda").manual_seed(levels)
    x = torch.randint(0, levels, (40, 5000), generator=g, device="cuda").float() / 4
    u = torch.rand((40,), generator=g, device="cuda")
    for knobs in ({"top_k": 3}, {"top_k": 1234}, {"top_p": 0.37}, {"top_k": 2001, "top_p": 0.61}, {"min_p": 0.9}, {}):
        check(x, u, **knobs)
    x[:, ::3] = -x[:, ::3]                                    # -0 equals 0
    check(x, u, top_k=777)


def test_sums_that_fall_on_a_border(lib):
    """1000 equal weights: u = j / 1000 and top_p = j / 1000 where both are exact"""
    x = torch.zeros((5, 1024), device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    from baranet_bdml_b200 import ops
    assert ops.sample_rows(x, u).tolist() == [0, 256, 512, 768, 1023]
    assert ops.sample_rows(x, u, top_p=0.5).tolist() == [0, 128, 256, 384, 511]
    assert ops.sample_rows(x, u, top_k=4, top_p=0.5).tolist() == [0, 0, 1, 1, 1]
    check(x, u, top_p=0.125)


def test_ends_of_the_random_numbers(lib):
    x, _ = logits(6, 2000, 4, std=60.0)                       # weights down to 1e-80
    for value in (0.0, 1 - 2.0 ** -24, 1.0, 7.0, -1.0):
        u = torch.full((6,), value, device="cuda")
        inside = torch.full((6,), min(max(value, 0.0), 1.0), device="cuda")
        from baranet_bdml_b200 import ops
        for knobs in ({}, {"top_k": 10}, {"top_p": 0.99}):
            assert ops.sample_rows(x, u, **knobs).tolist() == want(x, inside, **knobs)
    u = torch.full((6,), float("nan"), device="cuda")
    assert ops.sample_rows(x, u).tolist() == ops.sample_rows(x, torch.zeros_like(u)).tolist()


def test_masked_rows(lib):
    """-inf, the type's lowest value, NaN and +inf among the logits, and rows with nothing left"""
    x, u = logits(12, 3000, 5)
    x[0] = -np.inf
    x[1] = float("nan")
    x[2, :-1] = -np.inf
    x[3] = torch.finfo(torch.float32).min
    x[4, 100:] = torch.finfo(torch.float32).min
    x[5, ::2] = float("nan")
    x[6, [5, 77, 2000]] = np.inf
    x[7, 1:] = -np.inf
    x[8] = torch.finfo(torch.float32).max
    x[9] *= 1e30
    x[10, :2990] = -1e4
    x[11, 0] = float("nan")
    for knobs in KNOBS:
        check(x, u, **knobs)
    check(x, u, top_k=2999)


@pytest.mark.parametrize("kept", [31, 127, 128, 129, 200, 255, 256, 257, 300, 384, 385, 511, 512, 513])
def test_as_many_as_a_list_holds(lib, kept):
    """Where the choice is made from a list and where not, and how the list is ranked"""
    x, u = logits(6, 4000, kept)
    check(x, u, top_k=kept, temperature=3.0)
    check(x, u, top_k=kept, top_p=0.95, temperature=3.0)
    x[:, kept:] -= 1000.0                                     # top-p: of kept ids, and of some more equals
    check(x, u, top_p=0.999, temperature=3.0)
    x[:, kept:2 * kept] = x[:, :1]
    check(x, u, top_p=0.6)


@pytest.mark.parametrize("temperature", [1e-45, 1e-38, 1e-30, 1e-20])
def test_the_smallest_temperatures(lib, temperature):
    x, u = logits(5, 3000, 12)
    x[1] *= 1e-18
    x[2] = x[2].round()
    for knobs in ({}, {"top_k": 30}, {"top_p": 0.9}, {"top_k": 300, "top_p": 0.5, "min_p": 0.1}):
        check(x, u, temperature=temperature, **knobs)


@pytest.mark.parametrize("knobs", KNOBS[3:8] + KNOBS[11:13], ids=str)
def test_bf16_and_strided_rows(lib, knobs):
    x, u = logits(9, 5005, 6, dtype=torch.bfloat16)
    check(x, u, **knobs)
    wide, _ = logits(9, 5100, 7)
    check(wide[:, 3:4900], u, **knobs)
    check(wide.to(torch.bfloat16)[:, 1:4900], u, **knobs)
    check(wide[::2], u[::2].contiguous(), **knobs)


def test_a_knob_for_each_row(lib):
    x, u = logits(64, 4000, 8)
    g = torch.Generator(device="cuda").manual_seed(9)
    knobs = {"temperature": torch.rand((64,), generator=g, device="cuda") * 2, "top_k": torch.randint(0, 300, (64,), generator=g, device="cuda").to(torch.int32),
             "top_p": torch.rand((64,), generator=g, device="cuda"), "min_p": torch.rand((64,), generator=g, device="cuda") * 0.1}
    knobs["temperature"][:5] = 0.0
    knobs["top_p"][10:20] = 1.0
    check(x, u, **knobs)
    for name in knobs:
        check(x, u, **{name: knobs[name]})
    # numbers that no check on the host has seen: below 0 is 0, above 1 is 1, NaN is no limit, a NaN temperature 0
    from baranet_bdml_b200 import ops
    odd = torch.tensor([-1.0, 2.0, float("nan"), 0.5], device="cuda").repeat(16)
    assert ops.sample_rows(x, u, top_p=odd).tolist() == want(x, u, top_p=torch.tensor([0.0, 1.0, 1.0, 0.5]).repeat(16))
    assert ops.sample_rows(x, u, min_p=odd).tolist() == want(x, u, min_p=torch.tensor([0.0, 1.0, 0.0, 0.5]).repeat(16))
    assert ops.sample_rows(x, u, temperature=odd).tolist() == want(x, u, temperature=torch.tensor([0.0, 2.0, 0.0, 0.5]).repeat(16))
    assert ops.sample_rows(x, u, top_k=torch.full((64,), -3, dtype=torch.int32, device="cuda")).tolist() == want(x, u)


def test_frequencies(lib):
    """Over evenly spread random numbers every id comes as often as its weight says, to one"""
    from baranet_bdml_b200 import ops
    n = 4096
    row = torch.tensor([[2.0, 0.0, 1.0, -np.inf, 1.5, -3.0]], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(ops.sample_rows(row.repeat(n, 1), u, temperature=0.7).long(), minlength=6).double().cpu()
    w = torch.softmax(row[0].double().cpu() / np.float32(0.7).item(), 0)
    assert ((got - n * w).abs() <= 1).all()


def test_streams_and_graphs(lib):
    from baranet_bdml_b200 import ops
    x, u = logits(20, 32000, 10)
    a = want(x, u, top_p=0.9, top_k=100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_rows(x, u, top_p=0.9, top_k=100)
    side.synchronize()
    assert got.tolist() == a
    out = torch.empty((20,), dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_rows(x, u, top_p=0.9, top_k=100, out=out)
    for seed in (11, 12):
        y, w = logits(20, 32000, seed)
        x.copy_(y)
        u.copy_(w)
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == want(x, u, top_p=0.9, top_k=100)


def test_refusals(lib):
    from baranet_bdml_b200 import ops
    x, u = logits(3, 100, 13)
    for call in (lambda: ops.sample_rows(x, u, temperature=-1.0), lambda: ops.sample_rows(x, u, temperature=float("nan")), lambda: ops.sample_rows(x, u, top_p=1.5),
                 lambda: ops.sample_rows(x, u, top_k=-1), lambda: ops.sample_rows(x, u, min_p=-0.1), lambda: ops.sample_rows(x, u[:2]),
                 lambda: ops.sample_rows(x, u.double()), lambda: ops.sample_rows(x.half(), u), lambda: ops.sample_rows(x.T, u), lambda: ops.sample_rows(x[0], u),
                 lambda: ops.sample_rows(x[:, :0], u), lambda: ops.sample_rows(x.cpu(), u.cpu()), lambda: ops.sample_rows(x, u.cpu()),
                 lambda: ops.sample_rows(x, u, top_k=torch.ones((3,), device="cuda")), lambda: ops.sample_rows(x[:1].expand(3, 100), u),
                 lambda: ops.sample_rows(torch.zeros((1, (1 << 18) + 1), device="cuda"), u[:1])):
        with pytest.raises(RuntimeError):
            call()
    assert ops.sample_rows(x[:0], u[:0]).shape == (0,)
