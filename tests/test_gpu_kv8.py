"""The paged cache in 8 bits: what is written, what is read back and attention over it, against the definitions in 64 bits.

Bounds.  A rotated number is off by no more than 2^-20 (|a| + |b|) of its pair (the reduced angle's and the functions' roundings, 2^-22.3
and 2^-22.4 together, and those of the products).  Rounding to e4m3 is off by half a step, 2^-4 of the number or 2^-10 of the scale,
to int8 by half the scale.  Reading back multiplies a number of at most 7 bits by one of at most 8: exact in fp32, one rounding to
bf16.  In attention q and p are rounded to fp16 (2^-11 each); scores are off by d = 2^-11 scale sum |q| |k|, so the weights by a factor
within exp(+-2 d), and sums run in fp32."""
import numpy as np
import pytest
import torch

import kv8_cases as K

pytestmark = pytest.mark.gpu
VALUES = ["e4m3", "int8"]


def make(lens, hkv, values, seed, extra=3, extra_width=0):
    """A cache with room for `lens` tokens, pages in no order"""
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    rng = np.random.default_rng(seed)
    per = [-(-n // K.PAGE) for n in lens]
    width = max(max(per), 1) + extra_width
    pages = sum(per) + extra
    cache = QuantizedKVCache(pages, len(lens), width, hkv, values=values)
    order = rng.permutation(pages)
    table = np.full((len(lens), width), -1, dtype=np.int32)     # nothing may look behind a sequence's pages
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    cache.page_table.copy_(torch.from_numpy(table))
    cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache, table, rng


def fill(cache, values, rng, poison=None):
    """Every block random; `poison`: the blocks' bytes behind a sequence's end are all ones (NaN in e4m3 and as a scale)"""
    pages, hkv = cache.num_pages, cache.num_kv_heads
    g = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    if values == "e4m3":
        k, v = (torch.randn((pages, hkv, K.PAGE, K.D), generator=g).mul(120).clamp(-448, 448).to(torch.float8_e4m3fn).double() for _ in range(2))
        ks, vs = (2.0 ** torch.randint(-9, -5, (pages, hkv, K.PAGE), generator=g).double() for _ in range(2))
    else:
        k, v = (torch.randint(-127, 128, (pages, hkv, K.PAGE, K.D), generator=g).double() for _ in range(2))
        ks, vs = ((0.01 + 0.03 * torch.rand((pages, hkv, K.PAGE), generator=g)).to(torch.bfloat16).double() for _ in range(2))
    pool = K.packed(k, v, ks, vs, values)
    if poison is not None:
        table, lens = poison
        for b, n in enumerate(lens):
            for s in range(n % K.PAGE if n % K.PAGE else K.PAGE, K.PAGE):
                block = pool[table[b, (n - 1) // K.PAGE]]
                block[:, s * 64:s * 64 + 64] = 255
                block[:, 1024 + s * 64:1024 + s * 64 + 64] = 255
                block[:, 2048 + s * 4:2048 + s * 4 + 4] = 255
    cache.pool.copy_(pool)
    return k * ks[..., None], v * vs[..., None]


def sequence(x, table, b, n):
    """(tokens, kv heads, 64) of sequence b out of (pages, kv heads, 16, 64)"""
    return x[table[b, :-(-n // K.PAGE)]].transpose(1, 2).reshape(-1, x.shape[1], K.D)[:n]


# ------------------------------------------------------------------------------------------------------------------ writing
def check_written(cache, table, seqs, positions, k, v, values, rotate=True, pool_before=None):
    gk, gv, ks, vs = K.unpacked(cache.pool, values)
    at = [(table[s, p // K.PAGE], p % K.PAGE) for s, p in zip(seqs, positions)]
    pages, slots = torch.tensor([a for a, _ in at]), torch.tensor([b for _, b in at])
    x = k.double().cpu().view(len(seqs), -1, K.D)
    rot = K.rotated(x, positions) if rotate else x
    slack = (x[..., 0::2].abs() + x[..., 1::2].abs()).repeat_interleave(2, -1) * 2.0 ** -20 * rotate
    for got, scale, want, off in ((gk, ks, rot, slack), (gv, vs, v.double().cpu().view_as(x), torch.zeros_like(x))):
        got, scale = got[pages, :, slots], scale[pages, :, slots]
        most = want.abs().amax(-1).numpy()
        low, high = (K.scale_rule(m, values) for m in (most * (1 - 2.0 ** -19), most * (1 + 2.0 ** -19)))
        s = scale.numpy()
        assert ((s >= low) & (s <= high)).all()
        step = want.abs() * 2.0 ** -4 + scale[..., None] * 2.0 ** -10 if values == "e4m3" else scale[..., None] * 0.5
        err = (got * scale[..., None] - want).abs()
        assert (err <= step * (1 + 2.0 ** -20) + off * 1.07).all(), (err - step).max()


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hkv,T", [(4, 1), (4, 16), (1, 37), (8, 100), (3, 5)])
def test_append(lib, values, dtype, hkv, T):
    cache, table, rng = make([200, 1000, 33], hkv, values, T + hkv)
    pairs = [(s, p) for s, n in enumerate([200, 1000, 33]) for p in range(n)]
    pick = rng.permutation(len(pairs))[:T]
    seqs, pos = np.array([pairs[i][0] for i in pick]), np.array([pairs[i][1] for i in pick])
    g = torch.Generator(device="cuda").manual_seed(T)
    k, v = (torch.randn((T, hkv * K.D), generator=g, device="cuda").mul(s).to(dtype) for s in (1.0, 30.0))
    before = torch.randint(0, 256, cache.pool.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(5))
    cache.pool.copy_(before)
    ids = torch.tensor(seqs, dtype=torch.int32, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")
    cache.append(*ids, k, v)
    check_written(cache, table, seqs, pos, k, v, values)
    # nothing else has changed
    after, mask = cache.pool.cpu(), torch.ones(cache.pool.shape, dtype=torch.bool)
    for s, p in zip(seqs, pos):
        page, slot = table[s, p // K.PAGE], p % K.PAGE
        for lo, n in ((slot * 64, 64), (1024 + slot * 64, 64), (2048 + slot * 4, 4)):
            mask[page, :, lo:lo + n] = False
    assert torch.equal(after[mask], before[mask])
    cache.append(*ids, k, v, rotated=True)
    check_written(cache, table, seqs, pos, k, v, values, rotate=False)


@pytest.mark.parametrize("values", VALUES)
def test_append_far_positions_strides_and_thetas(lib, values):
    """Angles far along a sequence; rows that are parts of wider ones, whose starts are on no 16-byte boundary"""
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    width = 1 << 17
    cache = QuantizedKVCache(4, 1, width, 2, values=values)
    pos = [0, 15, 123456, 999999, width * 16 - 1]
    table = np.zeros((1, width), dtype=np.int32)
    for i, page in enumerate(sorted({p // 16 for p in pos})):
        table[0, page] = i
    cache.page_table.copy_(torch.from_numpy(table))
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn((5, 2 * 128 + 3), generator=g, device="cuda")
    other = torch.randn((5, 200), generator=g, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        k, v = wide.to(dtype)[:, 3:131], other.to(dtype)[:, 8:136]
        cache.append(torch.zeros(5, dtype=torch.int32, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda"), k, v)
        check_written(cache, table, [0] * 5, pos, k, v, values)


@pytest.mark.parametrize("values", VALUES)
def test_append_extremes(lib, values):
    """Zeros, the smallest and largest numbers, powers of two and 448, and rows that are not finite, which concern nobody else"""
    cache, table, rng = make([32], 1, values, 3)
    rows = torch.zeros((12, K.D))
    rows[1] = 1e-42
    rows[2] = 3.0e38
    rows[3, 5] = 448.0
    rows[4, 5] = 448.0 * (1 + 2.0 ** -20)
    rows[5, 7] = float("inf")
    rows[6, 9] = float("nan")
    rows[7] = torch.linspace(-1, 1, K.D) * 2.0 ** -70
    rows[8] = 2.0 ** -100 * torch.linspace(-3, 3, K.D)
    rows[9, 0] = -127.0
    rows[10] = torch.linspace(-127.5, 127.5, K.D)
    rows[11] = 2.0 ** 100 * torch.linspace(-3, 3, K.D)
    rows = rows.cuda()
    n = rows.shape[0]
    ids, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    cache.append(ids, pos, rows, rows, rotated=True)
    gk, gv, ks, vs = K.unpacked(cache.pool, values)
    page = table[0, 0]
    for got, scale in ((gk, ks), (gv, vs)):
        got, scale = got[page, 0, :n], scale[page, 0, :n]
        assert torch.isnan(scale[5]) and torch.isnan(scale[6])
        fine = [i for i in range(n) if i not in (5, 6)]
        x, s = rows.double().cpu()[fine], scale[fine]
        assert np.array_equal(s.numpy(), K.scale_rule(x.abs().amax(-1).numpy(), values))
        step = x.abs() * 2.0 ** -4 + s[:, None] * 2.0 ** -10 if values == "e4m3" else s[:, None] * 0.5 * (1 + 2.0 ** -20)
        assert ((got[fine] * s[:, None] - x).abs() <= step).all()
    k, v = cache.gather(ids[:1], pos[:1], n)
    assert torch.isnan(k[0, [5, 6]]).all() and torch.isnan(v[0, [5, 6]]).all() and torch.isfinite(k[0, [0, 4, 7, 11]]).all()


def test_append_leaves_out_what_lies_outside(lib):
    cache, table, rng = make([20, 20], 2, "e4m3", 4)
    cache.page_table[1, 1] = cache.num_pages            # a page that is none
    before = cache.pool.clone()
    seqs = torch.tensor([-1, 2, 0, 0, 1, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 0, -1, 32, 17, 1 << 30], dtype=torch.int32, device="cuda")
    x = torch.ones((6, 128), device="cuda")
    cache.append(seqs, pos, x, x)
    assert torch.equal(cache.pool, before)
    cache.append(seqs[:0], pos[:0], x[:0], x[:0])
    assert torch.equal(cache.pool, before)


# ------------------------------------------------------------------------------------------------------------- reading back
@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gather(lib, values, dtype):
    lens = [0, 1, 16, 17, 333, 100]
    cache, table, rng = make(lens, 3, values, 7)
    k, v = fill(cache, values, rng, poison=(table, lens))
    for seqs, starts, n in (([4, 2, 0, 3, 1, 5], [0, 0, 0, 0, 0, 0], 340), ([5, 5, 4], [90, 99, 40], 7), ([3], [16], 1), ([4], [-3], 5), ([4], [1 << 30], 2),
                            ([6, -1, 3], [0, 0, 0], 2)):
        ids = (torch.tensor(a, dtype=torch.int32, device="cuda") for a in (seqs, starts))
        got = cache.gather(*ids, n, dtype=dtype)
        for x, out in zip((k, v), got):
            want = torch.zeros((len(seqs), n, 3, K.D), dtype=torch.float64)
            for i, (s, a) in enumerate(zip(seqs, starts)):
                for j in range(n):
                    if 0 <= s < len(lens) and 0 <= a + j < lens[s]:
                        want[i, j] = x[table[s, (a + j) // K.PAGE], :, (a + j) % K.PAGE]
            assert out.dtype == dtype and torch.equal(out.cpu(), want.to(dtype))
    empty = cache.gather(torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"), 4)
    assert empty[0].shape == (0, 4, 3, K.D)


# ---------------------------------------------------------------------------------------------------------------- attention
def check_decode(cache, k, v, table, lens, q, scale=None, rope=True, q_positions=None, **kw):
    B, heads, _ = q.shape
    tq = q.cuda()
    out, out32 = torch.empty_like(tq), torch.empty(q.shape, dtype=torch.float32, device="cuda")
    lse = torch.empty((B, heads), dtype=torch.float32, device="cuda")
    kw.setdefault("max_seq_len", max(max(lens), 1))
    cache.decode(tq, num_heads=heads, out=out, out_f32=out32, lse=lse, scale=scale, rope_q=rope, q_positions=q_positions, **kw)
    torch.cuda.synchronize()
    cache.status()
    scale = K.D ** -0.5 if scale is None else scale
    for b, n in enumerate(lens):
        if n == 0:
            assert not out[b].any() and not out32[b].any() and (lse[b] == -np.inf).all()
            continue
        at = n - 1 if q_positions is None else int(q_positions[b])
        qb = q[b].double()
        if rope:
            qb = K.rotated(qb[None], [at], cache.theta)[0]
        want, wlse, mass, size = K.attention(qb, sequence(k, table, b, n), sequence(v, table, b, n), scale)
        d = size[:, None] * (2.0 ** -11 + 2.0 ** -17)
        bound = mass * (torch.expm1(2 * d) + 2 * 2.0 ** -11 + 2.0 ** -16) + 1e-30
        err = (out32[b].double().cpu() - want).abs()
        assert (err <= bound).all(), (b, n, (err / bound).max())
        assert ((out[b].double().cpu() - want).abs() <= bound + (want.abs() + bound) * 2.0 ** -8).all()
        assert ((lse[b].double().cpu() - wlse).abs() <= d[:, 0] + 2.0 ** -11 + 2.0 ** -20 * wlse.abs()).all()
    return out, out32, lse


def queries(rng, B, heads, std=1.0):
    return torch.from_numpy(rng.standard_normal((B, heads, K.D)).astype(np.float32) * std).to(torch.bfloat16)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("heads,hkv", [(32, 4), (8, 8), (6, 2), (8, 1), (7, 1), (5, 5)])
@pytest.mark.parametrize("lens", [[1], [16], [17], [1024], [5, 130, 16, 511, 512, 513, 2049], [0, 3, 0, 700]])
def test_decode(lib, values, heads, hkv, lens):
    cache, table, rng = make(lens, hkv, values, sum(lens) + heads)
    k, v = fill(cache, values, rng, poison=(table, lens))
    check_decode(cache, k, v, table, lens, queries(rng, len(lens), heads))


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("lens", [[4096], [20000, 3], [5, 130, 16, 511, 512, 513, 2048, 1, 0, 257], [(37 * i) % 600 for i in range(50)],
                                  [0] * 30 + [1] * 200, [7] * 1024])
def test_decode_splits_and_batches(lib, values, lens):
    cache, table, rng = make(lens, 4, values, len(lens))
    k, v = fill(cache, values, rng, poison=(table, lens))
    check_decode(cache, k, v, table, lens, queries(rng, len(lens), 32))


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("chunk", [128, 256, 1024, 8192])
def test_decode_chunks(lib, values, chunk):
    lens = [3000, 777, 4096, 129]
    cache, table, rng = make(lens, 4, values, 21)
    k, v = fill(cache, values, rng, poison=(table, lens))
    q = queries(rng, 4, 32)
    a = check_decode(cache, k, v, table, lens, q, max_seq_len=4096, chunk_tokens=chunk)
    b = check_decode(cache, k, v, table, lens, q, max_seq_len=4096, chunk_tokens=chunk)
    assert all(torch.equal(x, y) for x, y in zip(a, b))          # the scratch buffer is left clean, and sums have one order


@pytest.mark.parametrize("values", VALUES)
def test_decode_arguments(lib, values):
    """Own scale, no rotation, positions apart from the lengths, a max_seq_len that cuts, another table, all outputs or one"""
    lens = [100, 700]
    cache, table, rng = make(lens, 2, values, 8)
    k, v = fill(cache, values, rng, poison=(table, lens))
    q = queries(rng, 2, 8)
    check_decode(cache, k, v, table, lens, q, scale=0.3, rope=False)
    check_decode(cache, k, v, table, lens, q, scale=-0.05)
    check_decode(cache, k, v, table, lens, q, q_positions=torch.tensor([1000003, 0], dtype=torch.int32, device="cuda"))
    check_decode(cache, k, v, table, [64, 64], q, max_seq_len=64, q_positions=torch.tensor([99, 699], dtype=torch.int32, device="cuda"))
    other = torch.from_numpy(np.ascontiguousarray(table[::-1])).cuda()
    check_decode(cache, k, v, table[::-1], [100, 90], q, page_table=other, seq_lens=torch.tensor([100, 90], dtype=torch.int32, device="cuda"))
    only = cache.decode(q.cuda(), num_heads=8)
    assert torch.equal(only, cache.decode(q.cuda(), num_heads=8, out=torch.empty_like(only)))
    assert cache.decode(q.cuda(), num_heads=8, out_f32=torch.empty((2, 8, 64), device="cuda")).dtype == torch.float32
    assert cache.decode(q[:0].cuda(), num_heads=8, seq_lens=cache.seq_lens[:0]).shape == (0, 8, 64)


@pytest.mark.parametrize("values", VALUES)
@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_decode_sizes_of_queries(lib, values, std):
    """Nearly equal weights, and a weight that stands alone"""
    lens = [333, 2500]
    cache, table, rng = make(lens, 4, values, 9)
    k, v = fill(cache, values, rng)
    check_decode(cache, k, v, table, lens, queries(rng, 2, 32, std))


@pytest.mark.parametrize("values", VALUES)
def test_decode_scales_far_apart(lib, values):
    """Values of very different sizes: a small weight on large values counts as much as a large one on small values"""
    lens = [600]
    cache, table, rng = make(lens, 1, values, 10)
    k, v = fill(cache, values, rng)
    # token sizes over 2^-60 .. 2^60, keys so small that all weights are about the same, or growing the other way
    pages = cache.num_pages
    gk, gv, ks, vs = K.unpacked(cache.pool, values)
    e = torch.randint(-60, 61, vs.shape, generator=torch.Generator().manual_seed(1))
    vs = 2.0 ** e.double()
    ks = torch.full_like(ks, 2.0 ** -40)
    cache.pool.copy_(K.packed(gk, gv, ks, vs, values))
    check_decode(cache, gk * ks[..., None], gv * vs[..., None], table, lens, queries(rng, 1, 8))
    # zero values, smallest scales
    zero = torch.zeros_like(gv)
    vs = torch.full_like(vs, K.LEAST)
    cache.pool.copy_(K.packed(gk, zero, ks, vs, values))
    out, out32, _ = check_decode(cache, gk * ks[..., None], zero, table, lens, queries(rng, 1, 8))
    assert not out32.any()
    assert pages > 37


@pytest.mark.parametrize("values", VALUES)
def test_decode_not_finite_concerns_one_sequence(lib, values):
    lens = [300, 300, 300]
    cache, table, rng = make(lens, 2, values, 11)
    k, v = fill(cache, values, rng)
    q = queries(rng, 3, 16)
    clean = cache.decode(q.cuda(), num_heads=16)
    bad = torch.zeros((2, 128), device="cuda")
    bad[0, 3], bad[1, 70] = float("nan"), float("inf")
    ids, pos = torch.tensor([1, 2], dtype=torch.int32, device="cuda"), torch.tensor([77, 299], dtype=torch.int32, device="cuda")
    cache.append(ids, pos, torch.zeros_like(bad), bad)
    got = cache.decode(q.cuda(), num_heads=16)
    assert torch.equal(got[0], clean[0])
    assert torch.isnan(got[1, :8]).all() and torch.isfinite(got[1, 8:]).all()      # the key heads of a token are apart
    assert torch.isnan(got[2, 8:]).all() and torch.isfinite(got[2, :8]).all()
    cache.append(ids, pos, bad, torch.zeros_like(bad), rotated=True)
    got = cache.decode(q.cuda(), num_heads=16)
    assert torch.equal(got[0], clean[0]) and torch.isnan(got[1, :8]).all() and torch.isnan(got[2, 8:]).all() and torch.isfinite(got[2, :8]).all()
    # behind the sequence's end they concern nobody
    cache.append(ids, torch.tensor([301, 303], dtype=torch.int32, device="cuda"), bad, bad)
    cache.seq_lens.copy_(torch.tensor([300, 70, 299], dtype=torch.int32))
    assert torch.isfinite(cache.decode(q.cuda(), num_heads=16)).all()


def test_a_page_outside_the_pool_is_reported(lib):
    cache, table, rng = make([100, 100], 2, "e4m3", 12)
    k, v = fill(cache, "e4m3", rng)
    q = queries(rng, 2, 8).cuda()
    good = cache.decode(q, num_heads=8)
    cache.status()
    for page in (cache.num_pages, -1, 1 << 30):
        broken = cache.page_table.clone()
        broken[1, 3] = page
        cache.decode(q, num_heads=8, page_table=broken)
        with pytest.raises(RuntimeError, match="outside the pool"):
            cache.status()
        for ws in cache._ws.values():
            ws.buf.zero_()
    assert torch.equal(cache.decode(q, num_heads=8), good)
    cache.status()


@pytest.mark.parametrize("values", VALUES)
def test_blocks_beyond_4_gb(lib, values):
    """Offsets into a pool that pass 32 bits"""
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    pages, hkv = (1 << 32) // (K.BLOCK * 4) + 40, 4
    storage = (torch.empty((pages, hkv, K.BLOCK), dtype=torch.uint8, device="cuda"), torch.zeros((1, 4), dtype=torch.int32, device="cuda"),
               torch.full((1,), 50, dtype=torch.int32, device="cuda"))
    cache = QuantizedKVCache(pages, 1, 4, hkv, values=values, storage=storage)
    table = np.array([[pages - 1, 0, pages - 17, pages - 2]], dtype=np.int32)
    cache.page_table.copy_(torch.from_numpy(table))
    g = torch.Generator(device="cuda").manual_seed(2)
    kk, vv = (torch.randn((50, hkv * K.D), generator=g, device="cuda") for _ in range(2))
    ids, pos = torch.zeros(50, dtype=torch.int32, device="cuda"), torch.arange(50, dtype=torch.int32, device="cuda")
    cache.append(ids, pos, kk, vv, rotated=True)
    k, v = (x[0].double().cpu() for x in cache.gather(ids[:1], pos[:1], 50, dtype=torch.float32))
    unit = 2.0 ** -4 if values == "e4m3" else 2.0 ** -6
    assert (k - kk.double().cpu().view_as(k)).abs().max() <= unit * kk.abs().max().item()
    q = queries(np.random.default_rng(3), 1, 32)
    got = cache.decode(q.cuda(), num_heads=32, rope_q=False, out_f32=torch.empty((1, 32, 64), device="cuda"))
    want, _, mass, size = K.attention(q[0].double(), k, v, 0.125)
    d = size[:, None] * (2.0 ** -11 + 2.0 ** -17)
    assert ((got[0].double().cpu() - want).abs() <= mass * (torch.expm1(2 * d) + 2.0 ** -10 + 2.0 ** -16)).all()


@pytest.mark.parametrize("values", VALUES)
def test_streams_graphs_and_two_at_once(lib, values):
    """Written, read and attended on a stream of their own, captured and replayed with other contents and lengths, and two caches at once"""
    lens = [300, 40, 2000]
    made = [make(lens, 4, values, 30 + i, extra_width=2) for i in range(2)]
    caches = [m[0] for m in made]
    for cache, table, rng in made:
        fill(cache, values, rng)
        cache.page_table.clamp_(min=0)
    q = queries(np.random.default_rng(1), 3, 32).cuda()
    g = torch.Generator(device="cuda").manual_seed(3)
    kn, vn = (torch.randn((3, 256), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ids = torch.arange(3, dtype=torch.int32, device="cuda")
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")

    def step(cache):
        cache.append(ids, pos, kn, vn)
        return cache.decode(q, num_heads=32), *cache.gather(ids, pos, 1)

    want = [[t.clone() for t in step(c)] for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(caches[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, h in zip(want, got) for a, b in zip(w, h))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(caches[0])
    for shift in (0, 3):
        vn.copy_(torch.roll(vn, shift, 1))
        pos.sub_(shift)
        caches[0].seq_lens.sub_(shift)
        graph.replay()
        torch.cuda.synchronize()
        again = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(again, step(caches[0])))


@pytest.mark.parametrize("values", VALUES)
def test_one_cache_on_two_streams(lib, values):
    """Two batches of queries against one cache at the same time, each long enough to be split over CTAs and merged"""
    lens = [9000, 5000, 7]
    cache, table, rng = make(lens, 4, values, 40)
    k, v = fill(cache, values, rng)
    qs = [queries(rng, 3, 32) for _ in range(2)]
    want = [check_decode(cache, k, v, table, lens, q)[1].clone() for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    on_gpu = [q.cuda() for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.decode(on_gpu[i], num_heads=32, out_f32=torch.empty((3, 32, 64), device="cuda")))
    torch.cuda.synchronize()
    cache.status()
    assert all(torch.equal(g, w) for w, rows in zip(want, got) for g in rows)


def test_graphs_of_one_cache_side_by_side(lib):
    """Captured before any call, behind calls, and behind another capture; replayed last one first, on two streams at once"""
    lens = [9000, 5000, 7]
    cache, table, rng = make(lens, 4, "e4m3", 41)
    k, v = fill(cache, "e4m3", rng)
    qs = [queries(rng, 3, 32) for _ in range(4)]
    on_gpu, got = [q.cuda() for q in qs], [torch.empty((3, 32, 64), device="cuda") for _ in qs]
    graphs = [torch.cuda.CUDAGraph() for _ in qs]

    def capture(i):
        with torch.cuda.graph(graphs[i]):
            cache.decode(on_gpu[i], num_heads=32, out_f32=got[i])

    capture(0)
    capture(1)
    want = [check_decode(cache, k, v, table, lens, q)[1].clone() for q in qs]
    capture(2)
    capture(3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for first, second in ((1, 0), (3, 2), (0, 3), (2, 1)):
        for _ in range(10):
            for s, i in zip(streams, (first, second)):
                with torch.cuda.stream(s):
                    graphs[i].replay()
        torch.cuda.synchronize()
        cache.status()
        for i in (first, second):
            assert torch.equal(got[i], want[i])
            got[i].zero_()
        torch.cuda.synchronize()


def test_refusals_on_the_gpu(lib):
    cache, table, rng = make([100], 2, "e4m3", 13)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")      # noqa: E731
    x = torch.zeros((1, 128), device="cuda")
    q = torch.zeros((1, 8, 64), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: cache.append(i32(0), i32(0), x[:, :64], x), lambda: cache.append(i32(0), i32(0, 1), x, x), lambda: cache.append(i32(0).long(), i32(0), x, x),
                 lambda: cache.append(i32(0), i32(0), x, x.to(torch.bfloat16)), lambda: cache.append(i32(0), i32(0), x.half(), x.half()),
                 lambda: cache.append(i32(0).cpu(), i32(0), x, x), lambda: cache.append(i32(0), i32(0), x.cpu(), x.cpu()),
                 lambda: cache.append(i32(0), i32(0), torch.zeros((1, 256), device="cuda")[:, ::2], x),
                 lambda: cache.gather(i32(0), i32(0), -1), lambda: cache.gather(i32(0), i32(0), 1, dtype=torch.float16), lambda: cache.gather(i32(0), i32(), 1),
                 lambda: cache.decode(q.float(), num_heads=8), lambda: cache.decode(q, num_heads=4), lambda: cache.decode(q.cpu(), num_heads=8),
                 lambda: cache.decode(torch.zeros((1, 32, 64), dtype=torch.bfloat16, device="cuda"), num_heads=32),       # 16 heads a key head
                 lambda: cache.decode(torch.zeros((1, 3, 64), dtype=torch.bfloat16, device="cuda"), num_heads=3),
                 lambda: cache.decode(torch.zeros((1, 8, 32), dtype=torch.bfloat16, device="cuda"), num_heads=8),
                 lambda: cache.decode(q, num_heads=8, seq_lens=i32(1, 2)), lambda: cache.decode(q, num_heads=8, page_table=cache.page_table[:0]),
                 lambda: cache.decode(q, num_heads=8, max_seq_len=10000), lambda: cache.decode(q, num_heads=8, chunk_tokens=100),
                 lambda: cache.decode(q, num_heads=8, lse=torch.zeros((1, 7), device="cuda")), lambda: cache.decode(q, num_heads=8, q_positions=i32(1, 2))):
        with pytest.raises(RuntimeError):
            call()
