"""What the 8-bit cache and sampling refuse before anything reaches a GPU, and the layout that the tests themselves use."""
import pytest
import torch

import kv8_cases as K


def test_layout_round_trip():
    g = torch.Generator().manual_seed(0)
    for values in ("e4m3", "int8"):
        k, v = (torch.randint(-100, 101, (3, 2, 16, 64), generator=g).float().to(torch.float8_e4m3fn if values == "e4m3" else torch.int8).float().double()
                for _ in range(2))
        ks, vs = (2.0 ** torch.randint(-5, 5, (3, 2, 16), generator=g).double() for _ in range(2))
        pool = K.packed(k, v, ks, vs, values)
        assert pool.shape == (3, 2, 2112) and all(torch.equal(a, b) for a, b in zip(K.unpacked(pool, values), (k, v, ks, vs)))
    places = K.v_places()
    assert all(sorted(row.tolist()) == list(range(64)) for row in places)
    # eight neighbouring tokens' pieces of 16 bytes lie in different 16-byte columns of two rows of 64
    for c in range(4):
        assert len({(t % 2, int(places[t, 16 * c]) // 16) for t in range(8)}) == 8


def test_cache_refuses(lib):
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    make = lambda **kw: QuantizedKVCache(4, 2, 2, 2, device="cpu", **kw)      # noqa: E731
    for kw in ({"values": "fp8"}, {"head_dim": 128}, {"storage": (torch.zeros((4, 2, 2112)), torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))},
               {"storage": (torch.zeros((4, 2, 2048), dtype=torch.uint8), torch.zeros((2, 2), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))}):
        with pytest.raises(RuntimeError):
            make(**kw)
    cache, i = make(), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: cache.append(i, i, torch.zeros(1, 128), torch.zeros(1, 128)), lambda: cache.gather(i, i, 1),
                 lambda: cache.decode(torch.zeros(1, 8, 64, dtype=torch.bfloat16), num_heads=8)):
        with pytest.raises(RuntimeError, match="only GPU"):
            call()


def test_products_that_append_refuse_it(lib):
    """They write the bf16 cache's blocks, which are larger"""
    from baranet_bdml_b200 import ops
    from baranet_bdml_b200.kv_cache import QuantizedKVCache
    cache, i, x, w = QuantizedKVCache(4, 1, 2, 2, device="cpu"), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 256).bfloat16(), torch.zeros(768, 256).bfloat16()
    for call in (lambda: ops.gemm_qkv_append_bf16_skinny(x, w, cache, i, i, 8), lambda: ops.gemm_qkv_rope_bf16(x, w, 1, 1, 8, 2, 64, None, cache=cache)):
        with pytest.raises(RuntimeError, match="bf16 cache"):
            call()


def test_status_codes(lib):
    """The C entries check their arguments before they look for a device"""
    from baranet_bdml_b200 import _lib
    bad, none = _lib.BN_ERR_INVALID_ARG, _lib.BN_ERR_UNSUPPORTED
    p = 4096                                               # an address that is never read
    append = lambda pool=p, pages=4, seqs=2, width=2, T=1, dtype=1, values=0, rotate=1, hkv=2, d=64, theta=10000.0: lib.bn_kv8_append(      # noqa: E731
        pool, pages, p, seqs, width, p, p, T, p, 128, p, 128, dtype, values, rotate, hkv, d, theta, None)
    gather = lambda pool=p, n=1, tokens=1, dtype=1, values=0, out=p, d=64: lib.bn_kv8_gather(pool, 4, p, 2, 2, p, p, p, n, tokens, out, p, dtype, values, 2, d, None)      # noqa: E731
    decode = lambda q=p, pool=p, out=p, values=0, B=1, hq=8, hkv=2, d=64, longest=32, chunk=0, ws=p, n=1 << 30, width=2, theta=10000.0: lib.bn_attn_decode_kv8(      # noqa: E731
        q, pool, 4, p, width, p, None, out, None, None, values, B, hq, hkv, d, 0.125, theta, 1, longest, chunk, ws, n, None)
    sample = lambda x=p, u=p, out=p, stride=100, dtype=0, t=1.0, k=0, tp=1.0, mp=0.0, rows=1, cols=100: lib.bn_sample_rows(      # noqa: E731
        x, stride, dtype, u, None, t, None, k, None, tp, None, mp, out, rows, cols, None)
    for code, calls in ((bad, [append(pool=None), append(pool=p + 8), append(pages=0), append(seqs=0), append(width=0), append(T=-1), append(dtype=2), append(values=2),
                               append(hkv=0), append(theta=0.0), gather(pool=None), gather(n=-1), gather(tokens=-1), gather(dtype=3), gather(out=None), gather(out=p + 4),
                               gather(values=-1), decode(q=None), decode(out=None), decode(values=5), decode(B=-1), decode(chunk=100), decode(longest=33),
                               decode(pool=p + 4), decode(q=p + 2), decode(theta=-1.0), sample(x=None), sample(u=None), sample(out=None), sample(stride=99),
                               sample(dtype=2), sample(t=-1.0), sample(t=float("nan")), sample(t=float("inf")), sample(k=-1), sample(tp=1.1), sample(tp=float("nan")),
                               sample(mp=-0.5), sample(rows=-1), sample(cols=0)]),
                        (none, [append(d=128), gather(d=32), decode(d=128), decode(hq=7), decode(hq=18), decode(B=1025), sample(cols=1 << 21, stride=1 << 21)])):
        assert all(c == code for c in calls), calls
    assert lib.bn_attn_decode_kv8_workspace_bytes(1, 8, 2, 32, 100, 0) == 0 and lib.bn_attn_decode_kv8_workspace_bytes(64, 32, 4, 64, 4096, 0) > 0


def test_sizes_whose_products_overflow(lib):
    from baranet_bdml_b200 import _lib
    p, most = 4096, 2 ** 31 - 1
    assert lib.bn_kv8_gather(p, 4, p, 2, 2, p, p, p, most, most, p, p, 1, 0, 4, 64, None) == _lib.BN_ERR_INVALID_ARG
    assert lib.bn_kv8_append(p, 4, p, 2, 2, p, p, most, p, 128, p, 128, 1, 0, 1, 64, 64, 1e4, None) == _lib.BN_ERR_INVALID_ARG
    for B, hkv, longest in ((1024, 1 << 16, 16), (1024, 4, 1 << 30), (1, 1, most)):
        assert lib.bn_attn_decode_kv8(p, p, 4, p, most, p, None, p, None, None, 0, B, hkv, hkv, 64, 0.125, 1e4, 1, longest, 0, p, 1 << 30, None) == _lib.BN_ERR_UNSUPPORTED


def test_choice_by_hand():
    """The plain form of the choice itself"""
    x = [2.0, 1.0, 2.0, 0.0]
    import numpy as np
    x = np.log(np.array([4.0, 1.0, 4.0, 1.0]))
    pick = lambda u, **kw: K.choose(x, u, **kw)      # noqa: E731
    assert [pick(u) for u in (0.0, 0.39, 0.41, 0.49, 0.51, 0.89, 0.91)] == [0, 0, 1, 1, 2, 2, 3]
    assert [pick(u, top_k=3) for u in (0.43, 0.45, 0.56, 0.99)] == [0, 1, 2, 2]
    assert [pick(u, top_p=0.7) for u in (0.49, 0.51)] == [0, 2] and pick(0.99, top_p=0.3) == 0
    assert [pick(u, min_p=0.5) for u in (0.49, 0.51)] == [0, 2] and pick(0.9, temperature=0) == 0
