"""CPU: the cache's geometry and refusals, the entry points' checks, and the oracle's pins."""
import ctypes
import math

import pytest
import torch

from oracle import kvcache as ok
from vdn_amd import _lib
from vdn_amd import kvcache as kv


def test_cache_geometry():
    c = kv.empty_cache(5, 3, 128, 32, device="cpu")
    assert (c.pages, c.kv_heads, c.page, c.head_dim) == (5, 3, 32, 128)
    assert c.v_codes.shape == (5, 3, 128, 32) and c.faults.tolist() == [0]
    c.check()
    for args in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 96, 16), (1, 1, 64, 24), (1.0, 1, 64, 16)):
        with pytest.raises(ValueError):
            kv.empty_cache(*args, device="cpu")
    for i, bad in ((0, c.v_codes), (2, c.k_codes), (1, c.k_scales[:4]), (3, c.v_scales.int()),
                   (4, c.faults.long()), (4, torch.zeros(2, dtype=torch.int32)),
                   (0, c.k_codes.transpose(0, 1).contiguous().transpose(0, 1))):
        parts = [c.k_codes, c.k_scales, c.v_codes, c.v_scales, c.faults]
        parts[i] = bad
        with pytest.raises(ValueError):
            kv.KVCache(*parts)


def test_calls_need_a_device():
    c = kv.empty_cache(2, 1, 64, 16, device="cpu")
    x, t, n = torch.zeros(1, 1, 64).bfloat16(), torch.zeros(1, 1).int(), torch.zeros(1).int()
    with torch.no_grad():
        for call in (lambda: kv.write_cache(c, x, x, t, n), lambda: kv.read_cache(c, t, n, None, 1),
                     lambda: kv.cache_attention(x, c, t, n)):
            with pytest.raises(ValueError, match="CUDA"):
                call()


def test_no_stream_of_a_host_device():
    with pytest.raises(ValueError, match="device"):
        _lib.stream(torch.device("cpu"))


def test_entry_points_validate_before_launching():
    lib, p = _lib.load(), 1 << 20

    def cache(pages=4, heads=2, page=16, dim=64, codes=p):
        return (codes, p, p, p, p, pages, heads, page, dim)

    def move(fn, c=cache(), table=p, batch=2, width=2, starts=p, key=p, k_st=128, rows=2, dtype=0):
        return fn(*c, table, 2, batch, width, starts, None, key, k_st, 64, p, 128, 64, rows, dtype, None)

    def attend(c=cache(), q=p, width=2, batch=2, tokens=1, group=1, dtype=0, scale=0.1, q_st=128, ws=p,
               nbytes=1 << 30):
        return lib.vdn_cache_attention(q, 128, q_st, 64, *c, p, 2, batch, width, p, tokens, group, dtype,
                                       scale, p, 128, 128, 64, None, ws, nbytes, None)

    bad_caches = [cache(pages=0), cache(heads=0), cache(page=8), cache(page=48), cache(page=512), cache(dim=96)]
    for fn in (lib.vdn_cache_write, lib.vdn_cache_read):
        for c in bad_caches:
            assert move(fn, c) != 0 and b"geometry" in lib.vdn_last_error()
        for change, word in ((dict(dtype=2), b"dtype"), (dict(rows=-1), b"geometry"), (dict(batch=-1), b"geometry"),
                             (dict(c=cache(codes=None)), b"null"), (dict(key=None), b"null"),
                             (dict(starts=None), b"null"), (dict(table=None), b"null"),
                             (dict(k_st=132), b"16-byte"), (dict(key=p + 2), b"16-byte"),
                             (dict(c=cache(heads=1 << 30)), b"too many")):
            assert move(fn, **change) != 0, change
            assert word in lib.vdn_last_error(), change
        assert move(fn, rows=0, key=None) == 0
    for c in bad_caches:
        assert attend(c) != 0 and b"geometry" in lib.vdn_last_error()
    for change, word in ((dict(width=0), b"geometry"), (dict(tokens=0), b"geometry"), (dict(group=0), b"geometry"),
                         (dict(width=1 << 28), b"geometry"), (dict(dtype=3), b"dtype"),
                         (dict(scale=math.nan), b"scale"), (dict(q=None), b"null"),
                         (dict(q_st=4), b"16-byte"), (dict(batch=1 << 30, group=4), b"too many")):
        assert attend(**change) != 0, change
        assert word in lib.vdn_last_error(), change
    assert attend(batch=0, q=None) == 0
    out = ctypes.c_int64(0)
    assert lib.vdn_cache_attention_workspace(1, 1, 64, None) != 0
    assert lib.vdn_cache_attention_workspace(0, 1, 64, ctypes.addressof(out)) != 0


def test_oracle_rounds_as_e4m3():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    finite = codes[torch.isfinite(codes)]
    assert torch.equal(ok.nearest(finite), finite)
    x = torch.randn(20000, generator=torch.Generator().manual_seed(0)).double() * 30
    assert torch.equal(ok.nearest(x), x.float().to(torch.float8_e4m3fn).double())
    mid = (finite.sort().values[1:] + finite.sort().values[:-1]) / 2       # ties to even
    assert torch.equal(ok.nearest(mid), mid.float().to(torch.float8_e4m3fn).double())
    assert ok.nearest(torch.tensor([math.inf, math.nan])).isnan().all()


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.0001, 1), (224.0, -1), (1.0, -8), (0.0, -100),
                                    (1e-40, -100), (1.75 * 2.0 ** 127, 119), (3.3e38, 120)])
def test_oracle_exponent(amax, e):
    assert ok.exponent(amax) == e
    assert amax <= 448 * 2.0 ** e and (e == -100 or amax > 448 * 2.0 ** (e - 1))


def test_oracle_append_keeps_the_larger_scale():
    c = ok.Cache(1, 1, 16, 64)
    x = torch.full((3, 1, 64), 1.0)
    c.write(x, x, [[0]], [0], [3])
    c.write(x * 1000, x / 1000, [[0]], [3], [1])
    assert c.exponents[0][0, 0] == 2 and c.exponents[1][0, 0] == -8
    assert (c.values[0][0, 0, :3] == 1.0).all() and (c.values[0][0, 0, 3] == 1024.0).all()
    assert (c.values[1][0, 0, 3] == ok.nearest(torch.tensor(0.256)) * 2.0 ** -8).all()
