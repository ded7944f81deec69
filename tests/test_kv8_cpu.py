"""CPU tests of the 8-bit KV cache: the float64 oracle's format against PyTorch's float8, the scale
rule, and what the C ABI and the host classes refuse before they touch a device."""
import ctypes

import numpy as np
import pytest
import torch


def test_oracle_e4m3_matches_torch_float8():
    from oracle.kv8 import e4m3
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    finite = codes[np.isfinite(codes)]
    assert np.array_equal(e4m3(finite), finite)  # every e4m3 value is its own nearest
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 10.0 ** rng.integers(-5, 3, 20000),
                        (np.sort(finite)[1:] + np.sort(finite)[:-1]) / 2]).astype(np.float32)  # ties among them
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(e4m3(x), want)
    assert e4m3(1e9) == 448.0 and e4m3(-np.inf) == -448.0 and np.isnan(e4m3(np.nan))


def test_oracle_scale_is_the_smallest_power_of_two():
    from oracle.kv8 import scale_of
    for amax in [0.0, 1e-38, 448.0, np.nextafter(448.0, 449), 1.0, 0.875, 1.75, 1.7500001, 3e38] + list(np.abs(np.random.default_rng(1).standard_normal(50))):
        s = scale_of(float(amax))
        assert np.frexp(s)[0] == 0.5 and s >= 2.0 ** -120
        assert amax <= 448 * s
        assert s == 2.0 ** -120 or amax > 448 * (s / 2)


def _desc(**kw):
    from jax4j_b200._lib import Kv8CacheDesc
    d = dict(k=1 << 20, v=1 << 21, k_scale=1 << 22, v_scale=1 << 23, layers=1, pages=4, kv_heads=2, page=32, head_dim=128)
    d.update(kw)
    return ctypes.byref(Kv8CacheDesc(*d.values()))


@pytest.mark.parametrize("kw,match", [
    (dict(head_dim=96), "head_dim must be 64 or 128"), (dict(page=24), "multiple of 16"), (dict(page=0), "multiple of 16"),
    (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "must be positive"), (dict(pages=1 << 40), "2\\^31"),
    (dict(k=(1 << 20) + 8), "16-byte aligned"), (dict(v_scale=0), "aligned")])
def test_abi_refuses_bad_cache_descriptions(kw, match):
    from jax4j_b200._lib import call
    with pytest.raises(ValueError, match=match):
        call("j4b_kv8_copy_pages", _desc(**kw), 0, None, None, None, None)


def test_abi_refuses_a_null_cache_and_a_bad_layer():
    from jax4j_b200._lib import call
    with pytest.raises(ValueError, match="null cache"):
        call("j4b_kv8_copy_pages", None, 0, None, None, None, None)
    with pytest.raises(ValueError, match="layer 1 outside"):
        call("j4b_kv8_append", _desc(), 1, 0, 0, 0, 2, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, None)


def test_cache_wrap_checks_shapes():
    from jax4j_b200.kv8 import Kv8Cache

    def codes(*s):
        return torch.zeros(s, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ok = (codes(1, 3, 2, 32, 64), codes(1, 3, 2, 32, 64), torch.zeros(1, 3, 2, 2), torch.zeros(1, 3, 2, 2))
    assert Kv8Cache.wrap(*ok).page == 32
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Kv8Cache.wrap(ok[0].view(torch.uint8), *ok[1:])
    with pytest.raises(ValueError, match="multiple of 16"):
        Kv8Cache.wrap(codes(1, 3, 2, 24, 64), codes(1, 3, 2, 24, 64), *ok[2:])
    with pytest.raises(ValueError, match="head_dim"):
        Kv8Cache.wrap(codes(1, 3, 2, 32, 96), codes(1, 3, 2, 32, 96), *ok[2:])
    with pytest.raises(ValueError, match="scales"):
        Kv8Cache.wrap(*ok[:2], torch.zeros(1, 3, 2, 32), ok[3])
    with pytest.raises(ValueError, match="contiguous"):
        Kv8Cache.wrap(*ok[:3], torch.zeros(1, 3, 2, 4)[..., ::2])


def test_rope_table_holds_cos_and_sin():
    from jax4j_b200.kv8 import rope_table
    t = rope_table(50, 64, 500.0).double().numpy()
    ang = np.arange(50)[:, None] * 500.0 ** (-2.0 * np.arange(32) / 64)
    assert np.abs(t[..., 0] - np.cos(ang)).max() < 1e-7 and np.abs(t[..., 1] - np.sin(ang)).max() < 1e-7
