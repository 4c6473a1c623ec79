"""Marks of values that are not finite (they send a head's 16-bit tokens down a
slower path of the attention): set for the head that has one, gone once its
sequence begins anew, and right outputs throughout."""
import importlib

import pytest
import torch

from oracle import kv8 as ok

pytestmark = pytest.mark.gpu
DEV = "cuda"
pkg = importlib.import_module("numerics-and-sparse-attn_b200")
GROUP, D = 2, 64


def _lens(*x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def _check(cache, q, k, v, n):
    o = cache.attend(q)
    for b in range(2):
        ref, spread, reach = ok.attend(q[b][:, None], ok.held(k[b], n, "e4m3"), ok.held(v[b], n, "e4m3"), 1, D ** -0.5)
        nan = torch.isnan(ref[:, 0])
        assert torch.equal(torch.isnan(o[b]), nan)
        far = (o[b].double() - ref[:, 0]).abs() - ok.bound(ref, spread, reach, q.dtype, D)[:, 0]
        assert far[~nan].max().item() <= 0
    assert pkg.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("begin", ["truncate", "step", "prompt", "adopt"])
@pytest.mark.parametrize("hkv", [1, 3, 32, 40])
@pytest.mark.parametrize("n", [40, 100])  # tokens; with 100 the kernel of whole blocks
def test_marks_go_when_a_sequence_begins_anew(n, hkv, begin):
    g = torch.Generator(device=DEV).manual_seed(70)
    k, v = torch.randn(2, 2, hkv, n, D, device=DEV, generator=g).half()
    q = torch.randn(2, hkv * GROUP, D, device=DEV, generator=g).half()
    h, bad = hkv - 1, v.clone()
    bad[1, h, n - 1, 5] = float("inf")
    cache = pkg.Kv8Cache(2, hkv, 256, head_dim=D, device=DEV)
    for _ in range(2):  # a second time over what the first left
        cache.append(k, bad, starts=_lens(0, 0))
        assert cache._unclean.tolist() == [0, torch.tensor(1 << (h & 31)).int().item()]
        _check(cache, q, k, bad, n)
        if begin == "truncate":
            cache.truncate(_lens(0, 0))
        elif begin == "adopt":
            cache.adopt(_lens(0, 0))
        if begin == "step":
            cache.append(k[:, :, 0], v[:, :, 0], starts=_lens(0, 0))
            cache.append(k[:, :, 1:], v[:, :, 1:])
        else:
            cache.append(k, v, starts=_lens(0, 0))
        if hkv <= 32 or begin == "adopt":
            assert cache._unclean.tolist() == [0, 0]
        _check(cache, q, k, v, n)


def test_marks_stay_while_the_ring_can_hold_the_value():
    """Not where tokens before the start are still in the ring: going back and on keeps them."""
    g = torch.Generator(device=DEV).manual_seed(71)
    k, v = torch.randn(2, 2, 2, 150, D, device=DEV, generator=g).half()
    q = torch.randn(2, 2 * GROUP, D, device=DEV, generator=g).half()
    v[0, 1, 70, 3] = float("nan")
    cache = pkg.Kv8Cache(2, 2, 256, head_dim=D, device=DEV)
    cache.append(k[:, :, :100], v[:, :, :100])
    cache.append(k[:, :, 100:], v[:, :, 100:])  # completes its block
    _check(cache, q, k, v, 150)
    cache.truncate(_lens(128, 128))
    cache.truncate(_lens(71, 71))
    assert cache._unclean.tolist() == [2, 0]
    _check(cache, q, k, v, 71)
    cache.truncate(_lens(70, 70))
    _check(cache, q, k, v, 70)
    cache.append(k[:, :, 70:90], v[:, :, 70:90])
    _check(cache, q, k, v, 90)
