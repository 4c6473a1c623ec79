"""Softmax weights of the 8-bit cache's attention (Kv8Cache.attend) where the
precision that they are held in shows: each weight's own output element, within
half a step of the output's type, and long tails of small weights beside one
large weight whose value is 0.

Queries have one element other than 0, so that a score is one product and has
no rounding of a sum of D of them.  Its roundings in float32, each at most
2^-24 of it: of scale * log2(e) (two), of the block's and the query's scale
(two), of the product, of the distance to the maximum; a weight moves by twice
6 * 2^-24 * |score| (numerator and denominator) at most."""
import importlib

import pytest
import torch

from oracle import kv8 as ok

pytestmark = pytest.mark.gpu
DEV = "cuda"
pkg = importlib.import_module("numerics-and-sparse-attn_b200")
F16, BF16 = torch.float16, torch.bfloat16


def _half_step(x, dtype):
    """Half the distance of the type's numbers around x, element by element."""
    fi = torch.finfo(dtype)
    _, e = torch.frexp(x.abs().clamp_min(fi.smallest_normal))
    return torch.ldexp(torch.full_like(x, fi.eps / 4), e)  # x = f 2^e, 0.5 <= f < 1


@pytest.mark.parametrize("wide", [1, 8])  # scores within 4 and 32 of one another
@pytest.mark.parametrize("n", [64, 63])  # a block of codes; the 16-bit tokens
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_every_weight_is_right_to_half_a_step_of_the_output(dtype, codes, n, wide):
    """V is the unit matrix: output element j is token j's weight.  A weight held in as many bits as the output adds
    errors of its own and misses the nearest number at every tenth element or so."""
    b, hkv, group, d = 24, 2, 4, 64
    g = torch.Generator(device=DEV).manual_seed(50)
    k, v = torch.zeros(2, b, hkv, n, d, dtype=dtype, device=DEV)
    k[..., 0] = (wide * (2 * torch.rand(b, hkv, n, device=DEV, generator=g) - 1)).to(dtype)
    v[...] = torch.eye(d, device=DEV)[:n].to(dtype)
    q = torch.zeros(b, hkv * group, d, dtype=dtype, device=DEV)
    q[..., 0] = (0.5 + 1.5 * torch.rand(b, hkv * group, device=DEV, generator=g)).to(dtype)
    cache = pkg.Kv8Cache(b, hkv, 64, head_dim=d, dtype=dtype, codes=codes, device=DEV)
    cache.append(k, v)
    o = cache.attend(q, sm_scale=1.0)
    for i in range(b):
        kk, vv = ok.held(k[i], n, codes), ok.held(v[i], n, codes)
        ref, spread, reach = ok.attend(q[i][:, None], kk, vv, 1, 1.0)
        # weights in two parts (2^-18 where they are bfloat16; at least 2^-40 of the largest in fp16 ones), the
        # exponentials and sums 2^-20 each
        rel = 2 * 6 * 2.0 ** -24 * reach + 2.0 ** -18 + 2 * 2.0 ** -20
        far = (o[i].double() - ref[:, 0]).abs() - _half_step(ref, dtype)[:, 0] - (rel * spread)[:, 0] - 2.0 ** -40
        assert far.max().item() <= 0, (i, far.max().item(), (far > 0).double().mean().item())
    assert pkg.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("above", [10, 16, 20, 24])  # of the mean, in units of the exponent
@pytest.mark.parametrize("dtype,codes", [(F16, "e4m3"), (F16, "int8"), (BF16, "e4m3"), (BF16, "int8")])
@pytest.mark.parametrize("place", [0, 4000, -1])  # in the first block, in the middle, among the 16-bit tokens
@pytest.mark.parametrize("b,hkv,n,wide", [(64, 32, 8192 + 40, 0.0), (64, 32, 4096 + 7, 2.0), (1, 2, 70_000, 0.0)])
def test_a_long_tail_beside_one_large_weight(b, hkv, n, wide, place, dtype, codes, above):
    """An attention sink: one token far above the rest, its value 0, so the output is the tail's.  With 64 x 32 units
    most workers take a whole one; the long ones are cut into many pieces."""
    d = 64
    g = torch.Generator(device=DEV).manual_seed(51)
    k, v = torch.zeros(2, 1, 1, n, d, dtype=dtype, device=DEV)
    k[0, 0, :, 0] = (wide * torch.randn(n, device=DEV, generator=g)).to(dtype)
    k[0, 0, place, 0] = above
    v[0, 0] = (1 + 0.25 * torch.randn(n, d, device=DEV, generator=g)).to(dtype)
    v[0, 0, place] = 0
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, dtype=dtype, codes=codes, device=DEV)
    cache.append(k.expand(b, hkv, n, d), v.expand(b, hkv, n, d))
    q = torch.zeros(b, hkv, d, dtype=dtype, device=DEV)
    q[..., 0] = 1
    o = cache.attend(q, sm_scale=1.0)
    ref, spread, reach = ok.attend(q[0, :1, None], ok.held(k[0], n, codes), ok.held(v[0], n, codes), 1, 1.0)
    # Sums: a lane adds every eighth token to the denominator, a sum of the numerator is added to once in 32 tokens
    # with four roundings of its own; the weights in two parts (2^-18 where they are bfloat16).
    rel = 2 * 6 * 2.0 ** -24 * reach + (n / 8 + n / 8) * 2.0 ** -24 + 2.0 ** -18 + 2 * 2.0 ** -20
    # In the 32 tokens that the large weight (at most 1) is among, the others' have an absolute error of 2^-40 of it.
    near = 32 * 2.0 ** -40 * v.abs().max().item()
    far = (o[:, :, None].double() - ref).abs() - _half_step(ref, dtype) - rel * spread - near
    assert far.max().item() <= 0, (far.max().item(), ((o[:, :, None].double() - ref) / ref).abs().max().item())
    assert pkg.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("d,dtype,codes", [(64, F16, "e4m3"), (128, F16, "int8"), (64, BF16, "int8"), (128, BF16, "e4m3")])
@pytest.mark.parametrize("large", [2.0 ** 10, 65504.0, 2.0 ** 18])
def test_small_query_elements_beside_a_large_one(d, dtype, codes, large):
    """A query channel far above the others, where the keys are 0: scores are the others' alone, exact to their own
    roundings (elements 2^-19 to 2^-30 of their row's largest; float16 ends at 65504)."""
    if dtype == F16 and large > 65504:
        return
    b, hkv, group, n = 4, 2, 4, 100
    small = 2.0 ** -9 if dtype == F16 else 2.0 ** -10
    g = torch.Generator(device=DEV).manual_seed(52)
    k, v = torch.randn(2, b, hkv, n, d, device=DEV, generator=g).to(dtype)
    k[..., 0] = 0
    q = (small * torch.randn(b, hkv * group, d, device=DEV, generator=g)).to(dtype)
    q[..., 0] = large
    scale = 2.0 / (small * d ** 0.5)
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, dtype=dtype, codes=codes, device=DEV)
    cache.append(k, v)
    o = cache.attend(q, sm_scale=scale)
    for i in range(b):
        ref, spread, reach = ok.attend(q[i][:, None], ok.held(k[i], n, codes), ok.held(v[i], n, codes), 1,
                                       torch.tensor(scale, dtype=torch.float32).item())
        far = (o[i].double() - ref[:, 0]).abs() - ok.bound(ref, spread, reach, dtype, d)[:, 0]
        assert far.max().item() <= 0, (i, far.max().item())
    assert pkg.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("dtype,factor", [(F16, 2.0 ** -20), (F16, 2.0 ** 12), (BF16, 2.0 ** -126), (BF16, 2.0 ** -100), (BF16, 2.0 ** 123)])
def test_queries_at_the_ends_of_their_range(dtype, factor):
    """Rows whose largest element is among the smallest or largest numbers of the type (also subnormal ones), and zeros."""
    b, hkv, group, n, d = 2, 2, 4, 100, 64
    g = torch.Generator(device=DEV).manual_seed(53)
    k, v = torch.randn(2, b, hkv, n, d, device=DEV, generator=g).to(dtype)
    q = (factor * torch.randn(b, hkv * group, d, device=DEV, generator=g)).to(dtype)
    q[:, 1] = 0
    scale = torch.tensor(0.25 / factor, dtype=torch.float32).item()
    assert 0 < scale < float("inf")
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, dtype=dtype, device=DEV)
    cache.append(k, v)
    o = cache.attend(q, sm_scale=scale)
    for i in range(b):
        ref, spread, reach = ok.attend(q[i][:, None], ok.held(k[i], n, "e4m3"), ok.held(v[i], n, "e4m3"), 1, scale)
        far = (o[i].double() - ref[:, 0]).abs() - ok.bound(ref, spread, reach, dtype, d)[:, 0]
        assert far.max().item() <= 0, (i, far.max().item())
    assert pkg.device_error(torch.device(DEV)) == 0
