"""The 8-bit paged KV cache (Kv8Cache / nsa_kv8_*) against its oracle: codes,
scales and ring bit for bit, attention within bounds derived in oracle/kv8.py
(the sum of its roundings), over types, head layouts, lengths, masks, strides,
page orders, ragged calls, rewinds, streams, graphs and bad inputs."""
import importlib

import pytest
import torch

from oracle import kv8 as ok

pytestmark = pytest.mark.gpu
DEV = "cuda"
pkg = importlib.import_module("numerics-and-sparse-attn_b200")
F16, BF16 = torch.float16, torch.bfloat16


def _tokens(b, h, n, d, dtype, seed, factor=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    k = torch.randn(b, h, n, d, device=DEV, generator=g)
    k[..., ::37] *= 8.0
    v = torch.randn(b, h, n, d, device=DEV, generator=g)
    return (k * factor).to(dtype), (v * factor).to(dtype)


def _queries(b, h, t, d, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed + 7777)
    return torch.randn(b, h, t, d, device=DEV, generator=g).to(dtype)


def _fill(cache, k, v, lens):
    """Prompts of lens[b] tokens in one ragged append."""
    n = max(max(lens), 1)
    cache.append(k[:, :, :n], v[:, :, :n], counts=torch.tensor(lens, device=DEV))


def _clean():
    torch.cuda.synchronize()
    assert pkg.device_error(torch.device(DEV)) == 0


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


def _check_state(cache, k, v, lens):
    """Codes, scales, ring (of the incomplete block) and lengths, bit for bit."""
    assert cache.lens.tolist() == list(lens)
    for b, n in enumerate(lens):
        full = n // 64
        for c, (x, codes, ring) in enumerate(((k, cache.k_codes, cache.k_ring), (v, cache.v_codes, cache.v_ring))):
            if full:
                want, scale = ok.quantize_blocks(x[b, :, :full * 64].reshape(x.shape[1], full, 64, -1), cache.codes)
                pages = cache.page_table[b, :full].long()
                got = codes.view(torch.uint8)[pages].view(codes.dtype).float().transpose(0, 1)
                assert _same(got, want), (b, n)
                assert _same(cache.scales[pages][..., c].transpose(0, 1), scale), (b, n)
            slots = torch.arange(full * 64, n, device=DEV) % 128
            tail = x[b, :, full * 64:n]
            assert _same(ring[b, :, slots], torch.where(torch.isfinite(tail), tail, float("nan"))), (b, n)


def _check_attend(cache, o, q, k, v, lens, counts=None, window=None, sink=4, scale=None):
    """o, q [B, H, T, D]; the history k, v."""
    t, d = q.shape[2], q.shape[3]
    scale = d ** -0.5 if scale is None else scale
    assert o.shape == q.shape and o.dtype == q.dtype
    for b, n in enumerate(lens):
        cnt = t if counts is None else counts[b]
        ref, spread, reach = ok.attend(q[b], ok.held(k[b], n, cache.codes), ok.held(v[b], n, cache.codes), cnt, scale,
                                       window, sink)
        got = o[b].double()
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(got), nan), (b, n)
        lim = ok.bound(ref, spread, reach, q.dtype, d)
        far = ((got - ref).abs() - lim)[~nan]
        assert far.numel() == 0 or far.max().item() <= 0, (b, n, far.max().item(), (got - ref).abs()[~nan].max().item())


CASES = [  # batch lengths, Hkv, group, D, dtype, codes
    ([1, 63, 64, 65, 127, 128, 129, 500], 8, 8, 128, F16, "e4m3"),
    ([1000, 0, 5, 4097], 2, 4, 128, BF16, "int8"),
    ([300, 31, 33, 700], 3, 1, 64, F16, "int8"),
    ([777, 64], 1, 16, 64, BF16, "e4m3"),
    ([130, 2500], 2, 7, 128, F16, "int8"),
    ([640], 1, 40, 128, BF16, "e4m3"),
]


@pytest.mark.parametrize("lens,hkv,group,d,dtype,codes", CASES)
def test_prompt_state_read_and_attend(lens, hkv, group, d, dtype, codes):
    b, n = len(lens), max(lens)
    k, v = _tokens(b, hkv, n, d, dtype, 1)
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, dtype=dtype, codes=codes, device=DEV)
    _fill(cache, k, v, lens)
    _clean()
    _check_state(cache, k, v, lens)
    for out in (dtype, torch.float32):
        rk, rv = cache.read(n, dtype=out)
        for i, ln in enumerate(lens):
            for got, x in ((rk, k), (rv, v)):
                want = ok.held(x[i], ln, codes).to(torch.float32).to(out)  # scale * code: one float32 rounding, then the type's
                assert torch.equal(got[i, :, :ln], want) and not got[i, :, ln:].any()
    q = _queries(b, hkv * group, 1, d, dtype, 3)
    o = cache.attend(q[:, :, 0])
    _clean()
    _check_attend(cache, o[:, :, None], q, k, v, lens)
    assert torch.equal(cache.attend(q)[:, :, 0], o)  # the form with T = 1, and the same bits again
