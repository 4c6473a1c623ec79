"""The 8-bit paged KV cache without a GPU: the oracle against its definition in
exact arithmetic, the constructor's refusals, and the C entries' checks, which
come before any CUDA call."""
import ctypes
import importlib
from fractions import Fraction

import pytest
import torch

from oracle import kv8 as ok

PKG = importlib.import_module("numerics-and-sparse-attn_b200")
KV8 = importlib.import_module("numerics-and-sparse-attn_b200.kv8")
LIB = importlib.import_module("numerics-and-sparse-attn_b200._lib")


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_oracle_codes_are_the_nearest(codes, dtype):
    """Every code is a nearest one of x * fl(1 / s), s the block's largest over the largest code."""
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(1, 64, 64, generator=g) * torch.tensor([1e-3, 1.0, 30.0, 8.0]).repeat(16)).to(dtype)
    c, s = ok.quantize_blocks(x, codes)
    top = ok.TOP[codes]
    assert abs(Fraction(s.item()) * int(top) / Fraction(x.abs().max().item()) - 1) < Fraction(1, 2 ** 23)
    values = torch.arange(-127, 128).float() if codes == "int8" else \
        torch.arange(256).to(torch.uint8).view(torch.float8_e4m3fn).float()
    values = sorted({v for v in values.tolist() if v == v})
    inv = (1.0 / s).item()
    for xi, ci in list(zip(x.flatten().tolist(), c.flatten().tolist()))[::7]:
        y = torch.tensor(xi, dtype=torch.float32).mul(torch.tensor(inv, dtype=torch.float32)).item()
        assert abs(ci - y) <= min(abs(v - y) for v in values)


def test_oracle_attention_is_softmax_over_what_is_seen():
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(2, 90, 64, generator=g).half() for _ in range(2))
    q = torch.randn(4, 3, 64, generator=g).half()
    kk, vv = ok.held(k, 90, "int8"), ok.held(v, 90, "int8")
    assert torch.equal(kk[:, 64:], k[:, 64:].double()) and not torch.equal(kk[:, :64], k[:, :64].double())
    o, _, _ = ok.attend(q, kk, vv, 2, 0.125, window=20, sink=4)
    assert not o[:, 2].any()  # the third row is behind the count
    for i, pos in ((0, 88), (1, 89)):
        see = [p for p in range(pos + 1) if p < 4 or p > pos - 20]
        for h in range(4):
            s = torch.tensor([float(q[h, i].double() @ kk[h // 2, p]) * 0.125 for p in see], dtype=torch.float64)
            w = torch.exp(s - s.max())
            want = sum(w[j] * vv[h // 2, p] for j, p in enumerate(see)) / w.sum()
            torch.testing.assert_close(o[h, i], want, rtol=1e-12, atol=1e-13)


def test_constructor_refusals():
    with pytest.raises(ValueError, match="CUDA device"):
        PKG.Kv8Cache(1, 1, 10, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        PKG.Kv8Cache(1, 1, 10, head_dim=96, device="cpu")
    with pytest.raises(TypeError, match="dtype"):
        PKG.Kv8Cache(1, 1, 10, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="codes"):
        PKG.Kv8Cache(1, 1, 10, codes="e5m2", device="cpu")
    with pytest.raises(ValueError, match="max_len"):
        PKG.Kv8Cache(1, 1, 0, device="cpu")
    with pytest.raises(ValueError, match="n_pages"):
        PKG.Kv8Cache(1, 1, 10, n_pages=0, device="cpu")


def _desc(**over):
    d = KV8.Kv8CacheDesc(2, 2, 128, 8, 4, 1, 0)
    for n in ("k_codes", "v_codes", "scales", "page_table", "k_ring", "v_ring", "lens", "ring_floor", "unclean", "tickets"):
        setattr(d, n, 4096)
    for n, x in over.items():
        setattr(d, n, x)
    return ctypes.byref(d)


def _rows(data=4096, stride=128):
    return ctypes.byref(KV8.Kv8Rows(data, 16 * stride, 2 * stride, stride))


@pytest.mark.parametrize("over,status", [
    (dict(head_dim=96), 3), (dict(dtype=0), 3), (dict(codes=2), 3), (dict(batch=-1), 1), (dict(n_kv_heads=0), 1),
    (dict(n_pages=0), 1), (dict(max_blocks=0), 1), (dict(max_blocks=1 << 30), 3), (dict(n_pages=1 << 26), 3),
    (dict(lens=None), 1), (dict(unclean=None), 1), (dict(k_codes=4100), 2), (dict(scales=4104), 2)])
def test_descriptors_are_checked(over, status):
    lib = LIB.load()
    d = _desc(**over)
    r = _rows()
    assert lib.nsa_kv8_append(d, r, r, 1, None, None, None) == status
    assert lib.nsa_kv8_read(d, 1, None, 4096, 4096, 1, None) == status
    assert lib.nsa_kv8_attend(d, r, r, 4, 1, None, -1, 4, 0.1, 4096, 1 << 30, 4096, None) == status
    assert lib.nsa_kv8_workspace_bytes(d, 4, 1) == 0
    assert lib.nsa_last_error_message()


def test_arguments_are_checked():
    lib = LIB.load()
    d, r = _desc(), _rows()
    assert lib.nsa_kv8_append(None, r, r, 1, None, None, None) == 1
    assert lib.nsa_kv8_append(d, None, r, 1, None, None, None) == 1
    assert lib.nsa_kv8_append(d, r, r, -1, None, None, None) == 1
    assert lib.nsa_kv8_append(d, _rows(4098), r, 1, None, None, None) == 2
    assert lib.nsa_kv8_append(d, r, _rows(stride=129), 1, None, None, None) == 2
    assert lib.nsa_kv8_append(d, None, None, 0, None, None, None) == 0  # nothing to do
    assert lib.nsa_kv8_append(_desc(batch=0), None, None, 1, None, None, None) == 0
    assert lib.nsa_kv8_read(d, 1, None, None, 4096, 1, None) == 1
    assert lib.nsa_kv8_read(d, 1, None, 4096, 4098, 1, None) == 2
    assert lib.nsa_kv8_read(d, 1, None, 4096, 4096, 3, None) == 3

    def attend(q=r, o=r, heads=4, t=1, window=-1, sink=4, scale=0.1, ws=4096, n=1 << 30, tickets=4096, desc=d):
        return lib.nsa_kv8_attend(desc, q, o, heads, t, None, window, sink, scale, ws, n, tickets, None)

    assert attend(q=None) == 1 and attend(o=_rows(4097)) == 2 and attend(heads=3) == 1 and attend(heads=0) == 1
    assert attend(heads=4096) == 3 and attend(t=0) == 1 and attend(t=65) == 1 and attend(sink=-1) == 1
    assert attend(window=1 << 40) == 1 and attend(scale=float("inf")) == 1 and attend(scale=float("nan")) == 1
    assert attend(ws=None) == 4 and attend(n=16) == 4 and attend(tickets=None) == 4 and attend(ws=4100) == 2
    assert attend(desc=_desc(batch=0), q=None) == 0
    def step(k=r, v=r, scale=0.1, ws=4096):
        return lib.nsa_kv8_decode_step(d, k, v, r, r, 4, 1, None, None, -1, 4, scale, ws, 1 << 30, 4096, None)

    assert step(scale=float("nan")) == 1 and step(ws=None) == 4
    assert lib.nsa_kv8_ticket_count() > 0 and lib.nsa_kv8_workspace_bytes(d, 4, 1) > 0
    assert lib.nsa_kv8_workspace_bytes(d, 4, 65) == 0
