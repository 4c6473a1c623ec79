"""Prefixes taken over from another sequence's pages (Kv8Cache.adopt): the ring
holds none of their tokens, so going back into them is refused unless it is by
whole blocks, and everything else goes on as if the tokens had been appended."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
pkg = importlib.import_module("numerics-and-sparse-attn_b200")
HKV, GROUP, D = 2, 4, 64


def _lens(*x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def _tokens(b, n, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(b, HKV, n, D, device=DEV, generator=g).half() for _ in range(2))


def _shared(seed, how, prefix=256):
    """Sequence 0 with `prefix` + 40 tokens; sequence 1 begins with its first pages (page 10 is its next)."""
    cache = pkg.Kv8Cache(2, HKV, 512, head_dim=D, n_pages=20, device=DEV)
    cache.page_table[0] = torch.arange(8, dtype=torch.int32)
    cache.page_table[1] = torch.arange(8, 16, dtype=torch.int32)
    k, v = _tokens(2, prefix + 40, seed)
    # the second slot had an occupant of the same length before, whose tokens are still in its ring
    cache.append(k[:, :, :prefix], v[:, :, :prefix])
    cache.append(k[:, :, prefix:], v[:, :, prefix:], counts=_lens(40, 0))
    cache.page_table[1, :prefix // 64] = cache.page_table[0, :prefix // 64]
    if how == "adopt":
        cache.adopt(_lens(-1, prefix))
    else:  # written: seen where the length is another than the calls left
        cache.truncate(_lens(prefix + 40, 64))
        cache.lens[1] = prefix
    return cache, k, v


def _state(cache):
    return [t.clone() for t in (cache.lens, cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8), cache.scales,
                                cache.k_ring, cache.v_ring)]


def _refused(cache, call):
    before = _state(cache)
    call()
    assert pkg.device_error(torch.device(DEV)) == 1
    assert all(torch.equal(a, b) for a, b in zip(before, _state(cache)))


@pytest.mark.parametrize("how", ["adopt", "written"])
def test_going_back_into_a_prefix_is_refused(how):
    cache, k, v = _shared(1, how)
    new, q = k[:, :, :6], torch.zeros(2, HKV * GROUP, 6, D, dtype=torch.float16, device=DEV)
    good = cache.attend(q)
    for start in (255, 250, 193, 129, 1):
        at, none = _lens(296, start), _lens(0, 6)
        _refused(cache, lambda: cache.truncate(at))
        _refused(cache, lambda: cache.append(new, new, starts=at, counts=none))
        _refused(cache, lambda: cache.decode_step(q, new, new, starts=at, counts=none))
    assert torch.equal(cache.attend(q), good)
    # by whole blocks, into a page of its own, it goes
    shared = [t[3].clone() for t in (cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8), cache.scales)]
    cache.page_table[1, 3] = 17
    cache.append(k[:, :, 192:256], v[:, :, 192:256], starts=_lens(296, 192), counts=_lens(0, 64))
    assert torch.equal(cache.scales[17], cache.scales[11])  # (the page that the earlier occupant wrote the same tokens to)
    assert all(torch.equal(t[3], x) for t, x in zip((cache.k_codes.view(torch.uint8), cache.v_codes.view(torch.uint8),
                                                     cache.scales), shared))
    cache.truncate(_lens(296, 250))  # these are in the ring now
    assert cache.lens.tolist() == [296, 250] and pkg.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("how", ["adopt", "written"])
@pytest.mark.parametrize("steps", [3, 70])
def test_a_prefix_goes_on_as_if_appended(how, steps):
    """After tokens behind the prefix: the same state and outputs as a sequence that took all of them itself, and rewinds
    as far as the tokens behind the prefix only."""
    cache, k, v = _shared(2, how)
    ref = pkg.Kv8Cache(1, HKV, 512, head_dim=D, device=DEV)
    ref.append(k[:1, :, :256], v[:1, :, :256])
    nk, nv = _tokens(2, steps, 3)
    g = torch.Generator(device=DEV).manual_seed(4)
    for i in range(steps):
        q = torch.randn(2, HKV * GROUP, D, device=DEV, generator=g).half()
        o = cache.decode_step(q, nk[:, :, i], nv[:, :, i])
        p = ref.decode_step(q[1:], nk[1:, :, i], nv[1:, :, i])
        torch.testing.assert_close(o[1:].double(), p.double(), rtol=2.0 ** -10, atol=2.0 ** -18)  # a step: other cuts
    for a, b in zip(cache.read(256 + steps), ref.read(256 + steps)):
        assert torch.equal(a[1], b[0])
    for start in (255, 200):
        _refused(cache, lambda: cache.truncate(_lens(296 + steps, start)))
    cache.truncate(_lens(296 + steps, 257))
    ref.truncate(_lens(257))
    for a, b in zip(cache.read(257), ref.read(257)):
        assert torch.equal(a[1], b[0])
    assert cache.lens.tolist() == [296 + steps, 257] and pkg.device_error(torch.device(DEV)) == 0


def test_adopt_checks_its_lengths():
    cache, _, _ = _shared(5, "adopt")
    for bad in (7, 65, -2, -64, 576, 1 << 40):
        _refused(cache, lambda: cache.adopt(_lens(-1, bad)))
    cache.adopt(_lens(0, 512))  # all of the table's room, and nothing
    assert cache.lens.tolist() == [0, 512]
    for bad in (None, [0, 0], _lens(0), _lens(0, 0).int(), _lens(0, 0).cpu()):
        with pytest.raises(ValueError, match="lens"):
            cache.adopt(bad)
    assert pkg.device_error(torch.device(DEV)) == 0
    pkg.Kv8Cache(0, 2, 100, device=DEV).adopt(torch.empty(0, dtype=torch.int64, device=DEV))


def test_adopt_of_many_sequences_in_a_graph():
    b = 600
    cache = pkg.Kv8Cache(b, 1, 128, head_dim=D, device=DEV)
    want = torch.zeros(b, dtype=torch.int64, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.adopt(want)
    for i in range(3):
        want.copy_((torch.arange(b) + i) % 3 * 64)
        graph.replay()
        assert torch.equal(cache.lens, want)
    cache.truncate(want - want.clamp_max(1))  # back by one token of an adopted block
    assert pkg.device_error(torch.device(DEV)) == 1 and torch.equal(cache.lens, want)
