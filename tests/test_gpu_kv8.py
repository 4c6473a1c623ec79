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


@pytest.mark.parametrize("d,dtype,codes,starts", [(128, F16, "e4m3", [0, 40, 64]), (64, BF16, "int8", [63, 0, 100])])
def test_decode_steps_through_block_completions(d, dtype, codes, starts):
    """Single-token steps: state bit for bit, attention of each, and decode_step equal to append + attend."""
    hkv, group, steps, b = 2, 4, 70, len(starts)
    k, v = _tokens(b, hkv, max(starts) + steps, d, dtype, 5)
    one, two = (pkg.Kv8Cache(b, hkv, 256, head_dim=d, dtype=dtype, codes=codes, device=DEV) for _ in range(2))
    for c in (one, two):
        _fill(c, k, v, starts)
    for i in range(steps):
        at = [s + i for s in starts]
        nk = torch.stack([k[j, :, n] for j, n in enumerate(at)])
        nv = torch.stack([v[j, :, n] for j, n in enumerate(at)])
        q = _queries(b, hkv * group, 1, d, dtype, i)
        o = one.decode_step(q[:, :, 0], nk, nv)
        two.append(nk, nv)
        assert torch.equal(o, two.attend(q[:, :, 0])), i
        if i % 9 == 0 or any(n % 64 in (62, 63, 0) for n in at):
            _check_state(one, k, v, [n + 1 for n in at])
            _check_attend(one, o[:, :, None], q, k, v, [n + 1 for n in at])
    assert torch.equal(one.k_codes.view(torch.uint8), two.k_codes.view(torch.uint8))
    _clean()


@pytest.mark.parametrize("d,dtype,codes", [(128, BF16, "e4m3"), (64, F16, "int8")])
def test_ragged_appends_hold_what_one_append_holds(d, dtype, codes):
    """However calls cut the tokens (0 to 200 at a time, ragged), the cache is the same to the bit."""
    b, hkv, n = 3, 2, 700
    k, v = _tokens(b, hkv, n, d, dtype, 6)
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, dtype=dtype, codes=codes, device=DEV)
    at = [0] * b
    for sizes in ([1, 63, 64], [65, 1, 0], [0, 200, 128], [7, 129, 3], [190, 70, 150], [63, 64, 65], [2, 0, 190]):
        t = max(sizes)
        nk, nv = torch.zeros(2, b, hkv, t, d, dtype=dtype, device=DEV)
        for i, s in enumerate(sizes):
            nk[i, :, :s], nv[i, :, :s] = k[i, :, at[i]:at[i] + s], v[i, :, at[i]:at[i] + s]
            nk[i, :, s:] = float("nan")  # tokens behind a sequence's count are not looked at
        cache.append(nk, nv, counts=torch.tensor(sizes, device=DEV))
        at = [a + s for a, s in zip(at, sizes)]
        _check_state(cache, k, v, at)
    assert not cache._unclean.any()
    _clean()


def test_drafts_are_causal_and_can_be_taken_back():
    """Four drafted tokens a sequence: each sees its own past; a smaller start takes rejected ones back
    without loss, across a block border too."""
    b, hkv, group, d, dtype = 4, 2, 8, 128, F16
    lens, t = [61, 126, 5, 300], 4
    k, v = _tokens(b, hkv, 320, d, dtype, 7)
    cache = pkg.Kv8Cache(b, hkv, 320, dtype=dtype, device=DEV)
    _fill(cache, k, v, lens)
    bad_k, bad_v = _tokens(b, hkv, t, d, dtype, 8)
    q = _queries(b, hkv * group, t, d, dtype, 9)
    counts = [4, 3, 0, 4]
    o = cache.decode_step(q, bad_k, bad_v, counts=torch.tensor(counts, device=DEV))
    kk, vv = k.clone(), v.clone()
    for i, (n, c) in enumerate(zip(lens, counts)):
        kk[i, :, n:n + c], vv[i, :, n:n + c] = bad_k[i, :, :c], bad_v[i, :, :c]
    now = [n + c for n, c in zip(lens, counts)]
    _check_state(cache, kk, vv, now)
    _check_attend(cache, o, q, kk, vv, now, counts=counts)
    # one draft of each is accepted, the true tokens follow
    accepted = [min(1, c) for c in counts]
    starts = [n + a for n, a in zip(lens, accepted)]
    for i, (n, a) in enumerate(zip(lens, accepted)):
        k[i, :, n:n + a], v[i, :, n:n + a] = bad_k[i, :, :a], bad_v[i, :, :a]
    nk = torch.stack([k[i, :, s:s + t] for i, s in enumerate(starts)])
    nv = torch.stack([v[i, :, s:s + t] for i, s in enumerate(starts)])
    o = cache.decode_step(q, nk, nv, starts=torch.tensor(starts, device=DEV))
    now = [s + t for s in starts]
    _check_state(cache, k, v, now)
    _check_attend(cache, o, q, k, v, now)
    # truncate as far as the ring reaches, and to a multiple of 64; then on
    lens = [n // 64 * 64 - 5 if n // 64 > 0 else 1 for n in now]
    cache.truncate(torch.tensor(lens, device=DEV))
    _clean()
    _check_state(cache, k, v, lens)
    cache.truncate(torch.tensor([0, 64, 0, 128], device=DEV))
    cache.append(k[:, :, 128:190], v[:, :, 128:190], counts=torch.tensor([0, 0, 0, 62], device=DEV))
    assert cache.lens.tolist() == [0, 64, 0, 190]
    _check_attend(cache, cache.attend(q), q, k, v, [0, 64, 0, 190])
    _clean()


@pytest.mark.parametrize("window,sink", [(0, 4), (0, 0), (1, 0), (16, 4), (64, 4), (100, 130), (700, 4), (5000, 4)])
@pytest.mark.parametrize("t", [1, 3])
def test_sink_and_window(window, sink, t):
    lens, hkv, group, d, dtype = [1, 2, 64, 700, 333, 129, 0], 2, 4, 128, BF16
    k, v = _tokens(len(lens), hkv, 700, d, dtype, 10)
    cache = pkg.Kv8Cache(len(lens), hkv, 700, dtype=dtype, codes="int8", device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(len(lens), hkv * group, t, d, dtype, 11)
    o = cache.attend(q, window=window, sink=sink)
    _clean()
    _check_attend(cache, o, q, k, v, lens, window=window, sink=sink)


@pytest.mark.parametrize("t,group,d,dtype", [(64, 8, 128, F16), (17, 3, 64, BF16), (5, 1, 128, BF16), (2, 64, 64, F16)])
def test_many_query_rows(t, group, d, dtype):
    """More rows than a unit takes, rows of tokens the sequence does not have, scales other than the default."""
    lens, hkv = [t, 400, t - 1, 97], 2
    k, v = _tokens(4, hkv, 400, d, dtype, 12)
    cache = pkg.Kv8Cache(4, hkv, 400, head_dim=d, dtype=dtype, device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(4, hkv * group, t, d, dtype, 13)
    for scale in (None, 0.0, -0.3):
        o = cache.attend(q, sm_scale=scale)
        _check_attend(cache, o, q, k, v, lens, scale=scale)
    _clean()


@pytest.mark.parametrize("hkv,group,d,dtype,n", [(1, 1, 128, F16, 40_000), (2, 8, 64, BF16, 70_001), (8, 8, 128, F16, 9_000),
                                                 (1, 16, 128, F16, 25_000)])
def test_long_sequences_are_split_and_merged(hkv, group, d, dtype, n):
    """Units cut between workers and CTAs; beside one of them a ragged rest; the same bits every time."""
    lens = [n, 0, 3000, 17, 2111]
    k, v = _tokens(5, hkv, n, d, dtype, 14)
    cache = pkg.Kv8Cache(5, hkv, n, head_dim=d, dtype=dtype, device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(5, hkv * group, 1, d, dtype, 15)
    o = cache.attend(q)
    _check_attend(cache, o, q, k, v, lens)
    for _ in range(3):
        assert torch.equal(cache.attend(q), o)
    _clean()


def test_more_sequences_than_the_split_keeps_at_hand():
    b, hkv, d = 1500, 1, 64
    lens = [(i * 37) % 140 for i in range(b)]
    k, v = _tokens(b, hkv, 140, d, F16, 16)
    cache = pkg.Kv8Cache(b, hkv, 140, head_dim=d, device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(b, 2, 1, d, F16, 17)
    o = cache.attend(q)
    some = list(range(0, b, 53)) + [b - 1]
    sub = torch.tensor(some, device=DEV)
    _check_attend(cache, o[sub], q[sub], k[sub], v[sub], [lens[i] for i in some])
    assert not o[[i for i in range(b) if lens[i] == 0]].any()
    _clean()


def test_strides_of_projections_and_broadcasts():
    """Token-major projections, slices of a fused one, and a broadcast head, without copies."""
    b, hkv, group, t, d = 2, 4, 2, 70, 128
    fused = torch.randn(b, t, (hkv * group + 2 * hkv) * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(18)).half()
    q, k, v = fused.split([hkv * group * d, hkv * d, hkv * d], dim=-1)
    q, k, v = (x.unflatten(-1, (-1, d)).transpose(1, 2) for x in (q, k, v))
    one, two = (pkg.Kv8Cache(b, hkv, 128, device=DEV) for _ in range(2))
    one.append(k, v)
    two.append(k.contiguous(), v.contiguous())
    assert torch.equal(one.k_codes.view(torch.uint8), two.k_codes.view(torch.uint8)) and torch.equal(one.v_ring, two.v_ring)
    o = one.attend(q[:, :, -3:])
    assert torch.equal(o, two.attend(q[:, :, -3:].contiguous()))
    _check_attend(one, o, q[:, :, -3:], k, v, [t, t])
    shared = k[:, :1].expand(b, hkv, t, d)
    three = pkg.Kv8Cache(b, hkv, 128, device=DEV)
    three.append(shared, shared)
    _check_state(three, shared, shared, [t, t])
    _clean()


def test_pages_in_any_order_and_shared():
    """A pool, pages handed out in a random order; two sequences share a prefix's pages."""
    hkv, group, d, n = 2, 4, 128, 500
    k, v = _tokens(2, hkv, n, d, BF16, 19)
    k[1, :, :256], v[1, :, :256] = k[0, :, :256], v[0, :, :256]
    cache = pkg.Kv8Cache(2, hkv, 512, dtype=BF16, n_pages=21, device=DEV)
    order = torch.randperm(21, generator=torch.Generator().manual_seed(20)).to(torch.int32)
    cache.page_table[0] = order[:8].to(DEV)
    cache.page_table[1] = torch.cat([order[:4], order[8:12]]).to(DEV)
    cache.append(k[:, :, :256], v[:, :, :256], counts=torch.tensor([256, 0], device=DEV))
    cache.lens[1] = 256  # the second sequence begins with the first one's pages
    cache.append(k[:, :, 256:n], v[:, :, 256:n])
    _check_state(cache, k, v, [n, n])
    q = _queries(2, hkv * group, 1, d, BF16, 21)
    _check_attend(cache, cache.attend(q), q, k, v, [n, n])
    rest = order[12:].long().to(DEV)
    assert not cache.scales[rest].any() and not cache.k_codes.view(torch.uint8)[rest].any()  # pages nobody has
    _clean()


def test_bad_pages_lengths_and_starts_are_reported():
    """They are left out or NaN, in bounds, and the device error word says so; others are untouched."""
    b, hkv, d, n = 3, 2, 64, 200
    k, v = _tokens(b, hkv, n, d, F16, 22)
    cache = pkg.Kv8Cache(b, hkv, n, head_dim=d, device=DEV)
    _fill(cache, k, v, [n, n, n])
    q = _queries(b, hkv, 1, d, F16, 23)
    good = cache.attend(q)
    dev = torch.device(DEV)
    _clean()
    for page in (cache.n_pages, -1, 2 ** 31 - 1):
        keep = int(cache.page_table[1, 1])
        cache.page_table[1, 1] = page
        o = cache.attend(q)
        rk, _ = cache.read(n)
        assert pkg.device_error(dev) == 1
        assert torch.isnan(o[1]).all() and torch.equal(o[0], good[0]) and torch.equal(o[2], good[2])
        assert torch.isnan(rk[1, :, 64:128]).all() and not torch.isnan(rk[0]).any()
        cache.append(k[:, :, :64], v[:, :, :64], starts=torch.tensor([64, 64, 64], device=DEV))  # completes that block
        assert pkg.device_error(dev) == 1
        cache.page_table[1, 1] = keep
        cache.append(k[:, :, 64:n], v[:, :, 64:n], starts=torch.tensor([64, 64, 64], device=DEV))
        assert torch.equal(cache.attend(q), good) and pkg.device_error(dev) == 0
    room = cache.max_blocks * 64
    for starts, counts in (([-1, 0, 0], [1, 0, 0]), ([n + 1, 0, 0], [1, 0, 0]), ([70, 0, 0], [1, 0, 0]),
                           ([n, 0, 0], [room - n + 1, 0, 0]), ([n, 0, 0], [-1, 0, 0])):
        t = max(1, counts[0])
        new = torch.zeros(b, hkv, t, d, dtype=F16, device=DEV)
        starts = [starts[0], n, n]
        cache.append(new, new, starts=torch.tensor(starts, device=DEV), counts=torch.tensor(counts, device=DEV))
        assert pkg.device_error(dev) == 1
        assert cache.lens.tolist() == [n, n, n] and torch.equal(cache.attend(q), good)
    for bad in (-1, room + 1):
        cache.lens[2] = bad
        o = cache.attend(q)
        assert pkg.device_error(dev) == 1 and not o[2].any() and torch.equal(o[0], good[0])
    cache.lens[2] = n
    o = cache.attend(q, counts=torch.tensor([1, 2, 1], device=DEV))
    assert pkg.device_error(dev) == 1 and not o[1].any() and torch.equal(o[2], good[2])


@pytest.mark.parametrize("dtype,codes", [(F16, "e4m3"), (BF16, "int8")])
def test_values_that_are_not_finite_stay_where_they_are_seen(dtype, codes):
    """inf and NaN in drafts, in the incomplete block and in a block: NaN for rows that see them, exact for
    rows that do not (causal order, window), and for other heads and sequences."""
    b, hkv, group, t, d = 4, 2, 2, 4, 128
    lens = [150, 150, 250, 70]
    k, v = _tokens(b, hkv, 260, d, dtype, 24)
    v[0, 0, 151, 5] = float("inf")     # the second draft's value
    k[1, 1, 152, 9] = float("nan")     # the third draft's key
    v[2, 0, 30, 3] = float("-inf")     # in the first block: its whole values are NaN
    k[3, 1, 66, 1] = float("inf")      # in the incomplete block, before the drafts
    cache = pkg.Kv8Cache(b, hkv, 260, dtype=dtype, codes=codes, device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(b, hkv * group, t, d, dtype, 25)
    drafts = [torch.stack([x[i, :, n:n + t] for i, n in enumerate(lens)]) for x in (k, v)]
    o = cache.decode_step(q, *drafts)
    now = [n + t for n in lens]
    _check_state(cache, k, v, now)
    ref = o.isnan()
    assert ref[0, :group, 1:, 5].all() and not ref[0, :group, 0].any() and int(ref[0].sum()) == group * 3
    assert ref[1, group:, 2:].all() and int(ref[1].sum()) == group * 2 * d
    assert ref[2, :group].all() and not ref[2, group:].any()
    assert ref[3, group:].all() and not ref[3, :group].any()
    ok_rows = [(0, slice(group, None), slice(None)), (1, slice(0, group), slice(None))]
    for i, h, r in ok_rows:
        assert torch.isfinite(o[i, h, r]).all()
    _check_attend(cache, o[1:2, :, :2], q[1:2, :, :2], k[1:2], v[1:2], [152], scale=d ** -0.5)
    # a window that leaves them out
    o = cache.attend(q[:, :, :1], window=7, sink=0)
    assert torch.isfinite(o[2]).all() and torch.isfinite(o[3]).all()
    _check_attend(cache, o[2:4], q[2:4, :, :1], torch.nan_to_num(k[2:4], posinf=1.0), torch.nan_to_num(v[2:4], neginf=1.0),
                  now[2:4], window=7, sink=0)
    _clean()


@pytest.mark.parametrize("factor", [2.0 ** -120, 2.0 ** -60, 2.0 ** 60, 2.0 ** 120])
def test_bf16_range(factor):
    """Keys, values and queries far outside fp16's range: scales and powers of two carry them."""
    lens, hkv, group, d = [70, 200, 64], 2, 4, 64
    k, v = _tokens(3, hkv, 200, d, BF16, 26, factor)
    cache = pkg.Kv8Cache(3, hkv, 200, head_dim=d, dtype=BF16, device=DEV)
    _fill(cache, k, v, lens)
    _check_state(cache, k, v, lens)
    q = _queries(3, hkv * group, 1, d, BF16, 27)
    for qf in (1.0, 2.0 ** 100 if factor < 1 else 2.0 ** -100):
        scale = d ** -0.5 / factor / qf
        if scale in (0.0, float("inf")) or scale > 3e38 or scale < 1e-37:
            continue
        _check_attend(cache, cache.attend(q * qf, sm_scale=scale), q * qf, k, v, lens, scale=torch.tensor(scale, dtype=torch.float32).item())
    _clean()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_scales_of_any_sign(scale):
    b, hkv, group, d = 2, 2, 4, 128
    lens = [200, 67]
    k, v = _tokens(b, hkv, 200, d, F16, 71)
    cache = pkg.Kv8Cache(b, hkv, 200, device=DEV)
    _fill(cache, k, v, lens)
    q = _queries(b, hkv * group, 2, d, F16, 72)
    scale = torch.tensor(scale, dtype=torch.float32).item()
    _check_attend(cache, cache.attend(q, sm_scale=scale), q, k, v, lens, scale=scale)
    _clean()


def test_zero_blocks_and_zero_queries():
    k = torch.zeros(2, 1, 130, 64, dtype=F16, device=DEV)
    v = k.clone()
    v[1, 0, :64] = 1.0
    cache = pkg.Kv8Cache(2, 1, 130, head_dim=64, device=DEV)
    cache.append(k, v)
    _check_state(cache, k, v, [130, 130])
    q = torch.zeros(2, 3, 64, dtype=F16, device=DEV)
    o = cache.attend(q)
    assert not o[0].any()
    torch.testing.assert_close(o[1].float(), torch.full_like(o[1], 64 / 130).float(), rtol=2.0 ** -11, atol=0)


def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of codes."""
    hkv, d, n, pages = 8, 128, 300, 66_000  # 4.3e9 bytes of K codes
    k, v = _tokens(1, hkv, n, d, F16, 28)
    cache = pkg.Kv8Cache(1, hkv, n, n_pages=pages, device=DEV)
    cache.page_table[0] = torch.arange(pages - 1, pages - 1 - cache.max_blocks, -1, dtype=torch.int32, device=DEV)
    cache.append(k, v)
    _check_state(cache, k, v, [n])
    q = _queries(1, 64, 1, d, F16, 29)
    _check_attend(cache, cache.attend(q), q, k, v, [n])
    assert torch.equal(cache.read(n)[0][0], ok.held(k[0], n, "e4m3").float().half())
    _clean()


def test_read_spans():
    b, hkv, d, n = 3, 2, 128, 300
    k, v = _tokens(b, hkv, n, d, BF16, 30)
    lens = [300, 64, 10]
    cache = pkg.Kv8Cache(b, hkv, n, dtype=BF16, device=DEV)
    _fill(cache, k, v, lens)
    starts = [250, -5, 7]
    rk, rv = cache.read(77, starts=torch.tensor(starts, device=DEV), dtype=torch.float32)
    for i, (s, ln) in enumerate(zip(starts, lens)):
        for got, x in ((rk, k), (rv, v)):
            want = torch.zeros(hkv, 77, d, device=DEV)
            h = ok.held(x[i], ln, "e4m3").float()
            for j in range(77):
                if 0 <= s + j < ln:
                    want[:, j] = h[:, s + j]
            assert torch.equal(got[i], want)
    assert cache.read(0)[0].shape == (b, hkv, 0, d)
    _clean()


def test_graph_of_steps_equals_eager_steps():
    """A captured decode step replayed over changing inputs."""
    b, hkv, group, d, dtype = 3, 2, 8, 128, BF16
    k, v = _tokens(b, hkv, 300, d, dtype, 31)
    caches = [pkg.Kv8Cache(b, hkv, 300, dtype=dtype, device=DEV) for _ in range(2)]
    for c in caches:
        _fill(c, k, v, [60, 0, 127])
    q, nk, nv = (torch.zeros(b, h, d, dtype=dtype, device=DEV) for h in (hkv * group, hkv, hkv))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # captured cold: nothing of this shape has run before
        out = caches[0].decode_step(q, nk, nv)
    for i in range(75):
        q.copy_(_queries(b, hkv * group, 1, d, dtype, i)[:, :, 0])
        nk.copy_(k[:, :, 130 + i])
        nv.copy_(v[:, :, 130 + i])
        graph.replay()
        assert torch.equal(out, caches[1].decode_step(q, nk, nv)), i
    assert torch.equal(caches[0].lens, caches[1].lens) and torch.equal(caches[0].k_ring, caches[1].k_ring)
    _clean()


def test_graphs_and_streams_side_by_side():
    """Attention captured twice and replayed on two streams at once, beside eager calls on a third."""
    hkv, group, d, n = 2, 8, 128, 6000
    k, v = _tokens(2, hkv, n, d, F16, 32)
    caches = [pkg.Kv8Cache(2, hkv, n, device=DEV) for _ in range(3)]
    qs = [_queries(2, hkv * group, 1, d, F16, 33 + i)[:, :, 0] for i in range(3)]
    for c in caches:
        c.append(k, v)
    want = [c.attend(q) for c, q in zip(caches, qs)]
    graphs, outs = [], []
    for c, q in zip(caches[:2], qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c.attend(q) for _ in range(4)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = caches[2].attend(qs[2])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i]) and torch.equal(eager, want[2])
    _clean()


def test_empty_batch():
    cache = pkg.Kv8Cache(0, 2, 100, device=DEV)
    new, q = (torch.empty(0, h, 128, dtype=F16, device=DEV) for h in (2, 16))
    cache.append(new, new)
    assert cache.attend(q).shape == (0, 16, 128) and cache.decode_step(q, new, new).shape == (0, 16, 128)
    assert cache.read(5)[0].shape == (0, 2, 5, 128)
    empty = pkg.Kv8Cache(2, 2, 100, device=DEV)
    none = torch.empty(2, 2, 0, 128, dtype=F16, device=DEV)
    empty.append(none, none)  # no tokens
    assert empty.lens.tolist() == [0, 0]
    _clean()


def test_refusals():
    c = pkg.Kv8Cache(2, 2, 100, device=DEV)
    new, q = (torch.zeros(2, h, 128, dtype=F16, device=DEV) for h in (2, 8))
    with pytest.raises(TypeError):
        c.append(new.bfloat16(), new.bfloat16())
    with pytest.raises(ValueError, match="device"):
        c.append(new.cpu(), new.cpu())
    with pytest.raises(ValueError, match="same shape"):
        c.append(new, new[:, :, None].expand(2, 2, 3, 128))
    with pytest.raises(ValueError, match="must be"):
        c.append(new[:, :1], new[:, :1])
    with pytest.raises(ValueError, match="multiple of 2"):
        c.attend(q[:, :7])
    with pytest.raises(ValueError, match="last dimension"):
        c.attend(torch.zeros(2, 128, 8, dtype=F16, device=DEV).transpose(1, 2))
    with pytest.raises(ValueError, match="aligned"):
        c.attend(torch.zeros(2 * 8 * 128 + 1, dtype=F16, device=DEV)[1:].view(2, 8, 128))
    with pytest.raises(ValueError, match="n_tokens"):
        c.attend(torch.zeros(2, 8, 65, 128, dtype=F16, device=DEV))
    with pytest.raises(ValueError, match="window"):
        c.attend(q, window=-1)
    with pytest.raises(ValueError, match="sink"):
        c.attend(q, window=5, sink=-1)
    with pytest.raises(ValueError, match="finite"):
        c.attend(q, sm_scale=float("nan"))
    with pytest.raises(ValueError, match="counts"):
        c.attend(q, counts=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="starts"):
        c.append(new, new, starts=torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="same number"):
        c.decode_step(q, new[:, :, None].expand(2, 2, 3, 128), new)
    with pytest.raises(TypeError):
        c.read(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens"):
        c.truncate(None)
    with pytest.raises(ValueError, match="finite"):
        c.decode_step(q, new, new, sm_scale=float("inf"))  # and nothing is appended
    with pytest.raises(ValueError, match="aligned"):
        c.decode_step(q, new, torch.zeros(2 * 2 * 128 + 1, dtype=F16, device=DEV)[1:].view(2, 2, 128))
    assert c.lens.tolist() == [0, 0] and not c.k_ring.any()
    _clean()


@pytest.mark.parametrize("n", [126, 127, 400])
def test_step_equals_append_and_attend_in_every_form(n):
    """Ragged counts, a rewind, a window, a start that is refused and one that is not; a batch beyond what the split keeps
    at hand; repeated back to back, so that steps follow one another without a pause."""
    hkv, group, d, t = 2, 4, 64, 3
    for b in (4, 700):
        k, v = _tokens(b, hkv, n + 4 * t, d, BF16, 40)
        one, two = (pkg.Kv8Cache(b, hkv, n + 4 * t, head_dim=d, dtype=BF16, device=DEV) for _ in range(2))
        lens = [(n - 7 * i) % n + 1 for i in range(b)]
        for c in (one, two):
            _fill(c, k, v, lens)
        counts = torch.tensor([i % (t + 1) for i in range(b)], device=DEV)
        starts = torch.tensor(lens, device=DEV)
        starts[0] = -3  # refused: this sequence stays as it is
        starts[1] = lens[1] // 64 * 64
        q = _queries(b, hkv * group, t, d, BF16, 41)
        nk, nv = k[:, :, n:n + t], v[:, :, n:n + t]
        pairs = []
        for i in range(4):
            kw = dict(counts=counts, starts=starts if i % 2 == 0 else None)
            mask = dict(window=50, sink=2) if i > 1 else {}
            o = one.decode_step(q, nk, nv, **kw, **mask)
            two.append(nk, nv, **kw)
            pairs.append((o, two.attend(q, counts=counts, **mask), one.lens.clone(), two.lens.clone()))
        for o, p, a, c in pairs:
            assert torch.equal(o, p) and torch.equal(a, c)
        assert pkg.device_error(torch.device(DEV)) == 1
        assert one.lens[0] == lens[0] + 0 and one.lens.tolist()[1:3] == two.lens.tolist()[1:3]
        for x in ("k_ring", "v_ring", "scales", "_ring_floor"):
            assert torch.equal(getattr(one, x), getattr(two, x)), x
        assert torch.equal(one.k_codes.view(torch.uint8), two.k_codes.view(torch.uint8))
        assert not one._append_tickets.any() and not two._append_tickets.any()
