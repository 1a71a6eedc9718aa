"""The paged 8-bit key/value cache - written, read back, attended to - against plain formulas in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv(B, S, H, seed, scale=1.0):
    g = _gen(seed)
    ch = torch.exp(0.7 * torch.randn(2, 1, 1, H, D, device="cuda", generator=g))
    x = (torch.randn(2, B, S, H, D, device="cuda", generator=g) * ch * scale).bfloat16()
    return x[0], x[1]


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(B, cols, seed, spare=3):
    """Page ids in no order, and how many pages the cache needs."""
    n = B * cols + spare
    return torch.randperm(n, device="cuda", generator=_gen(seed))[:B * cols].int().view(B, cols).contiguous(), n


def _exponent(amax):
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875).int()
    return torch.where(amax > 0, e, torch.full_like(e, -120)).clamp(-120, 120)


def _quantised(x, page, lens):
    """fp64 [B, T, H, D] -> what the cache holds of tokens t < lens[b] written in one call from token 0."""
    B, T, H, _ = x.shape
    pad = (-T) % page
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, 0, 0, pad))
    seen = (torch.arange(T + pad, device="cuda")[None] < torch.as_tensor(lens, device="cuda")[:, None])
    x = (x * seen[:, :, None, None]).view(B, -1, page, H, D)
    f = torch.exp2(_exponent(x.abs().amax(dim=(2, 4))).double())[:, :, None, :, None]
    return ((x / f).clamp(-448, 448).to(torch.float8_e4m3fn).double() * f).view(B, -1, H, D)[:, :T]


def _filled(k, v, page, lens, seed, spare_cols=0, cache=None):
    from commbench_b200.ops.kvcache import KVCache8

    B, T, H = k.shape[:3]
    pages, n = _table(B, max(1, (T + page - 1) // page) + spare_cols, seed)
    cache = cache or KVCache8(n, H, page=page)
    cache.append(k, v, pages, torch.zeros(B, dtype=torch.int32, device="cuda"), count=_ints(*lens))
    return cache, pages


# ------------------------------------------------------------------------------------- write and read back
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [(1,), (16, 130), (127, 0, 129), (300, 64)])
def test_cache_holds_the_rounded_values(native_lib, page, lens):
    B, T = len(lens), max(lens)
    k, v = _kv(B, T, 3, 1)
    cache, pages = _filled(k, v, page, lens, 2)
    rk, rv = cache.read(pages, None, T, length=_ints(*lens))
    for x, r in ((k, rk), (v, rv)):
        want = _quantised(x, page, lens)
        assert torch.equal(r.double(), want)          # bf16 holds every such number
    # any range, before the first token and past the last
    begin = _ints(*[n // 2 - 20 for n in lens])
    sk, _ = cache.read(pages, begin, T, length=_ints(*lens))
    t = begin[:, None] + torch.arange(T, device="cuda")
    inside = (t >= 0) & (t < _ints(*lens)[:, None])
    pick = torch.where(inside, t, 0).long()[:, :, None, None].expand(-1, -1, 3, D)
    assert torch.equal(sk, rk.gather(1, pick) * inside[:, :, None, None])


@pytest.mark.parametrize("page", [16, 64])
def test_cache_grows_token_by_token(native_lib, page):
    """Tokens of growing size, one or three at a time: the block's scale follows the largest, older tokens are
    rounded again to it - each time by half a step of the scale of that time at most."""
    from commbench_b200.ops.kvcache import KVCache8

    B, T, H = 2, 150, 2
    k, v = _kv(B, T, H, 3)
    size = torch.exp2(torch.arange(T, device="cuda") % 37 / 4.0).bfloat16()[None, :, None, None]
    k, v = k * size, v * size
    pages, n = _table(B, (T + page - 1) // page, 4)
    cache = KVCache8(n, H, page=page)
    at, step = 0, 0
    while at < T:
        s = min((1, 3, 1, 2)[step % 4], T - at)
        cache.append(k[:, at:at + s], v[:, at:at + s], pages, _ints(at, at))
        at, step = at + s, step + 1
    rk, rv = cache.read(pages, None, T)
    for x, r in ((k, rk), (v, rv)):
        pad = torch.nn.functional.pad(x.double(), (0, 0, 0, 0, 0, (-T) % page)).view(B, -1, page, H, D)
        f = torch.exp2(_exponent(pad.abs().amax(dim=(2, 4))).double())[:, :, None, :, None].expand_as(pad)
        f = f.reshape(B, -1, H, D)[:, :T]
        # normal numbers: 2^-4 relative, once (a power of two changes nothing); below 2^-6 f the steps are 2^-9 f,
        # and the sum of the halves over scales that double is a whole one
        assert ((r.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -9 * f).all()
        assert torch.equal(r[:, -1].double(), _quantised_with(x[:, -1], f[:, -1]))


def _quantised_with(x, f):
    return (x.double() / f).clamp(-448, 448).to(torch.float8_e4m3fn).double() * f


def test_cache_reuses_a_page_without_its_old_scale(native_lib):
    k, v = _kv(1, 64, 2, 5, scale=1000.0)
    cache, pages = _filled(k, v, 64, (64,), 6)
    k2, v2 = _kv(1, 10, 2, 7, scale=0.01)
    cache.append(k2, v2, pages, _ints(0))
    rk, rv = cache.read(pages, None, 10)
    assert torch.equal(rk.double(), _quantised(k2, 64, (10,))) and torch.equal(rv.double(), _quantised(v2, 64, (10,)))


@pytest.mark.parametrize("value", [0.0, 1e-38, 1e-20, 448.0, 449.0, 3e38])
def test_cache_of_extreme_values(native_lib, value):
    x = torch.full((1, 5, 1, D), value, dtype=torch.bfloat16, device="cuda")
    cache, pages = _filled(x, x, 32, (5,), 8)
    for r in cache.read(pages, None, 5):
        # below 2^-120 * 448 a block is zero; above, one e4m3 rounding
        want = 0.0 if value < 1e-30 else float(x[0, 0, 0, 0])
        assert ((r.double() - want).abs() <= 2.0 ** -4 * want).all()


def test_cache_of_infinities_and_nan(native_lib):
    k, v = _kv(1, 20, 1, 9)
    k[0, 3, 0, 5], v[0, 4, 0, 6], k[0, 7, 0, 1], v[0, 9, 0, 2] = math.inf, -math.inf, math.nan, math.nan
    cache, pages = _filled(k, v, 32, (20,), 10)
    rk, rv = cache.read(pages, None, 20)
    assert torch.isnan(rk[0, 7, 0, 1]) and torch.isnan(rk[0, 9, 0, 0]) and rv[0, 9, 0, 2] == 0
    assert torch.isnan(rk).sum() == 2 and torch.isfinite(rv).all()
    assert rk[0, 3, 0, 5] >= rk[0, torch.arange(20, device="cuda") < 3].abs().max()
    clean = k.clone()
    clean[0, 3, 0, 5] = clean[0, 7, 0, 1] = 0
    others = torch.ones_like(k, dtype=torch.bool)
    others[0, 3, 0, 5] = others[0, 7, 0, 1] = others[0, 9, 0, 0] = False
    assert torch.equal(rk.double()[others], _quantised(clean, 32, (20,))[others])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [128, 64, 8, 48])
def test_append_rotates_keys_and_queries(native_lib, rot, interleaved):
    from commbench_b200.ops.kvcache import KVCache8
    from commbench_b200.ops.rope import RopeTable, rope

    B, S, H, Hq = 3, 37, 2, 10
    qkv = torch.randn(B, S, Hq + 2 * H, D, device="cuda", generator=_gen(11)).bfloat16()   # a fused projection
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + H], qkv[:, :, Hq + H:]
    start, count = _ints(0, 50, 13), _ints(37, 20, 0)
    pages, n = _table(B, 6, 12)
    cache, table = KVCache8(n, H, page=16), RopeTable(rot, 120, interleaved=interleaved)
    # the tokens before
    old = torch.zeros(B, 50, H, D, dtype=torch.bfloat16, device="cuda")
    cache.append(old, old, pages, _ints(0, 0, 0), count=start)
    out = cache.append(k, v, pages, start, count=count, rope=table, q=q)
    pos = start[:, None] + torch.arange(S, device="cuda")
    want = rope(q, pos, table)
    there = torch.arange(S, device="cuda")[None] < count[:, None]
    # the same products, with or without a fused multiply-add
    tol = 2.0 ** -7 * want.float().abs() + 2.0 ** -22
    assert (((out.float() - want.float()).abs() <= tol) | ~there[:, :, None, None]).all()
    assert (out[~there] == 0).all()
    rk, rv = cache.read(pages, start, S, length=start + count)
    k64 = rope(k.float(), pos, table).double()
    for b, (s, c) in enumerate(((0, 37), (50, 20))):
        for x, r in ((k64, rk), (v.double(), rv)):
            # whole blocks: the tokens before are zeros, so a block's scale is that of its new tokens
            lead = s % 16
            y = torch.nn.functional.pad(x[b:b + 1, :c], (0, 0, 0, 0, lead, (-(lead + c)) % 16))
            want = _quantised(y, 16, (lead + c,))[:, lead:lead + c]
            near = (r[b:b + 1, :c].double() - want).abs() <= 2.0 ** -3 * want.abs()    # a step at a boundary
            assert near.all() and (r[b:b + 1, :c].double() == want).float().mean() > 0.999


# ------------------------------------------------------------------------------------------- attention
def _attend64(q, kc, vc, start, count, window, sinks, scale=None):
    """q [B, S, Hq, D], dequantised caches [B, T, H, D] in fp64: o, lse, and sum of p |v| (for tolerances)."""
    B, S, Hq, _ = q.shape
    H = kc.shape[2]
    o = torch.zeros(B, S, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(o)
    for b in range(B):
        for i in range(min(S, int(count[b]))):
            p = int(start[b]) + i
            j = torch.arange(p + 1, device="cuda")
            j = j if not window else j[(j > p - window) | (j < sinks)]
            k = kc[b, j].repeat_interleave(Hq // H, dim=1)
            v = vc[b, j].repeat_interleave(Hq // H, dim=1)
            s = torch.einsum("hd,jhd->hj", q[b, i].double(), k) * (scale if scale is not None else D ** -0.5)
            lse[b, :, i] = torch.logsumexp(s, dim=1)
            w = torch.softmax(s, dim=1)
            o[b, i] = torch.einsum("hj,jhd->hd", w, v)
            mag[b, i] = torch.einsum("hj,jhd->hd", w, v.abs())
    return o, lse, mag


def _check(o, lse, want):
    ro, rl, mag = want
    # half a unit of bf16 on the result; probabilities rounded to 8 bits at worst; scores of |s| < 2^7 in fp32
    # with sums of 128 products and a 2^-22 exponential
    tol = 2.0 ** -8 * (ro.abs() + mag) * 1.1 + 2.0 ** -24
    err = (o.double() - ro).abs()
    assert torch.isfinite(o).all() and (err <= tol).all(), (err / tol).max()
    empty = rl == -math.inf
    assert (lse[empty] == -math.inf).all()
    assert ((lse.double() - rl).abs()[~empty] <= 1e-4).all()


def _tiles_take(B, S, group):
    """The form of tiles takes at most 128 query tiles of 128 rows."""
    return group <= 128 and B * -(-S // (128 // group)) <= 128


def _case(lens, S, Hq, H, page, window=0, sinks=0, seed=20, max_len=None, count=None, scale=None, cache=None):
    """lens: tokens of each sequence with the new ones; the last S of them are queried."""
    B, T = len(lens), max(max(lens), 1)
    k, v = _kv(B, T, H, seed)
    cache, pages = _filled(k, v, page, lens, seed + 1, cache=cache)
    q = torch.randn(B, S, Hq, D, device="cuda", generator=_gen(seed + 2)).bfloat16()
    cnt = count if count is not None else [S] * B
    start = [n - c for n, c in zip(lens, cnt)]
    want = _attend64(q, _quantised(k, page, lens), _quantised(v, page, lens), start, cnt, window, sinks, scale)
    for impl in (None, "decode", "prefill") + (("tiles",) if _tiles_take(B, S, Hq // H) else ()):
        o, lse = cache.attend(q, pages, _ints(*start), count=None if count is None else _ints(*count), window=window,
                              sinks=sinks, max_len=max_len, scale=scale, impl=impl)
        _check(o, lse, want)
    return cache


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 255, 1000, 1100])
def test_attend_one_token(native_lib, n, page):
    _case([n], 1, 4, 1, page)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 8, 16, 17, 40])
def test_attend_head_groups(native_lib, group):
    _case([300, 77], 1, 2 * group, 2, 64)


@pytest.mark.parametrize("S,group", [(2, 1), (3, 4), (4, 8), (5, 7), (8, 4), (33, 4), (100, 1), (64, 8), (130, 2),
                                     (255, 1), (256, 1), (257, 1)])
def test_attend_several_tokens(native_lib, S, group):
    _case([S, S + 1, S + 700], S, 2 * group, 2, 32)


@pytest.mark.parametrize("B", [1, 5, 40, 300])
def test_attend_many_sequences(native_lib, B):
    """Items that are cut over CTAs and items that are not, of different lengths."""
    lens = [1 + (i * 7919) % 900 for i in range(B)]
    _case(lens, 1, 4, 2, 32, max_len=900)


def test_attend_long_sequence_is_cut_over_the_chip(native_lib):
    _case([20001], 1, 8, 1, 64)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 0), (32, 4), (33, 40), (100, 0), (100, 4), (100, 130),
                                          (257, 64), (1000, 4), (5000, 4)])
@pytest.mark.parametrize("S", [1, 4, 70, 300])
def test_attend_window_and_sinks(native_lib, S, window, sinks):
    _case([max(S, 3), max(S, 70), 333, 900], S, 4, 2, 16 if S == 4 else 64, window=window, sinks=sinks)


def test_attend_counts_and_empty_rows(native_lib):
    """Sequences with fewer new tokens than the batch, none at all, and no token at all."""
    for page in (16, 64):
        _case([100, 5, 40, 0, 513], 5, 4, 2, page, count=[5, 5, 2, 0, 0])


def test_attend_strides_and_scale(native_lib):
    k, v = _kv(2, 90, 2, 40)
    cache, pages = _filled(k, v, 64, (90, 90), 41)
    big = torch.randn(2, 3, 20, D + 4, device="cuda", generator=_gen(42)).bfloat16()
    q = big[:, :, 1:20:2, 4:].transpose(0, 0)[:, :, :8]
    q = q if q.data_ptr() % 8 == 0 else big[:, :, :8, :D]
    start = _ints(87, 87)
    for impl in ("prefill", "tiles", "decode"):
        o, lse = cache.attend(q, pages, start, scale=0.03, impl=impl)
        o2, lse2 = cache.attend(q.contiguous(), pages, start, scale=0.03, impl=impl)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    _check(o, lse, _attend64(q, _quantised(k, 64, (90, 90)), _quantised(v, 64, (90, 90)), (87, 87), (3, 3), 0, 0, 0.03))


@pytest.mark.parametrize("S", [1, 3, 200])
def test_attend_does_not_read_what_it_does_not_see(native_lib, S):
    """NaN, infinities and large numbers in tokens past the end, in pages of nobody and outside the window."""
    from commbench_b200.ops.kvcache import KVCache8

    page, T, n = 32, 500, 420
    k, v = _kv(1, T, 2, 50)
    cache, pages = _filled(k, v, page, (n,), 51, spare_cols=0)
    q = torch.randn(1, S, 4, D, device="cuda", generator=_gen(52)).bfloat16()
    want = {}
    for w in (0, 60):
        want[w] = cache.attend(q, pages, _ints(n - S), window=w, sinks=2)
    junk = torch.full((1, T - n, 2, D), math.nan, dtype=torch.bfloat16, device="cuda")
    junk[:, :, 0] = math.inf
    # written into the cache behind the end: the scale of the shared page stays that of its finite numbers
    cache.append(junk, junk, pages, _ints(n))
    for w in (0, 60):
        o, lse = cache.attend(q, pages, _ints(n - S), window=w, sinks=2)
        assert torch.equal(o, want[w][0]) and torch.equal(lse, want[w][1])
    # and a NaN that every query sees
    k2 = k[:, n - S:n - S + 1].clone()
    k2[0, 0, 1, 3] = math.nan
    cache.append(k2, v[:, n - S:n - S + 1], pages, _ints(n - S))
    o, lse = cache.attend(q, pages, _ints(n - S))
    assert torch.isnan(o[:, :, 2:]).all() and torch.isfinite(o[:, :, :2]).all()


def test_attend_of_value_blocks_of_very_different_size(native_lib):
    """Blocks whose values are zero, tiny or huge count in the sum of the probabilities like any other."""
    lens = (300,)
    k, v = _kv(1, 300, 1, 60, scale=0.3)
    v[:, 64:128] = 0
    v[:, 128:160] *= 2.0 ** -40
    v[:, 200:220] *= 2.0 ** 30
    cache, pages = _filled(k, v, 32, lens, 61)
    q = torch.randn(1, 1, 2, D, device="cuda", generator=_gen(62)).bfloat16()
    for n in (100, 160, 190, 300):
        o, lse = cache.attend(q, pages, _ints(n - 1))
        _check(o, lse, _attend64(q, _quantised(k, 32, lens), _quantised(v, 32, lens), (n - 1,), (1,), 0, 0))


def test_attend_of_large_scores(native_lib):
    """One key far above the others, late: the running maximum rises on the way."""
    k, v = _kv(1, 600, 1, 63)
    size = torch.exp2(torch.arange(600, device="cuda") / 150.0).bfloat16()[None, :, None, None]
    k = k * size
    cache, pages = _filled(k, v, 64, (600,), 64)
    q = (2 * torch.randn(1, 2, 16, D, device="cuda", generator=_gen(65))).bfloat16()
    q[:, :, 3] = 0
    q[:, :, 4] *= 2.0 ** -100
    o, lse = cache.attend(q, pages, _ints(598))
    ro, rl, mag = _attend64(q, _quantised(k, 64, (600,)), _quantised(v, 64, (600,)), (598,), (2,), 0, 0)
    # |s| up to 2^9: a score is off by 2^9 * 2^-24 * a few, the weights by as much relative to each other
    tol = 2.0 ** -8 * (ro.abs() + mag) * 1.1 + 2.0 ** -11 * mag
    assert ((o.double() - ro).abs() <= tol).all() and ((lse.double() - rl).abs() <= 2.0 ** -11).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("S,Hq", [(4, 16), (5, 18), (12, 8), (30, 8), (33, 14)])
def test_attend_tiles_of_pages_with_different_scales(native_lib, page, S, Hq):
    """32, 64 and 128 rows to a tile, keys and values whose size changes by 2^8 within a block."""
    lens = (900, 700)
    k, v = _kv(2, 900, 2, 100)
    size = torch.exp2((torch.arange(900, device="cuda") // 13 % 9).float()).bfloat16()[None, :, None, None]
    k, v = k * size / 32, v * size.flip(1)
    cache, pages = _filled(k, v, page, lens, 101)
    q = torch.randn(2, S, Hq, D, device="cuda", generator=_gen(102)).bfloat16()
    start = [n - S for n in lens]
    ro, rl, mag = _attend64(q, _quantised(k, page, lens), _quantised(v, page, lens), start, [S] * 2, 0, 0)
    # sums of |q k| up to 2^7, held to 2^-18 of that; the weights are off by as much relative to each other
    tol = 2.0 ** -8 * (ro.abs() + mag) * 1.1 + 2.0 ** -11 * mag + 2.0 ** -24
    for impl in ("tiles", "decode", "prefill"):
        o, lse = cache.attend(q, pages, _ints(*start), impl=impl)
        assert ((o.double() - ro).abs() <= tol).all(), impl
        assert ((lse.double() - rl).abs() <= 2.0 ** -11).all(), impl


@pytest.mark.parametrize("S", [3, 12, 40])
def test_attend_tiles_of_small_large_and_infinite_queries(native_lib, S):
    """A row's own power of two carries it from 2^-60 to 2^60; an infinity makes its row no numbers, and no other."""
    k, v = _kv(1, 600, 1, 110)
    cache, pages = _filled(k * 2.0 ** -8, v, 32, (600,), 111)
    q = torch.randn(1, S, 8, D, device="cuda", generator=_gen(112)).bfloat16()
    q[:, :, 1] *= 2.0 ** -60
    q[:, :, 2] = 0
    q[:, :, 4, 5] *= 2.0 ** -30
    start = [600 - S]
    want = _attend64(q, _quantised(k * 2.0 ** -8, 32, (600,)), _quantised(v, 32, (600,)), start, [S], 0, 0)
    _check(*cache.attend(q, pages, _ints(*start), impl="tiles"), want)
    q2 = q.clone()
    q2[:, 1, 3, 7] = math.inf
    o, lse = cache.attend(q2, pages, _ints(*start), impl="tiles")
    assert not torch.isfinite(o[0, 1, 3]).any() and not torch.isfinite(lse[0, 3, 1])
    o[0, 1, 3], lse[0, 3, 1] = want[0][0, 1, 3].to(o.dtype), want[1][0, 3, 1].float()
    _check(o, lse, want)


@pytest.mark.parametrize("B", [33, 100, 128])
def test_attend_tiles_of_many_sequences(native_lib, B):
    _case([8 + (i * 7919) % 500 for i in range(B)], 4, 8, 1, 32, max_len=520, seed=120)


def test_pages_past_32_bits(native_lib):
    """A cache of more than 4 GB whose last pages are used, beside its first."""
    from commbench_b200.ops.kvcache import KVCache8

    page, H, lens = 64, 8, (700, 300)
    n = 2 ** 32 // (H * 2 * page * D) + 40
    cache = KVCache8(n, H, page=page)
    k, v = _kv(2, 700, H, 130)
    pages = torch.stack([torch.arange(n - 11, n, device="cuda"), torch.arange(11, device="cuda")]).int()
    cache.append(k, v, pages, _ints(0, 0), count=_ints(*lens))
    rk, rv = cache.read(pages, None, 700, length=_ints(*lens))
    kc, vc = _quantised(k, page, lens), _quantised(v, page, lens)
    assert torch.equal(rk.double(), kc) and torch.equal(rv.double(), vc)
    q = torch.randn(2, 5, 16, D, device="cuda", generator=_gen(131)).bfloat16()
    want = _attend64(q, kc, vc, (695, 295), (5, 5), 0, 0)
    for impl in ("decode", "prefill", "tiles"):
        _check(*cache.attend(q, pages, _ints(695, 295), impl=impl), want)


def test_attend_repeats_its_bits_and_runs_on_another_stream(native_lib):
    k, v = _kv(3, 1500, 2, 70)
    cache, pages = _filled(k, v, 64, (1500, 700, 64), 71)
    q = torch.randn(3, 2, 8, D, device="cuda", generator=_gen(72)).bfloat16()
    start = _ints(1498, 698, 62)
    for impl in ("decode", "prefill", "tiles"):
        o, lse = cache.attend(q, pages, start, impl=impl)
        s = torch.cuda.Stream()
        for i in range(4):
            s.wait_stream(torch.cuda.current_stream())
            o2, lse2 = cache.attend(q, pages, start, stream=s if i % 2 else None, impl=impl)
            torch.cuda.current_stream().wait_stream(s)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_decode_steps_in_a_graph(native_lib):
    """Append and attend captured once, replayed with other tokens and lengths."""
    from commbench_b200.ops.kvcache import KVCache8
    from commbench_b200.ops.rope import RopeTable

    B, H, Hq, page = 4, 2, 8, 32
    pages, n = _table(B, 8, 80)
    cache, eager = KVCache8(n, H, page=page), KVCache8(n, H, page=page)
    table = RopeTable(128, 256)
    k, v, q = (torch.empty(B, 1, h, D, dtype=torch.bfloat16, device="cuda") for h in (H, H, Hq))
    start = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(c):
        r = c.append(k, v, pages, start, rope=table, q=q)
        return c.attend(r, pages, start)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t in (k, v, q):
        t.zero_()
    with torch.cuda.stream(side):
        step(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step(cache)
    for i in range(70):
        for t, s in ((k, 81), (v, 82), (q, 83)):
            t.copy_(torch.randn(t.shape, device="cuda", generator=_gen(s + 10 * i)))
        start.fill_(i)
        graph.replay()
        ro, rl = step(eager)
        assert torch.equal(o, ro) and torch.equal(lse, rl), i


def test_pages_out_of_range(native_lib):
    """An id that is no page, and a table that is too narrow: nothing written or read there, a status word."""
    from commbench_b200.ops.kvcache import KVCache8

    k, v = _kv(1, 100, 1, 90)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = KVCache8(4, 1, page=32)
    for bad in (-1, 4, 1 << 30):
        pages = _ints(0, bad, 2, 3).view(1, 4)
        status.zero_()
        cache.append(k, v, pages, _ints(0), status_ptr=status.data_ptr())
        assert (status.item() >> 24) == 5
        status.zero_()
        rk, _ = cache.read(pages, None, 100, status_ptr=status.data_ptr())
        assert (status.item() >> 24) == 5 and (rk[:, 32:64] == 0).all() and (rk[:, :32] != 0).any()
        for S in (1, 100):
            q = torch.randn(1, S, 2, D, device="cuda", generator=_gen(91)).bfloat16()
            status.zero_()
            o, lse = cache.attend(q, pages, _ints(100 - S), status_ptr=status.data_ptr())
            assert (status.item() >> 24) == 5 and torch.isfinite(o).all()
    cache.append(k, v, pages[:, :1], _ints(0), status_ptr=status.data_ptr())


def test_cache_refusals(native_lib):
    from commbench_b200.ops.kvcache import KVCache8
    from commbench_b200.ops.rope import RopeTable
    from commbench_b200.runtime.context import CommError

    cache = KVCache8(4, 2, page=32)
    k, v = _kv(1, 8, 2, 95)
    q = torch.zeros(1, 8, 4, D, dtype=torch.bfloat16, device="cuda")
    pages, start = _ints(0, 1).view(1, 2), _ints(0)
    for bad in (lambda: KVCache8(4, 2, page=48), lambda: KVCache8(0, 2), lambda: KVCache8(4, 0),
                lambda: cache.append(k.float(), v, pages, start), lambda: cache.append(k, v[:, :4], pages, start),
                lambda: cache.append(k[:, :, :1], v[:, :, :1], pages, start), lambda: cache.append(k, v, pages.long(), start),
                lambda: cache.append(k, v, pages, start.long()), lambda: cache.append(k, v, pages, _ints(0, 0)),
                lambda: cache.append(k, v, pages, start, q=q), lambda: cache.append(k.cpu(), v.cpu(), pages, start),
                lambda: cache.append(k, v, pages, start, rope=RopeTable(12, 64)),
                lambda: cache.append(k[..., ::2], v, pages, start), lambda: cache.read(pages, start, -1),
                lambda: cache.read(pages, start.float(), 3), lambda: cache.attend(q[:, :, :3], pages, start),
                lambda: cache.attend(q, pages, start, window=-1), lambda: cache.attend(q, pages, start, sinks=-1),
                lambda: cache.attend(q.half(), pages, start), lambda: cache.attend(q, pages, start, count=_ints(1, 1)),
                lambda: cache.attend(q, pages.cpu(), start), lambda: cache.attend(q, pages, start, impl="other")):
        with pytest.raises(CommError):
            bad()
    assert cache.attend(q[:, :0], pages, start)[0].shape == (1, 0, 4, D)
    assert cache.read(pages, None, 0)[0].shape == (1, 0, 2, D)
    cache.append(k[:, :0], v[:, :0], pages, start)
