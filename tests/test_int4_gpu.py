"""GPU tests of the 4-bit paged cache: the quantizing write, the read-back and decode,
against plain forms in 64 bits.

Tolerances.  A half step of fp16 is 2^-11 of the value, of bf16 2^-8.
* Codes: equal to the 64-bit quantizer's but where fp32's (x - m) is inexact, which these
  inputs do not do beside a border: equal, bit for bit.
* Read-back: s * c is exact in fp32 and the sum rounds to fp32 and to the output type: half a
  step of the type plus 2^-24 of the larger summand.
* Decode, in fp32 (u = 2^-24 a rounding).  A score s' (q . c') + m' sum(q) is a sum of at most
  D + 8 roundings of summands that add up to S = |scale| (s' sum |q| c' + |m'| sum |q|), so it is
  off by at most (D + 8) u S, and a token's weight p by that share of itself: the output moves by
  at most sum p_t (D + 8) u S_t (|v_t| + |out|) / sum p.  The weighted sums, the weights' rounding
  and the quotient are roundings of summands |s c| + |m|: 2^11 of them, u 2^11 = 2^-13, are
  allowed (they go both ways).  Then the output's own half step, and a smallest step of its type.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module", autouse=True)
def _lib(built):
    import pa_int8

    pa_int8.ext()


# ------------------------------------------------------------------ plain forms, 64 bits

def quantize64(x):
    """x [..., D] -> codes, scale, minimum (fp16 values as float64)."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    c = torch.round((x - m.double()) / s.double()).clamp(0, 15)
    c = torch.where((s == 0) | bad, torch.zeros_like(c), c).to(torch.uint8)
    nan = torch.full_like(s, float("nan"))
    return c, torch.where(bad, nan, s), torch.where(bad, nan, m)


def pack(c):
    """Codes [..., D] -> bytes [..., D / 8, 4]: dim e of 8 in bits 4e..4e+3."""
    c = c.view(*c.shape[:-1], c.shape[-1] // 8, 4, 2)
    return c[..., 0] + 16 * c[..., 1]


def unpack_cache(cache):
    """[NB, Hkv, bs/4, D/8, 4, 4] -> codes [NB, Hkv, bs, D]."""
    nb, h, quads, ch = cache.shape[:4]
    b = cache.transpose(3, 4)
    return torch.stack([b % 16, b // 16], -1).reshape(nb, h, quads * 4, ch * 8)


def values64(cache, scales):
    return unpack_cache(cache).double() * scales[..., :1].double() + scales[..., 1:].double()


def new_cache(nb, hkv, d, bs, fill=None):
    shape = (nb, hkv, bs // 4, d // 8, 4, 4)
    if fill is None:
        c = lambda: torch.zeros(shape, dtype=torch.uint8, device=DEV)  # noqa: E731
        s = lambda: torch.zeros((nb, hkv, bs, 2), dtype=torch.float16, device=DEV)  # noqa: E731
    else:
        c = lambda: torch.randint(0, 256, shape, dtype=torch.uint8, device=DEV)  # noqa: E731
        s = lambda: torch.full((nb, hkv, bs, 2), fill, dtype=torch.float16, device=DEV)  # noqa: E731
    return c(), c(), s(), s()


def write64(k, v, slots, kc, vc, ks, vs):
    bs, pool = ks.shape[2], ks.shape[0] * ks.shape[2]
    ok = (slots >= 0) & (slots < pool)
    at = slots[ok]
    for x, cache, scales in ((k, kc, ks), (v, vc, vs)):
        c, s, m = quantize64(x[ok])
        off = at % bs
        cache[at // bs, :, off // 4, :, off % 4] = pack(c)
        scales[at // bs, :, off] = torch.cat([s, m], -1)


def decode64(q, kc, vc, ks, vs, bt, lens, scale):
    """(out, what fp32 may be off by) in float64, sequence by sequence; blocks outside the pool
    hold no tokens."""
    s, h, d = q.shape
    nb, hkv, bs = ks.shape[:3]
    out = torch.zeros(s, h, d, dtype=torch.float64, device=DEV)
    off = torch.zeros_like(out)
    for i, n in enumerate(lens):
        n = min(max(int(n), 0), bt.shape[1] * bs)
        blk = bt[i, :-(-n // bs)].long()
        ok = (blk >= 0) & (blk < nb)
        pick = ok.repeat_interleave(bs)[:n]
        if not bool(pick.any()):
            continue
        blk = blk.clamp(0, nb - 1)

        def take(x):                           # [n, ...] of kv head j
            x = x[:, j]
            return x.reshape(-1, x.shape[-1])[:n][pick].double()

        kcode, vcode = unpack_cache(kc[blk]), unpack_cache(vc[blk])
        for j in range(hkv):
            qj = q[i, j * (h // hkv):(j + 1) * (h // hkv)].double()
            kj, ksj, vj, vsj = take(kcode), take(ks[blk]), take(vcode), take(vs[blk])
            k, v = kj * ksj[:, :1] + ksj[:, 1:], vj * vsj[:, :1] + vsj[:, 1:]
            p = torch.softmax(torch.mm(qj, k.t().contiguous()) * scale, -1)
            size = torch.mm(qj.abs(), (kj * ksj[:, :1].abs() + ksj[:, 1:].abs()).t().contiguous())
            w = p * (size * (abs(scale) * (d + 8) * 2.0 ** -24))
            r = slice(j * (h // hkv), (j + 1) * (h // hkv))
            o = torch.mm(p, v)
            out[i, r] = o
            off[i, r] = (torch.mm(w, v.abs()) + w.sum(-1, keepdim=True) * o.abs() +
                         2.0 ** -13 * torch.mm(p, vj * vsj[:, :1].abs() + vsj[:, 1:].abs()))
    return out, off


def close(got, want, off, dtype):
    tiny = torch.finfo(dtype).smallest_normal * 2 * EPS[dtype]     # the smallest step
    bound = EPS[dtype] * want.abs() + off + tiny
    err = (got.double() - want).abs()
    nan = torch.isnan(want)                    # (a row without a value, from fp16's overflow)
    bad = torch.where(nan, ~torch.isnan(got), ~(err <= bound))
    assert not bool(bad.any()), (int(bad.sum()), bad.numel(), float((err / bound).max()),
                                 float(err.max()))


# ------------------------------------------------------------------ write and read-back

def rows(t, hkv, d, dtype, seed, fused=False):
    """K and V rows with the quantizer's corner cases among them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(t, (5 * hkv if fused else 0) + 2 * hkv, d, device=DEV, generator=g)
    x = (x * torch.exp(2 * torch.randn(t, x.shape[1], 1, device=DEV, generator=g))).to(dtype)
    k, v = x[:, -2 * hkv:-hkv], x[:, -hkv:]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    if t >= 6:
        k[0], v[1, 0] = 0.0, 0.0                       # a range of 0
        k[1], v[0, 0] = 3.5, -7.0
        k[2], v[2, 0] = 3e-8, 1e-7                     # below fp16's normal numbers
        k[2, :, :4] = 9e-7
        k[3, :, 0] = 1000.0                            # an outlier
        ramp = torch.arange(d, device=DEV) % 31 / 2.0  # every other value on a border of codes
        k[4], v[3, 0] = ramp.to(dtype), (ramp * 4 - 60).to(dtype)
        k[5, 0] = torch.linspace(-65504.0, 65504.0, d, device=DEV).to(dtype)
    return k, v


WRITE = [  # tokens, kv heads, head_dim, block size
    (1, 1, 128, 16), (3, 2, 64, 16), (37, 8, 128, 16), (130, 3, 80, 32), (64, 2, 256, 64),
    (77, 2, 8, 16), (50, 1, 24, 128), (41, 4, 96, 16), (33, 2, 200, 32), (19, 5, 136, 16),
    (2500, 8, 128, 16), (1111, 2, 256, 32), (900, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,hkv,d,bs", WRITE)
@pytest.mark.parametrize("order", ["run", "scattered"])
def test_write_and_gather(t, hkv, d, bs, dtype, order):
    import pa_int8

    nb = -(-t // bs) + 3
    fused = t % 2 == 1
    k, v = rows(t, hkv, d, dtype, t + d, fused)
    g = torch.Generator().manual_seed(t)
    if order == "run":                                  # from an odd position on
        slots = torch.arange(t) + 5
    else:
        slots = torch.randperm(nb * bs, generator=g)[:t]
        slots[torch.rand(t, generator=g) < 0.1] = -1
        slots[t // 2] = nb * bs + 3                     # past the pool
    slots = slots.to(DEV)
    got = new_cache(nb, hkv, d, bs, fill=0.25)
    want = [x.clone() for x in got]
    pa_int8.reshape_and_cache_int4(k, v, *got, slots)
    write64(k, v, slots, *want)
    for a, b, what in zip(got, want, ("k_cache", "v_cache", "k_scales", "v_scales")):
        a, b = (a.view(torch.int16), b.view(torch.int16)) if a.dtype == torch.float16 else (a, b)
        assert torch.equal(a, b), (what, int((a != b).sum()), a.numel())
    # read back, into rows with room between them
    wide = torch.full((2, t, hkv, d + 8), 7.0, dtype=dtype, device=DEV)
    key, value = wide[0, :, :, :d], wide[1, :, :, :d]
    pa_int8.gather_cache_int4(key, value, *got, slots)
    ok = (slots >= 0) & (slots < nb * bs)
    at = slots.clamp(0, nb * bs - 1)
    for x, cache, scales in ((key, want[0], want[2]), (value, want[1], want[3])):
        val = values64(cache, scales)[at // bs, :, at % bs]
        m = scales[at // bs, :, at % bs].double().abs()
        big = 15 * m[..., :1] + m[..., 1:]
        val = torch.where(ok[:, None, None], val, torch.zeros_like(val))
        inside = val.abs() <= torch.finfo(dtype).max
        assert torch.equal(torch.isfinite(x) | ~inside, torch.ones_like(inside))
        tiny = torch.finfo(dtype).smallest_normal * 2 * EPS[dtype]
        err = (x.double() - val).abs()[inside]
        assert bool((err <= (EPS[dtype] * val.abs() + 2.0 ** -24 * big + tiny)[inside]).all())
    assert bool((wide[..., d:] == 7.0).all())
    assert not bool((key[~ok] != 0).any()) and not bool((value[~ok] != 0).any())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_without_a_value(dtype):
    """A row with an infinity or a NaN reads back as NaN and leaves its neighbours alone; bf16
    rows beyond fp16's range saturate."""
    import pa_int8

    k, v = rows(8, 2, 128, dtype, 3)
    k[6, 0, 17], k[7, 1, 127], v[6, 1, 0] = float("inf"), float("nan"), float("-inf")
    if dtype == torch.bfloat16:
        k[1, 0, 3], k[1, 0, 4] = 3e38, -1e30
    got = new_cache(1, 2, 128, 16)
    want = [x.clone() for x in got]
    slots = torch.arange(8, device=DEV)
    pa_int8.reshape_and_cache_int4(k, v, *got, slots)
    write64(k, v, slots, *want)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(torch.nan_to_num(a, nan=-5.0), torch.nan_to_num(b, nan=-5.0))
    key, value = torch.empty_like(k), torch.empty_like(v)
    pa_int8.gather_cache_int4(key, value, *got, slots)
    nan = torch.isnan(key).all(-1)
    assert nan.nonzero().tolist() == [[6, 0], [7, 1]]
    assert torch.isnan(value).all(-1).nonzero().tolist() == [[6, 1]]
    assert not bool(torch.isnan(key[~nan]).any())


def test_write_of_nothing_and_all_skipped():
    import pa_int8

    got = new_cache(2, 2, 64, 16, fill=0.5)
    keep = [x.clone() for x in got]
    k = torch.ones(5, 2, 64, dtype=torch.float16, device=DEV)
    pa_int8.reshape_and_cache_int4(k[:0], k[:0], *got, torch.empty(0, dtype=torch.int64, device=DEV))
    pa_int8.reshape_and_cache_int4(k, k, *got, torch.full((5,), -1, dtype=torch.int64, device=DEV))
    pa_int8.gather_cache_int4(k[:0], k[:0], *got, torch.empty(0, dtype=torch.int64, device=DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, keep))


def test_one_tensor_for_key_and_value_is_refused():
    import pa_int8

    kc, vc, ks, vs = new_cache(2, 2, 64, 16, fill=0.5)
    k, i = torch.ones(5, 2, 64, dtype=torch.float16, device=DEV), torch.arange(5, device=DEV)
    pa_int8.reshape_and_cache_int4(k, k, kc, vc, ks, vs, i)      # (as rows to write it is fine)
    for caches in ((kc, kc, ks, vs), (kc, vc, ks, ks)):
        with pytest.raises(RuntimeError, match="one tensor"):
            pa_int8.reshape_and_cache_int4(k, k, *caches, i)
    with pytest.raises(RuntimeError, match="one tensor"):
        pa_int8.gather_cache_int4(k, k, kc, vc, ks, vs, i)
    out = torch.empty(2, 5, 2, 64, dtype=torch.float16, device=DEV)
    pa_int8.gather_cache_int4(out[0], out[1], kc, kc, ks, ks, i)  # (one cache read twice, too)
    assert bool((out == 1).all())


# ------------------------------------------------------------------ decode

def paged(lens, hkv, d, bs, dtype, seed, k_mul=1.0, v_mul=1.0, spread=0.0, extra_cols=0):
    """A 4-bit cache of the lengths at permuted blocks; everything no sequence holds is garbage
    (codes random, scales NaN).  `spread`: the rows' magnitudes vary by exp(spread * N(0,1))."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    nblk = [-(-int(n) // bs) for n in lens]
    nb = sum(nblk) + 2
    perm = torch.randperm(nb, device=DEV, generator=g)
    bt = torch.full((len(lens), max(max(nblk), 1) + extra_cols), -7, dtype=torch.int32, device=DEV)
    cache = new_cache(nb, hkv, d, bs, fill=float("nan"))
    at = 0
    for i, n in enumerate(lens):
        n = int(n)
        bt[i, :nblk[i]] = perm[at:at + nblk[i]].int()
        at += nblk[i]
        if n == 0:
            continue
        pos = torch.arange(n, device=DEV)
        slots = bt[i].long()[pos // bs] * bs + pos % bs
        kv = torch.randn(2, n, hkv, d, device=DEV, generator=g)
        kv = kv + torch.randn(2, 1, hkv, d, device=DEV, generator=g)
        if spread:
            kv = kv * torch.exp(spread * torch.randn(2, n, hkv, 1, device=DEV, generator=g))
        write64((kv[0] * k_mul).to(dtype), (kv[1] * v_mul).to(dtype), slots, *cache)
    return cache, bt


def check_decode(lens, heads, hkv, d, bs, dtype, seed, q_mul=1.0, scale=None, check=False, **kw):
    import pa_int8

    cache, bt = paged(lens, hkv, d, bs, dtype, seed, **kw)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = (torch.randn(len(lens), heads, d, device=DEV, generator=g) * q_mul).to(dtype)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    ctx = torch.tensor([int(n) for n in lens], dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 9.0)
    ret = pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, scale, bs, k_scales=cache[2],
                         v_scales=cache[3], check=check)
    assert ret is out
    close(out, *decode64(q, *cache, bt, lens, scale), dtype)
    return out, q, cache, bt, ctx, scale


LENS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500, 1025]


@pytest.mark.parametrize("n", LENS)
@pytest.mark.parametrize("heads,hkv", [(8, 8), (8, 2), (8, 1), (12, 2), (32, 1), (40, 1)])
def test_decode_lengths_and_groups(n, heads, hkv):
    check_decode([n, max(1, n - 5), n + 3], heads, hkv, 128, 16, torch.float16, n + heads)


@pytest.mark.parametrize("d", list(range(8, 257, 8)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_head_dims(d, dtype):
    check_decode([1, 70, 333], 6, 2, d, 16, dtype, d)
    check_decode([200, 41], 20, 1, d, 32, dtype, d + 1)


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_block_sizes(bs, d):
    check_decode([1, bs, bs + 1, 3 * bs - 1, 777], 16, 4, d, bs, torch.bfloat16, bs + d,
                 extra_cols=9)


@pytest.mark.parametrize("heads,hkv", [(1, 1), (16, 1), (17, 1), (32, 2), (48, 1), (64, 1), (64, 8),
                                       (28, 4), (71, 1)])
@pytest.mark.parametrize("d", [72, 128, 192])
def test_decode_group_sizes(heads, hkv, d):
    check_decode([130, 1, 67], heads, hkv, d, 16, torch.float16, heads + d)


@pytest.mark.parametrize("heads,hkv", [(2, 1), (8, 2), (10, 2), (8, 1), (18, 2)])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 128, 136, 200, 256])
@pytest.mark.parametrize("lens", [[20000, 3, 0, 700], [513, 64, 8, 9, 17]])
def test_decode_small_groups_of_every_width(heads, hkv, d, lens):
    """Groups of 2, 4, 5, 8 and 9 heads, whose unused columns hold parts of the work; pieces
    of one work-group and of many."""
    check_decode(lens, heads, hkv, d, 16, torch.bfloat16 if d % 16 else torch.float16, heads + d)


@pytest.mark.parametrize("lens", [
    [4096] * 4, [20000], [20000, 1, 3, 9000], list(range(1, 130)), [1] * 300,
    [0, 5, 0, 0, 700, 0], [0], [0, 0, 0],
    [2048 + 64 * (i % 7) for i in range(40)], [33] * 1500,
])
@pytest.mark.parametrize("heads,hkv,d", [(8, 2, 128), (4, 4, 64), (32, 1, 256)])
def test_decode_batches(lens, heads, hkv, d):
    check_decode(lens, heads, hkv, d, 16, torch.float16, len(lens) + d)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("v_mul", [1e-6, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize("spread", [0.0, 2.0])
def test_decode_magnitudes_of_v(dtype, v_mul, spread):
    """Rows of V from fp16's subnormal numbers up, alike and decades apart."""
    check_decode([300, 1000], 8, 2, 128, 16, dtype, 5, v_mul=v_mul, spread=spread, k_mul=0.3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_mul", [0.0, 1e-5, 1e-2, 30.0, 3000.0])
def test_decode_magnitudes_of_q(dtype, q_mul):
    """From an even softmax to one token that takes all; the scale brings scores back."""
    scale = 1.0 / math.sqrt(128) / max(q_mul, 1e-5) * 8
    check_decode([300, 1000, 2], 8, 2, 128, 16, dtype, 6, q_mul=q_mul, scale=scale)


def test_decode_query_elements_decades_apart():
    import pa_int8

    cache, bt = paged([200, 31], 2, 128, 16, torch.float16, 8)
    q = torch.randn(2, 8, 128, device=DEV)
    q = (q * torch.pow(2.0, torch.randint(-18, 4, q.shape, device=DEV))).half()
    q[0, 0] = 0.0
    q[0, 1] = 0.0
    q[0, 1, 5] = 6e-8
    ctx = torch.tensor([200, 31], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, 0.3, 16, k_scales=cache[2],
                   v_scales=cache[3], check=False)
    close(out, *decode64(q, *cache, bt, [200, 31], 0.3), torch.float16)


@pytest.mark.parametrize("heads,hkv,d,bs", [(32, 1, 64, 128), (40, 1, 128, 64), (71, 1, 96, 128),
                                            (34, 2, 24, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[300000, 1, 70001, 262144, 90000, 0, 64, 100000], [131072] * 6,
                                  [131072] * 5 + [131008]])
def test_decode_long_lists_of_wide_groups(heads, hkv, d, bs, dtype, lens):
    """Groups of more than 16 heads with tiles for every wave to have six (12288 and one fewer
    among the last two); sequences share the blocks of a small pool."""
    import pa_int8

    pool = 37
    cache, _ = paged([pool * bs], hkv, d, bs, dtype, heads)
    g = torch.Generator(device=DEV).manual_seed(heads + d)
    bt = torch.randint(0, pool, (len(lens), -(-max(lens) // bs)), device=DEV, generator=g).int()
    used = torch.isfinite(cache[2]).all(-1).all(-1).all(-1).nonzero()[:, 0].int()
    assert used.numel() == pool
    bt = used[bt.long()].contiguous()
    q = torch.randn(len(lens), heads, d, device=DEV, generator=g).to(dtype)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 9.0)
    pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, d ** -0.5, bs, k_scales=cache[2],
                   v_scales=cache[3], check=False)
    close(out, *decode64(q, *cache, bt, lens, d ** -0.5), dtype)


def test_decode_invalid_blocks_hold_no_tokens():
    import pa_int8

    lens = [300, 64, 90, 1000]
    cache, bt = paged(lens, 2, 128, 16, torch.float16, 9)
    nb = cache[0].shape[0]
    bt[0, 3], bt[0, 18], bt[1, :], bt[2, 0], bt[3, 5:40] = -1, nb, -5, nb + 1000, 2 ** 31 - 1
    q = torch.randn(4, 8, 128, device=DEV).half()
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 3.0)
    pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, 0.09, 16, k_scales=cache[2],
                   v_scales=cache[3], check=False)
    assert not bool(out[1].any())
    close(out, *decode64(q, *cache, bt, lens, 0.09), torch.float16)


def test_decode_lengths_past_the_table_are_clamped():
    import pa_int8

    cache, bt = paged([64, 32], 2, 64, 16, torch.float16, 10)
    q = torch.randn(2, 4, 64, device=DEV).half()
    bt = bt[:, :2].contiguous()
    ctx = torch.tensor([2 ** 31 - 1, -4], dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 3.0)
    pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, 0.2, 16, k_scales=cache[2],
                   v_scales=cache[3], check=False)
    close(out, *decode64(q, *cache, bt, [32, 0], 0.2), torch.float16)
    assert not bool(out[1].any())


def test_decode_nan_rows_stay_in_their_sequence():
    import pa_int8

    cache, bt = paged([100, 100], 1, 128, 16, torch.float16, 11)
    blk = int(bt[0, 2])
    cache[3][blk, 0, 5] = float("nan")
    q = torch.randn(2, 4, 128, device=DEV).half()
    ctx = torch.tensor([100, 100], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    pa_int8.decode("int4", out, q, cache[0], cache[1], bt, ctx, 0.1, 16, k_scales=cache[2],
                   v_scales=cache[3], check=False)
    assert bool(torch.isnan(out[0]).all()) and not bool(torch.isnan(out[1]).any())


def test_decode_checked_names_and_refusals():
    import pa_int8

    out, q, cache, bt, ctx, scale = check_decode([50, 9], 8, 2, 128, 16, torch.float16, 12,
                                                 check=True)
    o2 = torch.empty_like(out)
    pa_int8.VARIANTS_INT4["int4"](o2, q, *cache, bt, ctx, scale, 16)
    assert torch.equal(out, o2)
    bad = ctx.clone()
    bad[1] = 0
    with pytest.raises(RuntimeError, match="context_lens must be >= 1"):
        pa_int8.VARIANTS_INT4["int4"](o2, q, *cache, bt, bad, scale, 16)
    run = lambda **k: pa_int8.decode(  # noqa: E731
        "int4", k.get("out", out), k.get("q", q), k.get("kc", cache[0]), k.get("vc", cache[1]),
        k.get("bt", bt), k.get("ctx", ctx), scale, k.get("bs", 16), k_scales=k.get("ks", cache[2]),
        v_scales=cache[3], check=False, partition_tokens=k.get("part", 0))
    for kw, match in [
            (dict(q=q.float()), "fp16 or bf16"), (dict(out=out.bfloat16()), "one dtype"),
            (dict(kc=cache[0].to(torch.int8)), "uint8"), (dict(ks=cache[2].float()), "fp16"),
            (dict(ks=None), "scales"), (dict(ks=cache[2][:, :, :8]), "scales must be"),
            (dict(vc=cache[1][:, :1]), "4-bit caches"), (dict(bs=32), "block_size"),
            (dict(bt=bt.long()), "int32"), (dict(ctx=ctx[:1]), "num_seqs"),
            (dict(q=q[:, :, :64], out=out[:, :, :64]), "match"), (dict(part=64), "partition"),
            (dict(q=q[:, :5].contiguous(), out=out[:, :5].contiguous()), "shape|size"),
            (dict(bt=bt.t().contiguous().t()), "contiguous"), (dict(ctx=ctx.cpu()), "device")]:
        with pytest.raises(RuntimeError, match=match):
            run(**kw)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 300])
def test_checked_decode_finds_an_empty_sequence(n):
    """Wherever it is, with the output left alone; the call after it, and one whose lengths
    come from work still queued, run as the unchecked call does."""
    import pa_int8

    cache, bt = paged([20 + i % 7 for i in range(n)], 2, 64, 16, torch.float16, n)
    g = torch.Generator(device=DEV).manual_seed(n)
    q = torch.randn(n, 8, 64, device=DEV, generator=g).half()
    ctx = torch.tensor([20 + i % 7 for i in range(n)], dtype=torch.int32, device=DEV)
    want = pa_int8.decode("int4", torch.empty_like(q), q, cache[0], cache[1], bt, ctx, 0.1, 16,
                          k_scales=cache[2], v_scales=cache[3], check=False)
    checked = lambda out, c: pa_int8.VARIANTS_INT4["int4"](out, q, *cache, bt, c, 0.1, 16)  # noqa: E731
    for bad in (0, -5, -2 ** 31):
        for at in {0, n // 2, n - 1}:
            c = ctx.clone()
            c[at] = bad
            out = torch.full_like(q, 7)
            with pytest.raises(RuntimeError, match="context_lens must be >= 1"):
                checked(out, c)
            assert bool((out == 7).all())
            assert torch.equal(checked(out, ctx), want)
    a = torch.randn(4096, 4096, device=DEV)
    for _ in range(60):
        a = (a @ a) * 1e-3
    late = (ctx.float() + 0 * a[0, 0].nan_to_num()).to(torch.int32)
    assert torch.equal(checked(torch.empty_like(q), late), want)
    pa_int8.ext()._length_slot(1)              # no memory to poll for the next check
    assert torch.equal(checked(torch.empty_like(q), ctx), want)
    pa_int8.ext()._length_slot(1)
    out = torch.full_like(q, 7)
    with pytest.raises(RuntimeError, match="context_lens must be >= 1"):
        checked(out, c)
    assert bool((out == 7).all())
    none = pa_int8.VARIANTS_INT4["int4"](q[:0].clone(), q[:0], *cache, bt[:0], ctx[:0], 0.1, 16)
    assert none.numel() == 0


def test_decode_same_bits_again_and_on_another_stream():
    import pa_int8

    lens = [5000, 17, 900, 64, 2500]
    out, q, cache, bt, ctx, scale = check_decode(lens, 16, 2, 128, 16, torch.bfloat16, 13)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2 = torch.empty_like(out)
        for _ in range(3):
            pa_int8.decode("int4", o2, q, cache[0], cache[1], bt, ctx, scale, 16,
                           k_scales=cache[2], v_scales=cache[3], check=False)
    torch.cuda.synchronize()
    assert torch.equal(out, o2)


def test_offsets_past_32_bits():
    """A cache whose codes take more than 4 GiB: rows at its far end."""
    import pa_int8

    hkv, d, bs = 8, 256, 128
    nb = (1 << 32) // (hkv * d // 2 * bs) + 9
    kc = torch.zeros((nb, hkv, bs // 4, d // 8, 4, 4), dtype=torch.uint8, device=DEV)
    vc = torch.zeros_like(kc)
    ks = torch.zeros((nb, hkv, bs, 2), dtype=torch.float16, device=DEV)
    vs = torch.zeros_like(ks)
    n = 200
    k, v = rows(n, hkv, d, torch.float16, 21)
    k, v = k.clamp(-50, 50), v.clamp(-50, 50)
    bt = torch.tensor([[nb - 1, nb - 4]], dtype=torch.int32, device=DEV)
    pos = torch.arange(n, device=DEV)
    slots = bt[0].long()[pos // bs] * bs + pos % bs
    pa_int8.reshape_and_cache_int4(k, v, kc, vc, ks, vs, slots)
    key, value = torch.empty_like(k), torch.empty_like(v)
    pa_int8.gather_cache_int4(key, value, kc, vc, ks, vs, slots)
    c, s, m = quantize64(k)
    want = s.double() * c.double() + m.double()
    assert bool(((key.double() - want).abs() <= EPS[torch.float16] * want.abs() + 2.0 ** -20).all())
    q = torch.randn(1, 16, d, device=DEV).half()
    out = torch.empty_like(q)
    ctx = torch.tensor([n], dtype=torch.int32, device=DEV)
    pa_int8.decode("int4", out, q, kc, vc, bt, ctx, 0.02, bs, k_scales=ks, v_scales=vs, check=False)
    blk = bt[0].long()
    small = [x[blk] for x in (kc, vc, ks, vs)]
    close(out, *decode64(q, *small, torch.tensor([[0, 1]], device=DEV), [n], 0.02), torch.float16)
