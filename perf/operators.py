"""Measured calls of the 4-bit paged KV cache: its quantizing write, the read-back of cached
rows, decode attention over it, and the block tables and slot maps of a batch.

``run`` computes each of them in plain torch where ``own`` is false and through ``pa_int8``'s
entry points where it is true.  The cache holds, per (token, kv head) row of K and of V,
4-bit codes c and an fp16 pair (scale s, minimum m) that stand for the values s * c + m:

* codes   uint8 [blocks, kv_heads, block_size / 4, head_dim / 8, 4 tokens, 4 bytes], the
          four bytes being 8 dims, the lower dim of two in the lower half byte;
* scales  fp16 [blocks, kv_heads, block_size, 2].

Kinds of case:

* ``decode``  one decode call over a batch of cached sequences;
* ``write``   new rows quantized into the cache at their slots and read back as the values
              they stand for (what a prompt chunk attends over afterwards);
* ``gather``  rows of cached prefixes read back;
* ``extend``  a batch's tokens given blocks from the free list: tables, slots, positions.
"""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-pa-int8_amd")
DEV = "cuda"


def _ops():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import pa_int8
    return pa_int8


# ----------------------------------------------------------------------------- cases

def _decode(name, seqs, heads, kv_heads, head_dim, lens, lo, hi, dtype, block_size=16,
            table_tokens=0, check=False):
    return dict(name=name, kind="decode", seqs=seqs, heads=heads, kv_heads=kv_heads,
                head_dim=head_dim, lens=lens, lo=lo, hi=hi, dtype=dtype, block_size=block_size,
                table_tokens=table_tokens, check=check)


def _write(name, seqs, kv_heads, head_dim, lens, lo, hi, start, dtype, block_size=16, fused=False):
    return dict(name=name, kind="write", seqs=seqs, kv_heads=kv_heads, head_dim=head_dim,
                lens=lens, lo=lo, hi=hi, start=start, dtype=dtype, block_size=block_size,
                fused=fused)


def listed():
    return [
        # A handful of short chats, every head with its own K/V head: latency only.
        _decode("decode_tiny_mha", 4, 8, 8, 64, "uniform", 100, 512, "fp16"),
        # A mid-size serving batch of a 12/2-head model, by the checked call.
        _decode("decode_gqa_32x4096", 32, 12, 2, 128, "equal", 4096, 4096, "fp16", check=True),
        # Long documents at 32/8 heads: the largest read.
        _decode("decode_long_8x32k", 8, 32, 8, 128, "equal", 32768, 32768, "bf16"),
        # A continuous-batching mix at 32/8 heads: lognormal lengths of median 1024.
        _decode("decode_mix_192", 192, 32, 8, 128, "lognormal", 1024, 8192, "bf16"),
        # Wide heads, blocks of 32 tokens, tables sized for 16k tokens per sequence.
        _decode("decode_wide_24_d256", 24, 8, 4, 256, "uniform", 900, 9000, "fp16", 32, 16384),
        # A batch of ragged bf16 prompts into the cache, read back for their attention.
        _write("write_prompts_bf16", 48, 8, 128, "lognormal", 700, 8192, 0, "bf16"),
        # Prompt chunks that continue sequences at odd positions; K and V are views of a
        # fused QKV projection's rows.
        _write("write_chunks_fp16", 32, 8, 128, "uniform", 200, 1024, 1500, "fp16", 16, True),
        # New tokens of a decode batch, one per sequence.
        _write("write_append_256", 256, 8, 128, "equal", 1, 1, 3000, "bf16", 16, True),
        # The cached prefixes of a batch, read back for the attention of its next chunks.
        dict(name="gather_prefixes", kind="gather", seqs=16, kv_heads=8, head_dim=128,
             lens="lognormal", lo=2048, hi=16384, dtype="bf16", block_size=16),
        # One short prefix of a model with head_dim 80.
        dict(name="gather_short_d80", kind="gather", seqs=1, kv_heads=4, head_dim=80,
             lens="equal", lo=517, hi=517, dtype="fp16", block_size=16),
        # A decode step: one more token for each of 256 sequences.
        dict(name="extend_step_256", kind="extend", seqs=256, lens="equal", lo=1, hi=1, start=3000,
             block_size=16, pad=0),
        # The admission of 64 ragged prompts, token rows padded as a captured step has them.
        dict(name="extend_prompts_64", kind="extend", seqs=64, lens="lognormal", lo=900, hi=8192,
             start=0, block_size=16, pad=1000),
    ]


# No drawn case reads more cached values, or spans more when its lengths are padded to the
# longest, than the largest listed ones.
MAX_VALUES = 8 * 32768 * 8 * 128
MAX_PADDED = 4 * MAX_VALUES


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "write", "write", "gather", "extend"])
    head_dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    block_size = rng.choice([16, 16, 32, 64])
    heads, kv_heads = rng.choice([(8, 8), (8, 2), (8, 1), (16, 4), (12, 2), (32, 8), (32, 1),
                                  (28, 4)])
    dtype = rng.choice(["fp16", "bf16"])
    lens = rng.choice(["equal", "uniform", "lognormal"])

    def lengths(seqs, lo, padded):
        top = {"equal": 1, "uniform": 2, "lognormal": 4}[lens]
        per = kv_heads * head_dim
        while seqs > 1 and (2 * seqs * lo * per > MAX_VALUES or
                            padded and seqs * lo * top * per > MAX_PADDED):
            seqs = (seqs + 1) // 2
        return dict(seqs=seqs, lens=lens, lo=lo, hi=top * lo)

    if kind == "decode":
        d = lengths(_log_int(rng, 1, 256), _log_int(rng, 5, 32768), True)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                    block_size=block_size, table_tokens=rng.choice([0, 0, d["hi"] * 5 // 4]),
                    check=rng.random() < 0.3, **d)
    if kind == "write":
        fused = rng.random() < 0.5
        if rng.random() < 0.3:              # the append of a decode batch
            return dict(kind=kind, seqs=_log_int(rng, 1, 512), kv_heads=kv_heads,
                        head_dim=head_dim, lens="equal", lo=1, hi=1, start=_log_int(rng, 16, 8192),
                        dtype=dtype, block_size=block_size, fused=fused)
        d = lengths(_log_int(rng, 1, 48), _log_int(rng, 17, 4096), False)
        return dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                    start=rng.choice([0, 0, _log_int(rng, 1, 4096)]), block_size=block_size,
                    fused=fused, **d)
    if kind == "gather":
        return dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, dtype=dtype,
                    block_size=block_size, **lengths(_log_int(rng, 1, 32),
                                                     _log_int(rng, 5, 8192), False))
    lo = rng.choice([1, 1, _log_int(rng, 2, 2048)])
    return dict(kind=kind, seqs=_log_int(rng, 1, 512), lens="equal" if lo == 1 else lens, lo=lo,
                hi=lo if lo == 1 else 3 * lo, start=rng.choice([0, _log_int(rng, 1, 4096)]),
                block_size=block_size, pad=rng.choice([0, 0, 257]))


# ----------------------------------------------------------------------------- sizes

def _lens(case):
    """The sequence lengths (cached, or new), fixed by the case."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    if case["lens"] == "equal":
        return [lo] * n
    r = random.Random("%s %d %d %d" % (case["lens"], n, lo, hi))
    if case["lens"] == "uniform":
        return [r.randint(lo, hi) for _ in range(n)]
    return [int(min(max(round(r.lognormvariate(math.log(lo), 1.0)), 1), hi)) for _ in range(n)]


def _starts(case):
    return [case["start"] + 7 * s if case["start"] else 0 for s in range(case["seqs"])]


def _new_blocks(case):
    bs = case["block_size"]
    return sum(-(-(a + n) // bs) - -(-a // bs) for a, n in zip(_starts(case), _lens(case)))


def work(case):
    """Bytes: cached rows (codes and scales) once, queries, new rows, outputs, the table entries
    and lengths or the slots.  Flops: the two products of decode."""
    lens, kind, bs = _lens(case), case["kind"], case["block_size"]
    s, t = len(lens), sum(lens)
    if kind == "extend":
        # (start and new length in, new length and first row out; slot and position per row)
        return {"bytes": 16 * s + 16 * (t + case["pad"]) + 8 * _new_blocks(case), "flops": 0}
    d, hkv = case["head_dim"], case["kv_heads"]
    cached = t * hkv * (d + 8)
    if kind == "decode":
        return {"bytes": cached + 4 * s * case["heads"] * d + 4 * s + 4 * sum(-(-n // bs) for n in lens),
                "flops": 4 * t * case["heads"] * d}
    rows = t * hkv * 4 * d
    return {"bytes": cached + rows * (2 if kind == "write" else 1) + 8 * t, "flops": 0}


# ----------------------------------------------------------------------------- plain forms

def _quantize(x):
    """Codes (uint8, 0..15, round half even) and (scale, minimum) of rows, over the last axis.
    In 64 bits: the bf16 and fp16 grids put many values on the border of two codes."""
    lo, hi = x.amin(-1, keepdim=True).float(), x.amax(-1, keepdim=True).float()
    s = ((hi - lo) / 15).clamp(max=65504.0).to(torch.float16)
    m = lo.clamp(-65504.0, 65504.0).to(torch.float16)
    c = torch.round((x.double() - m.double()) / s.double()).clamp(0, 15)
    c = torch.where(s == 0, torch.zeros_like(c), c).to(torch.uint8)
    return c, torch.cat([s, m], -1)


def _pack(c):
    """Codes [..., D] -> bytes [..., D / 8, 4]."""
    c = c.reshape(*c.shape[:-1], c.shape[-1] // 8, 4, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _unpack(b):
    """Bytes [..., D / 8, 4] -> codes [..., D]."""
    return torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-2], b.shape[-2] * 8)


def _put(st, slots, k, v):
    """Rows into the cache at their slots."""
    bs = st["ks"].shape[2]
    blk, off = slots // bs, slots % bs
    for x, cache, scales in ((k, st["kc"], st["ks"]), (v, st["vc"], st["vs"])):
        c, sm = _quantize(x)
        cache[blk, :, off // 4, :, off % 4] = _pack(c)
        scales[blk, :, off] = sm


def _rows(cache, scales, slots, dtype):
    """The values of the cached rows at the slots, [T, kv_heads, D]."""
    bs = scales.shape[2]
    blk, off = slots // bs, slots % bs
    c = _unpack(cache[blk, :, off // 4, :, off % 4]).float()
    sm = scales[blk, :, off].float()
    return (c * sm[..., :1] + sm[..., 1:]).to(dtype)


def _dense(cache, scales, bt):
    """[S, kv_heads, table tokens, D] fp32 values behind the block table."""
    s, mb = bt.shape
    c = _unpack(cache[bt].permute(0, 2, 1, 3, 5, 4, 6)).float()     # [S, Hkv, MB, bs/4, 4, D]
    sm = scales[bt].permute(0, 2, 1, 3, 4).float()
    hkv, bs, d = c.shape[1], scales.shape[2], c.shape[-1]
    c = c.reshape(s, hkv, mb * bs, d)
    sm = sm.reshape(s, hkv, mb * bs, 2)
    return c.mul_(sm[..., :1]).add_(sm[..., 1:])


def _plain_decode(st):
    q, bt, ctx = st["q"], st["bt"].long(), st["ctx"]
    s, h, d = q.shape
    k = _dense(st["kc"], st["ks"], bt)
    hkv, n = k.shape[1], k.shape[2]
    p = torch.matmul(q.float().reshape(s, hkv, h // hkv, d), k.transpose(-1, -2).contiguous())
    del k
    p = p * st["scale"]
    live = torch.arange(n, device=DEV)[None, :] < ctx[:, None]
    p = p.masked_fill(~live[:, None, None, :], float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    v = _dense(st["vc"], st["vs"], bt)
    # (values behind a sequence's end may be anything)
    v = v.masked_fill_(~live[:, None, :, None], 0.0)
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return out.reshape(s, h, d).to(q.dtype)


def _plain_extend(st):
    bt, ctx, new = st["bt"], st["ctx"].long(), st["new"].long()
    bs, rows, free = st["bs"], st["slots"].shape[0], st["num_free"].long()
    have, want = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    need = want - have
    first = torch.cumsum(need, 0) - need
    j = torch.arange(bt.shape[1], device=DEV)[None, :]
    take = (j >= have[:, None]) & (j < want[:, None])
    at = free - 1 - (first[:, None] + j - have[:, None])
    table = torch.where(take, st["free"][at.clamp(0, st["free"].shape[0] - 1)], bt)
    ends = torch.cumsum(new, 0)
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(ends, row, right=True).clamp(max=bt.shape[0] - 1)
    pos = ctx[seq] + row - (ends - new)[seq]
    live = row < ends[-1]
    blk = table[seq, (pos // bs).clamp(0, bt.shape[1] - 1)]
    slots = torch.where(live, blk.long() * bs + pos % bs, torch.full_like(pos, -1))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), ends]).to(torch.int32)
    status = (need.sum() > free) * 1 + (want.amax() > bt.shape[1]) * 2 + (ends[-1:] > rows) * 4
    return [table, (ctx + new).to(torch.int32), (free - need.sum()).to(torch.int32), slots,
            torch.where(live, pos, torch.zeros_like(pos)), cu, status.to(torch.int32)]


# ----------------------------------------------------------------------------- inputs

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _tables(lens, bs, capacity, gen):
    """Randomly permuted physical blocks: (table [S, capacity blocks], blocks in the pool)."""
    nblk = torch.tensor([-(-n // bs) for n in lens], device=DEV)
    nb, width = int(nblk.sum()) + 1, max(int(nblk.max()), -(-capacity // bs))
    perm = torch.randperm(nb, device=DEV, generator=gen).to(torch.int32)
    j = torch.arange(width, device=DEV)[None, :]
    first = torch.cumsum(nblk, 0) - nblk
    bt = torch.where(j < nblk[:, None], perm[(first[:, None] + j).clamp(max=nb - 1)], 0)
    return bt.to(torch.int32), nb


def _slots(bt, lens, starts, bs):
    """The slots of `lens[s]` tokens of sequence s from position `starts[s]` on, in order."""
    n, a = torch.tensor(lens, device=DEV), torch.tensor(starts, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), n)
    pos = torch.arange(seq.shape[0], device=DEV) - (torch.cumsum(n, 0) - n)[seq] + a[seq]
    return bt[seq, pos // bs].to(torch.int64) * bs + pos % bs


def _empty_cache(nb, hkv, d, bs):
    z = lambda *shape, **kw: torch.zeros(shape, device=DEV, **kw)  # noqa: E731
    return dict(kc=z(nb, hkv, bs // 4, d // 8, 4, 4, dtype=torch.uint8),
                vc=z(nb, hkv, bs // 4, d // 8, 4, 4, dtype=torch.uint8),
                ks=z(nb, hkv, bs, 2, dtype=torch.float16), vs=z(nb, hkv, bs, 2, dtype=torch.float16))


def _full_cache(nb, hkv, d, bs, gen):
    """A full cache of quantized rows: N(0,1) values, for K about channel means, as keys have."""
    st = _empty_cache(nb, hkv, d, bs)
    mean = torch.randn(hkv, 1, d, device=DEV, generator=gen)
    step = max(1, (1 << 27) // (hkv * d * bs))
    for i in range(0, nb, step):
        n = min(step, nb - i)
        for cache, scales, mu in ((st["kc"], st["ks"], mean), (st["vc"], st["vs"], 0.0)):
            x = torch.randn(n, hkv, bs, d, device=DEV, generator=gen) + mu
            c, sm = _quantize(x.to(torch.bfloat16))
            cache[i:i + n] = _pack(c).view(n, hkv, bs // 4, 4, d // 8, 4).transpose(3, 4)
            scales[i:i + n] = sm
    return st


def prepare(case, seed):
    gen, kind, bs = _gen(seed), case["kind"], case["block_size"]
    lens = _lens(case)
    if kind == "extend":
        starts = _starts(case)
        used = [-(-a // bs) for a in starts]
        top = max(-(-(a + n) // bs) for a, n in zip(starts, lens))
        width, pool = top + 5, sum(used) + _new_blocks(case) + 100
        perm = torch.randperm(pool, device=DEV, generator=gen).to(torch.int32)
        u = torch.tensor(used, device=DEV)
        j = torch.arange(width, device=DEV)[None, :]
        first = torch.cumsum(u, 0) - u
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        rows = sum(lens) + case["pad"]
        st = dict(bt=torch.where(j < u[:, None], perm[(first[:, None] + j).clamp(max=pool - 1)], 0)
                  .to(torch.int32), ctx=i32(starts), new=i32(lens), bs=bs,
                  free=perm[sum(used):].contiguous(), num_free=i32([pool - sum(used)]),
                  slots=torch.empty(rows, dtype=torch.int64, device=DEV),
                  pos=torch.empty(rows, dtype=torch.int64, device=DEV),
                  cu=torch.empty(len(lens) + 1, dtype=torch.int32, device=DEV),
                  status=i32([0]), ctx_out=i32(starts), free_out=i32([0]))
        return dict(st, case=case)
    hkv, d, dt = case["kv_heads"], case["head_dim"], _dtype(case)
    if kind == "write":
        starts, t = _starts(case), sum(lens)
        bt, nb = _tables([a + n for a, n in zip(starts, lens)], bs, 0, gen)
        st = _empty_cache(nb, hkv, d, bs)
        mean = torch.randn(hkv, d, device=DEV, generator=gen)
        extra = 4 * hkv if case["fused"] else 0
        rows = torch.randn(t, extra + 2 * hkv, d, device=DEV, generator=gen)
        rows[:, extra:extra + hkv] += mean
        rows = rows.to(dt)
        k, v = rows[:, extra:extra + hkv], rows[:, extra + hkv:]
        if not case["fused"]:
            k, v = k.contiguous(), v.contiguous()
        return dict(st, case=case, k=k, v=v, slots=_slots(bt, lens, starts, bs),
                    key=torch.empty(t, hkv, d, dtype=dt, device=DEV),
                    value=torch.empty(t, hkv, d, dtype=dt, device=DEV))
    bt, nb = _tables(lens, bs, case.get("table_tokens", 0), gen)
    st = dict(_full_cache(nb, hkv, d, bs, gen), case=case)
    if kind == "gather":
        t = sum(lens)
        return dict(st, slots=_slots(bt, lens, [0] * len(lens), bs),
                    key=torch.empty(t, hkv, d, dtype=dt, device=DEV),
                    value=torch.empty(t, hkv, d, dtype=dt, device=DEV))
    q = torch.randn(len(lens), case["heads"], d, device=DEV, generator=gen).to(dt)
    return dict(st, bt=bt, q=q, out=torch.empty_like(q), scale=1.0 / math.sqrt(d),
                ctx=torch.tensor(lens, dtype=torch.int32, device=DEV))


# ----------------------------------------------------------------------------- passes

def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind == "decode":
            return _plain_decode(st)
        if kind == "extend":
            return _plain_extend(st)
        if kind == "write":
            _put(st, st["slots"], st["k"], st["v"])
        dt = _dtype(case)
        return [_rows(st["kc"], st["ks"], st["slots"], dt),
                _rows(st["vc"], st["vs"], st["slots"], dt)]
    ops = _ops()
    if kind == "decode":
        return ops.decode("int4", st["out"], st["q"], st["kc"], st["vc"], st["bt"], st["ctx"],
                          st["scale"], case["block_size"], k_scales=st["ks"], v_scales=st["vs"],
                          check=case["check"])
    if kind == "extend":
        ops.extend_block_tables(st["bt"], st["ctx"], st["new"], st["free"], st["num_free"],
                                st["slots"], st["pos"], st["cu"], st["status"], st["bs"],
                                context_lens_out=st["ctx_out"], num_free_out=st["free_out"])
        return [st["bt"], st["ctx_out"], st["free_out"], st["slots"], st["pos"], st["cu"],
                st["status"]]
    if kind == "write":
        ops.reshape_and_cache_int4(st["k"], st["v"], st["kc"], st["vc"], st["ks"], st["vs"],
                                   st["slots"])
    ops.gather_cache_int4(st["key"], st["value"], st["kc"], st["vc"], st["ks"], st["vs"],
                          st["slots"])
    return [st["key"], st["value"]]


# ----------------------------------------------------------------------------- 64 bits

def _bytes_to_values(cache, scales):
    """[blocks, kv_heads, block_size, D] float64 values of whole cache blocks."""
    nb, hkv, quads, chunks = cache.shape[:4]
    val = torch.empty(nb, hkv, quads, 4, chunks, 4, 2, dtype=torch.float64, device=DEV)
    b = cache.transpose(3, 4).to(torch.int64)
    val[..., 0], val[..., 1] = (b % 16).double(), (b // 16).double()
    val = val.reshape(nb, hkv, quads * 4, chunks * 8)
    return val * scales[..., 0:1].double() + scales[..., 1:2].double()


def exact(case, seed):
    if case["kind"] == "extend":
        return None                       # whole numbers: nothing is rounded
    st = prepare(case, seed)
    if case["kind"] == "write":
        res = []
        for x in (st["k"].double(), st["v"].double()):
            lo, hi = x.min(-1).values, x.max(-1).values
            m, s = lo.half().double().unsqueeze(-1), ((hi - lo) / 15).half().double().unsqueeze(-1)
            c = torch.where(s > 0, ((x - m) / s).round().clamp(0, 15), 0.0)
            res.append(s * c + m)
        return res
    bs = case["block_size"]
    if case["kind"] == "gather":
        res = []
        for cache, scales in ((st["kc"], st["ks"]), (st["vc"], st["vs"])):
            flat = _bytes_to_values(cache, scales).transpose(1, 2).reshape(-1, *st["key"].shape[1:])
            res.append(flat[st["slots"]])
        return res
    q, h, hkv = st["q"].double(), case["heads"], case["kv_heads"]
    g = h // hkv
    out = torch.empty_like(q)
    for i, n in enumerate(_lens(case)):
        blk = st["bt"][i, :-(-n // bs)].long()
        k = _bytes_to_values(st["kc"][blk], st["ks"][blk])
        v = _bytes_to_values(st["vc"][blk], st["vs"][blk])
        for j in range(hkv):
            kj = k[:, j].reshape(-1, k.shape[-1])[:n]
            vj = v[:, j].reshape(-1, v.shape[-1])[:n]
            a = torch.softmax(torch.mm(q[i, j * g:(j + 1) * g], kj.t().contiguous()) * st["scale"], -1)
            out[i, j * g:(j + 1) * g] = torch.mm(a, vj)
    return out
