"""CPU tests of the 4-bit cache's host side: what the C entry points and the torch ops refuse
before any device access, sizes, and the cache object's accounting."""

import pytest
import torch

OK, NULL, SHAPE, BLOCK, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3, 4, 5
P = 0x10000            # an aligned address that is never read


@pytest.fixture(scope="module")
def lib(built):
    import pa_int8

    return pa_int8.capi()


def rows_args(**kw):
    a = dict(key=P, value=P, kts=1024, khs=128, vts=1024, vhs=128, slots=P, tokens=5, hkv=8, d=128,
             kc=P, vc=P, ks=P, vs=P, blocks=10, bs=16, bf16=0, stream=None)
    a.update(kw)
    return [a[n] for n in ("key", "value", "kts", "khs", "vts", "vhs", "slots", "tokens", "hkv", "d",
                           "kc", "vc", "ks", "vs", "blocks", "bs", "bf16", "stream")]


@pytest.mark.parametrize("entry", ["pa_reshape_and_cache_int4", "pa_gather_cache_int4"])
@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), OK), (dict(tokens=0, key=None), OK), (dict(tokens=-1), SHAPE),
    (dict(key=None), NULL), (dict(value=None), NULL), (dict(slots=None), NULL),
    (dict(kc=None), NULL), (dict(vc=None), NULL), (dict(ks=None), NULL), (dict(vs=None), NULL),
    (dict(bs=8), BLOCK), (dict(bs=24), BLOCK), (dict(bs=256), BLOCK), (dict(bs=0), BLOCK),
    (dict(bs=-16), BLOCK), (dict(d=0), UNSUPPORTED), (dict(d=100), UNSUPPORTED),
    (dict(d=264), UNSUPPORTED), (dict(hkv=0), SHAPE), (dict(blocks=0), SHAPE),
    (dict(kts=1028), SHAPE), (dict(khs=-128), SHAPE), (dict(vts=4), SHAPE),
    (dict(key=P + 8), SHAPE), (dict(kc=P + 4), SHAPE), (dict(ks=P + 2), SHAPE),
    (dict(slots=P + 4), SHAPE), (dict(blocks=2 ** 31 - 1, hkv=4), SHAPE)])
def test_rows_refusals(lib, entry, kw, status):
    assert getattr(lib, entry)(*rows_args(**kw)) == status


def decode_args(**kw):
    a = dict(out=P, q=P, kc=P, vc=P, ks=P, vs=P, bt=P, ctx=P, scale=0.1, bs=16, seqs=2, heads=8,
             d=128, hkv=2, blocks=10, mb=4, bf16=0, cnt=P, cb=1 << 20, ws=P, wb=1 << 30, stream=None)
    a.update(kw)
    return [a[n] for n in ("out", "q", "kc", "vc", "ks", "vs", "bt", "ctx", "scale", "bs", "seqs",
                           "heads", "d", "hkv", "blocks", "mb", "bf16", "cnt", "cb", "ws", "wb",
                           "stream")]


@pytest.mark.parametrize("kw,status", [
    (dict(seqs=0), OK), (dict(seqs=-1), SHAPE), (dict(heads=0), SHAPE), (dict(heads=9), SHAPE),
    (dict(d=12), UNSUPPORTED), (dict(bs=48), BLOCK), (dict(mb=-1), SHAPE), (dict(out=None), NULL),
    (dict(q=None), NULL), (dict(kc=None), NULL), (dict(vs=None), NULL), (dict(bt=None), NULL),
    (dict(ctx=None), NULL), (dict(out=P + 8), SHAPE), (dict(q=P + 2), SHAPE),
    (dict(cnt=None), WORKSPACE), (dict(cb=100), WORKSPACE), (dict(cnt=P + 4), WORKSPACE),
    (dict(ws=None), WORKSPACE), (dict(wb=1000), WORKSPACE), (dict(ws=P + 16), WORKSPACE),
    (dict(mb=2 ** 27), SHAPE), (dict(seqs=2 ** 20, mb=2 ** 16), SHAPE),
    (dict(blocks=2 ** 31 - 1, hkv=8), SHAPE)])
def test_decode_refusals(lib, kw, status):
    assert lib.pa_paged_decode_attn_int4(*decode_args(**kw)) == status


@pytest.mark.parametrize("kw,report,status", [
    (dict(), None, NULL), (dict(), P + 4, SHAPE), (dict(q=None), P, NULL), (dict(wb=0), P, WORKSPACE),
    (dict(seqs=0), P, OK), (dict(d=12), P, UNSUPPORTED)])
def test_checked_decode_refusals(lib, kw, report, status):
    args = decode_args(**kw)
    args[-1:-1] = [report, 7]
    assert lib.pa_paged_decode_attn_int4_checked(*args) == status


def test_decode_sizes(lib):
    ws = lib.pa_decode_int4_workspace_bytes
    assert lib.pa_decode_int4_counter_bytes() <= 256 << 10
    assert 0 < ws(4, 8, 128, 8, 16, 100) <= 16 << 20
    # the same whatever the batch: pieces of work-groups, not of sequences
    assert ws(4, 8, 128, 8, 16, 100) == ws(500, 8, 128, 8, 16, 9000)
    assert ws(1, 32, 128, 1, 16, 10) == ws(1, 40, 128, 1, 16, 10) > ws(1, 16, 128, 1, 16, 10)
    for bad in ((1, 8, 100, 8, 16, 1), (1, 8, 128, 3, 16, 1), (1, 8, 128, 8, 20, 1)):
        assert ws(*bad) == 0


def extend_args(**kw):
    a = dict(bt=P, ctx=P, new=P, free=P, nfree=P, ctxo=P, nfo=P, slots=P, pos=None, cu=None, st=P,
             seqs=3, mb=4, bs=16, rows=8, cap=9, cnt=P, cb=4, stream=None)
    a.update(kw)
    return [a[n] for n in ("bt", "ctx", "new", "free", "nfree", "ctxo", "nfo", "slots", "pos", "cu",
                           "st", "seqs", "mb", "bs", "rows", "cap", "cnt", "cb", "stream")]


@pytest.mark.parametrize("kw,status", [
    (dict(seqs=0), SHAPE), (dict(seqs=4097), SHAPE), (dict(mb=-1), SHAPE), (dict(rows=-1), SHAPE),
    (dict(cap=-1), SHAPE), (dict(mb=2 ** 30), SHAPE), (dict(bs=0), BLOCK), (dict(bs=24), BLOCK),
    (dict(bs=256), BLOCK), (dict(bt=None), NULL), (dict(ctx=None), NULL), (dict(new=None), NULL),
    (dict(free=None), NULL), (dict(nfree=None), NULL), (dict(ctxo=None), NULL),
    (dict(nfo=None), NULL), (dict(slots=None), NULL), (dict(st=None), NULL),
    (dict(cnt=None), WORKSPACE), (dict(cb=0), WORKSPACE), (dict(cnt=P + 2), WORKSPACE)])
def test_extend_refusals(lib, kw, status):
    assert lib.pa_extend_block_tables(*extend_args(**kw)) == status


APART = {n: P + 4096 * (i + 1) for i, n in enumerate(
    ("bt", "ctx", "new", "free", "nfree", "ctxo", "nfo", "slots", "pos", "cu", "st"))}


@pytest.mark.parametrize("out", ["bt", "ctxo", "nfo", "slots", "pos", "cu", "st"])
def test_extend_outputs_stand_alone(lib, out):
    """An output that shares memory with another tensor is refused, by one element too."""
    size = dict(bt=48, ctx=12, new=12, free=36, nfree=4, ctxo=12, nfo=4, slots=64, pos=64, cu=16,
                st=4)
    for other, n in size.items():
        if other == out:
            continue
        for at in (APART[other] + n - 4, APART[other] - size[out] + 4):
            if at == APART[other] and (out, other) in (("ctxo", "ctx"), ("nfo", "nfree")):
                continue                   # (updated in place)
            assert lib.pa_extend_block_tables(*extend_args(**{**APART, out: at})) == SHAPE, other


def test_ops_reject_cpu_tensors(built):
    import pa_int8

    c = torch.zeros(4, 2, 4, 16, 4, 4, dtype=torch.uint8)
    s = torch.zeros(4, 2, 16, 2, dtype=torch.float16)
    x = torch.zeros(3, 2, 128, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int64)
    n = torch.ones(3, dtype=torch.int32)
    q = torch.zeros(3, 8, 128, dtype=torch.float16)
    bt = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa_int8.reshape_and_cache_int4(x, x, c, c, s, s, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa_int8.gather_cache_int4(x, x, c, c, s, s, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa_int8.VARIANTS_INT4["int4"](q, q, c, c, s, s, bt, n, 0.1, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        pa_int8.extend_block_tables(bt, n, n, n, n[:1], i, i, None, n[:1])
    with pytest.raises(RuntimeError, match="scales"):
        pa_int8.decode("int4", q, q, c, c, bt, n, 0.1)


def test_cache_object_accounting():
    import pa_int8

    kw = dict(num_layers=3, num_kv_heads=2, head_dim=128, max_len=2048, device="cpu")
    c = pa_int8.PagedKVCache(variant="int4_per_token", **kw)
    i8 = pa_int8.PagedKVCache(variant="int8_per_token", **kw)
    assert c.is_int4 and not c.is_int8 and i8.is_int8 and not i8.is_int4
    assert c.k_cache.shape == (3, 128, 2, 4, 16, 4, 4) and c.k_cache.dtype == torch.uint8
    assert c.v_scales.shape == (3, 128, 2, 16, 2) and c.v_scales.dtype == torch.float16
    # a token and head: 64 bytes of codes and 4 of scale and minimum, K and V
    assert c.layout.block_bytes() == 2 * 2 * 16 * (64 + 4)
    assert c.kv_bytes() == c.kv_bytes_for_len(2048) == 3 * 128 * c.layout.block_bytes()
    assert c.kv_bytes() / i8.kv_bytes() < 0.52
    with pytest.raises(RuntimeError, match="int4_per_token"):
        i8.gather(0)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.prefill(0, torch.zeros(5, 2, 128, dtype=torch.float16),
                  torch.zeros(5, 2, 128, dtype=torch.float16))


def test_python_names():
    import pa_int8

    assert set(pa_int8.VARIANTS_INT4) == {"int4"}
    for name in ("reshape_and_cache_int4", "gather_cache_int4", "extend_block_tables"):
        assert callable(getattr(pa_int8, name))
