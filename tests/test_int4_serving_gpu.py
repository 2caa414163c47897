"""GPU tests of the 4-bit cache's operators together, as a serving loop uses them: blocks and
slots for the new tokens, their rows into the cache, decode over it, the cached rows read
back; eager, captured in a graph, in PagedKVCache and in the model bridge.

Decode outputs are compared with the 64-bit forms of test_int4_gpu under its tolerances.
"""

import math

import numpy as np
import pytest
import torch

from _qwen import tiny_qwen
from test_int4_gpu import EPS, close, decode64, new_cache, quantize64, rows, write64

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built):
    import pa_int8

    pa_int8.ext()


class Batch:
    """What a serving loop holds for one layer: the cache, the tables and the free list."""

    def __init__(self, seqs, hkv, d, bs, blocks, width, rows, seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)  # noqa: E731
        self.cache = new_cache(blocks, hkv, d, bs, fill=float("nan"))
        self.bt, self.ctx, self.new = i32(seqs, width), i32(seqs), i32(seqs)
        self.free = torch.randperm(blocks, device=DEV, generator=g).int()
        self.nfree = i32(1) + blocks
        self.slots = torch.zeros(rows, dtype=torch.int64, device=DEV)
        self.pos = torch.zeros_like(self.slots)
        self.cu, self.status, self.bs = i32(seqs + 1), i32(1), bs

    def step(self, q, out, k, v, scale):
        """New tokens' rows (in the order of the sequences) written, then decode of all."""
        import pa_int8

        pa_int8.extend_block_tables(self.bt, self.ctx, self.new, self.free, self.nfree, self.slots,
                                    self.pos, self.cu, self.status, self.bs)
        kc, vc, ks, vs = self.cache
        pa_int8.reshape_and_cache_int4(k, v, kc, vc, ks, vs, self.slots)
        pa_int8.decode("int4", out, q, kc, vc, self.bt, self.ctx, scale, self.bs, k_scales=ks,
                       v_scales=vs, check=False)


def token_rows(n, hkv, d, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kv = torch.randn(2, n, hkv, d, device=DEV, generator=g).to(dtype)
    return kv[0], kv[1]


def oracle_out(hist, q, scale, bs=16):
    """Decode over the sequences' own rows, quantized in 64 bits, sequence by sequence."""
    outs, offs = [], []
    for i, (k, v) in enumerate(hist):
        n = k.shape[0]
        nb = -(-n // bs)
        cache = new_cache(nb, k.shape[1], k.shape[2], bs)
        write64(k, v, torch.arange(n, device=DEV), *cache)
        bt = torch.arange(nb, device=DEV)[None]
        o, f = decode64(q[i:i + 1], *cache, bt, [n], scale)
        outs.append(o)
        offs.append(f)
    return torch.cat(outs), torch.cat(offs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,hkv,d,bs", [(12, 2, 128, 16), (32, 1, 64, 32), (4, 4, 200, 16)])
def test_prompts_then_decode_steps(heads, hkv, d, bs, dtype):
    """Ragged prompts (one of them empty until a later step), then steps of one token each."""
    lens, cap = [37, 0, 129, 16], sum([37, 0, 129, 16]) + 9
    b = Batch(4, hkv, d, bs, 40, 16, cap, 1)
    scale = 1 / math.sqrt(d)
    b.new.copy_(torch.tensor(lens, dtype=torch.int32))
    k, v = token_rows(cap, hkv, d, dtype, 2)
    q = torch.randn(4, heads, d, device=DEV).to(dtype)
    out = torch.empty_like(q)
    b.step(q, out, k, v, scale)
    assert b.status.item() == 0 and b.ctx.tolist() == lens
    at = np.cumsum([0] + lens)
    hist = [(k[at[i]:at[i + 1]], v[at[i]:at[i + 1]]) for i in range(4)]
    assert not bool(out[1].any())
    some = [0, 2, 3]
    close(out[some], *oracle_out([hist[i] for i in some], q[some], scale), dtype)
    # the cached rows read back, in order
    import pa_int8

    key, value = torch.empty_like(k), torch.empty_like(v)
    pa_int8.gather_cache_int4(key, value, *b.cache, b.slots)
    c, s, m = quantize64(k[:at[-1]])
    want = s.double() * c.double() + m.double()
    assert bool(((key[:at[-1]].double() - want).abs() <= EPS[dtype] * want.abs() + 2.0 ** -18).all())
    assert not bool(key[at[-1]:].any())
    # decode steps: rows behind the sequences' are skipped
    b.new.fill_(1)
    for t in range(20):
        k, v = token_rows(cap, hkv, d, dtype, 10 + t)
        q = torch.randn(4, heads, d, device=DEV).to(dtype)
        b.step(q, out, k, v, scale)
        hist = [(torch.cat([a, k[i:i + 1]]), torch.cat([c, v[i:i + 1]]))
                for i, (a, c) in enumerate(hist)]
    assert b.status.item() == 0 and b.ctx.tolist() == [n + 20 for n in lens]
    close(out, *oracle_out(hist, q, scale), dtype)


def test_captured_step_replayed():
    """The step captured once and replayed over new rows, with eager work and synchronizations
    between the replays: every replay equals the eager loop, tables and lengths included."""
    seqs, heads, hkv, d = 5, 16, 2, 128
    scale = 0.09
    pair = [Batch(seqs, hkv, d, 16, 64, 12, seqs, 3) for _ in range(2)]
    first = [torch.tensor([15, 1, 100, 31, 64], dtype=torch.int32, device=DEV)] * 2
    pk, pv = token_rows(211, hkv, d, torch.float16, 4)
    import pa_int8

    for b, n in zip(pair, first):
        slots = torch.zeros(211, dtype=torch.int64, device=DEV)
        pa_int8.extend_block_tables(b.bt, b.ctx, n, b.free, b.nfree, slots, None, None, b.status)
        pa_int8.reshape_and_cache_int4(pk, pv, *b.cache, slots)
        b.new.fill_(1)
    eager, cap = pair
    q = torch.zeros(seqs, heads, d, dtype=torch.float16, device=DEV)
    k, v = (torch.zeros(seqs, hkv, d, dtype=torch.float16, device=DEV) for _ in range(2))
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    state = lambda b: [b.bt, b.ctx, b.nfree, b.slots, b.pos, b.status] + list(b.cache)  # noqa: E731
    keep = [x.clone() for x in state(cap)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cap.step(q, out2, k, v, scale)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(state(cap), keep):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap.step(q, out2, k, v, scale)
    for t in range(30):
        k0, v0 = token_rows(seqs, hkv, d, torch.float16, 50 + t)
        k.copy_(k0)
        v.copy_(v0)
        q.copy_(torch.randn(seqs, heads, d, device=DEV))
        eager.step(q, out, k, v, scale)
        if t % 3 == 0:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert eager.status.item() == 0 and cap.status.item() == 0
        assert torch.equal(out, out2), t
        for x, y in zip(state(eager)[:5], state(cap)[:5]):
            assert torch.equal(x, y), t
    assert cap.ctx.tolist() == [45, 31, 130, 61, 94]


def test_two_streams_at_once():
    """Decodes of two batches on two streams, whose counters and workspaces are apart."""
    import pa_int8

    made = []
    for seed, lens in ((1, [9000, 40, 3000]), (2, [5000, 6000])):
        b = Batch(len(lens), 2, 128, 16, 1200, 700, sum(lens), seed)
        b.new.copy_(torch.tensor(lens, dtype=torch.int32))
        k, v = token_rows(sum(lens), 2, 128, torch.float16, seed)
        q = torch.randn(len(lens), 8, 128, device=DEV).half()
        out = torch.empty_like(q)
        b.step(q, out, k, v, 0.1)
        made.append((b, q, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    again = [[torch.empty_like(o) for _ in range(20)] for _, _, o in made]
    for i in range(20):
        for s, (b, q, _), outs in zip(streams, made, again):
            with torch.cuda.stream(s):
                kc, vc, ks, vs = b.cache
                pa_int8.decode("int4", outs[i], q, kc, vc, b.bt, b.ctx, 0.1, 16, k_scales=ks,
                               v_scales=vs, check=False)
    torch.cuda.synchronize()
    for (_, _, o), outs in zip(made, again):
        assert all(torch.equal(o, x) for x in outs)


# ------------------------------------------------------------------ the cache object

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("length", [1, 17, 64, 300])
def test_paged_cache_variant(length, dtype):
    import pa_int8

    c = pa_int8.PagedKVCache(2, 2, 128, 400, variant="int4_per_token", device=DEV)
    k, v = rows(length, 2, 128, dtype, length)
    k, v = k.clamp(-40, 40), v.clamp(-40, 40)
    c.prefill(1, k, v)
    hist = [k, v]
    for t in range(3):
        k1, v1 = token_rows(1, 2, 128, dtype, t)
        assert c.decode_append(1, k1[0], v1[0]) == length + t + 1
        hist = [torch.cat([hist[0], k1]), torch.cat([hist[1], v1])]
    k2, v2 = token_rows(21, 2, 128, dtype, 9)
    assert c.append_chunk(1, k2, v2) == length + 24
    hist = [torch.cat([hist[0], k2]), torch.cat([hist[1], v2])]
    slot = torch.tensor([length + 24], device=DEV)
    k1, v1 = token_rows(1, 2, 128, dtype, 11)
    c.append_at(1, k1[0], v1[0], slot)
    c.lengths[1] += 1
    hist = [torch.cat([hist[0], k1]), torch.cat([hist[1], v1])]
    q = torch.randn(1, 12, 128, device=DEV).to(dtype)
    out = torch.empty_like(q)
    pa_int8.VARIANTS_INT4["int4"](out, q, c.k_cache[1], c.v_cache[1], c.k_scales[1], c.v_scales[1],
                                  c.block_table, c.context_lens(1), 0.09, 16)
    close(out, *oracle_out([hist], q, 0.09), dtype)
    gk, gv = c.gather(1, dtype)
    for got, x in ((gk, hist[0]), (gv, hist[1])):
        codes, s, m = quantize64(x)
        want = s.double() * codes.double() + m.double()
        assert got.shape == x.shape
        assert bool(((got.double() - want).abs() <= EPS[dtype] * want.abs() + 2.0 ** -16).all())
    assert not bool(c.k_cache[0].any()) and c.lengths[0] == 0
    with pytest.raises(AssertionError, match="full"):
        c.append_chunk(1, *token_rows(400, 2, 128, dtype, 1))


# ------------------------------------------------------------------ the bridge

@pytest.fixture(scope="module", params=[torch.float16, torch.bfloat16])
def model(request):
    pytest.importorskip("transformers")
    from pa_int8 import qwen_bridge as br

    br.register()
    m = tiny_qwen(dtype=request.param, device="cuda")
    m.set_attn_implementation(br.ATTN_NAME)
    return m


def _cache(model, n):
    from pa_int8 import PagedKVCache

    cfg = model.config
    return PagedKVCache(cfg.num_hidden_layers, cfg.num_key_value_heads, 128, n,
                        variant="int4_per_token", device=DEV)


def test_bridge_graph_steps_equal_eager(model):
    from pa_int8 import qwen_bridge as br

    ids = torch.randint(0, 512, (1, 50), generator=torch.Generator().manual_seed(1)).cuda()
    a, _, _, la = br.generate_greedy(model, ids, 24, _cache(model, 128))
    b, _, _, lb = br.generate_greedy_graph(model, ids, 24, _cache(model, 128), keep_logits=True)
    assert torch.equal(a, b)
    for x, y in zip(la, lb):
        assert torch.equal(x, y)


def test_bridge_prompt_in_chunks(model):
    """A prompt fed in chunks: each attends to the cached values of those before it, causally to
    itself; checked against fp32 attention over the 64-bit dequantized prefix."""
    from pa_int8 import qwen_bridge as br

    dtype = model.dtype
    c = _cache(model, 200)
    br.set_active_cache(c)
    module = type("M", (), {"layer_idx": 0})()
    past = None
    try:
        for i, n in enumerate([40, 7, 2, 33]):
            g = torch.Generator(device=DEV).manual_seed(i)
            q = torch.randn(1, 12, n, 128, device=DEV, generator=g).to(dtype)
            k, v = (torch.randn(1, 2, n, 128, device=DEV, generator=g).to(dtype) for _ in range(2))
            out, _ = br.paged_bridge_attention(module, q, k, v, None)
            if past is None:
                kk, vv = k, v
            else:
                vals = []
                for x in past:
                    codes, s, m = quantize64(x)
                    vals.append((s.double() * codes.double() + m.double()).to(dtype))
                kk, vv = (torch.cat([a, b], 2) for a, b in zip(vals, (k, v)))
            want = br._causal_fp32(q.float(), kk.float(), vv.float(), 128 ** -0.5).transpose(1, 2)
            # the first chunk's attention rounds its weights to the type as well: two half steps of
            # the weighted magnitudes, at most the values' largest
            bound = 4 * EPS[dtype] * vv.float().abs().max()
            assert float((out.float() - want).abs().max()) <= bound
            past = ((k, v) if past is None else
                    tuple(torch.cat([a, b], 2) for a, b in zip(past, (k, v))))
        assert c.lengths[0] == 82
    finally:
        br.set_active_cache(None)
