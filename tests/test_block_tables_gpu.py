"""GPU tests of extend_block_tables: blocks from the free list, slots and positions of new
tokens, against a restatement in Python integers.  Everything is whole numbers: equal."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built):
    import pa_int8

    pa_int8.ext()


def plain(bt, ctx, new, free, nfree, rows, bs):
    """(table, lengths, free count, slots, positions, cu, status) on lists."""
    bt, mb = [list(r) for r in bt], len(bt[0])
    st, need, cu = 0, 0, [0]
    for c, n in zip(ctx, new):
        if c < 0 or n < 0:
            st |= 8
            continue
        want = -(-(c + n) // bs)
        if want > mb or c + n > 2 ** 31 - 1:
            st |= 2
        need += want - -(-c // bs)
        cu.append(cu[-1] + n)
    if nfree < 0 or nfree > len(free):
        st |= 8
    elif need > nfree:
        st |= 1
    if cu[-1] > rows:
        st |= 4
    if st:
        return bt, list(ctx), nfree, [-1] * rows, [0] * rows, [0] * (len(ctx) + 1), st
    slots, pos, out = [], [], []
    for s, (c, n) in enumerate(zip(ctx, new)):
        for j in range(-(-c // bs), -(-(c + n) // bs)):
            nfree -= 1
            bt[s][j] = free[nfree]
        for p in range(c, c + n):
            slots.append(bt[s][p // bs] * bs + p % bs)
            pos.append(p)
        out.append(c + n)
    pad = rows - len(slots)
    return bt, out, nfree, slots + [-1] * pad, pos + [0] * pad, cu, 0


def tensors(ctx, new, bs, mb, spare, rows, seed):
    g = torch.Generator().manual_seed(seed)
    used = [-(-max(c, 0) // bs) for c in ctx]
    need = sum(-(-(max(c, 0) + max(n, 0)) // bs) for c, n in zip(ctx, new)) - sum(used)
    pool = sum(used) + max(need, 0) + spare + 3
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    bt = torch.full((len(ctx), mb), -9, dtype=torch.int32)
    at = 0
    for s, u in enumerate(used):
        bt[s, :min(u, mb)] = perm[at:at + u][:mb]
        at += u
    free = perm[at:]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(bt=bt.to(DEV), ctx=i32(ctx), new=i32(new), free=free.to(DEV).contiguous(),
                nfree=i32([max(need, 0) + spare]),
                slots=torch.full((rows,), 77, dtype=torch.int64, device=DEV),
                pos=torch.full((rows,), 77, dtype=torch.int64, device=DEV),
                cu=torch.full((len(ctx) + 1,), 77, dtype=torch.int32, device=DEV), st=i32([77]))


def run(t, bs, **out):
    import pa_int8

    pa_int8.extend_block_tables(t["bt"], t["ctx"], t["new"], t["free"], t["nfree"], t["slots"],
                                t["pos"], t["cu"], t["st"], bs, **out)


def expect(t, bs, rows):
    return plain(t["bt"].tolist(), t["ctx"].tolist(), t["new"].tolist(), t["free"].tolist(),
                 int(t["nfree"]), rows, bs)


def check(t, want, ctx=None, nfree=None):
    assert t["st"].tolist() == [want[6]]
    assert t["bt"].tolist() == want[0]
    assert (t["ctx"] if ctx is None else ctx).tolist() == want[1]
    assert (t["nfree"] if nfree is None else nfree).tolist() == [want[2]]
    assert t["slots"].tolist() == want[3] and t["pos"].tolist() == want[4]
    assert t["cu"].tolist() == want[5]


CASES = [  # lengths, new tokens, block size, spare rows
    ([0], [1], 16, 0), ([0], [0], 16, 0), ([16], [1], 16, 3), ([15, 16, 17], [1, 1, 1], 16, 0),
    ([0, 31, 0, 5, 0], [7, 0, 64, 1, 0], 16, 11), ([3000 + 7 * i for i in range(256)], [1] * 256, 16, 0),
    ([0] * 64, [100 + 37 * i for i in range(64)], 16, 1000), ([5] * 1025, [3] * 1025, 32, 1),
    ([i % 9 for i in range(4096)], [i % 5 for i in range(4096)], 8, 100),
    ([100, 200], [30000, 9], 128, 0), ([0] * 5, [0] * 5, 16, 40), ([1, 2, 3], [2, 2, 2], 1, 0),
]


@pytest.mark.parametrize("ctx,new,bs,pad", CASES)
@pytest.mark.parametrize("inplace", [True, False])
def test_extend(ctx, new, bs, pad, inplace):
    rows = sum(new) + pad
    mb = max(-(-(c + n) // bs) for c, n in zip(ctx, new)) + 2
    t = tensors(ctx, new, bs, mb, 5, rows, len(ctx))
    want = expect(t, bs, rows)
    assert want[6] == 0
    if inplace:
        run(t, bs)
        check(t, want)
    else:
        keep = t["ctx"].clone(), t["nfree"].clone()
        o = torch.full_like(t["ctx"], 77), torch.full_like(t["nfree"], 77)
        for _ in range(2):                  # the inputs are left as they are: the same again
            run(t, bs, context_lens_out=o[0], num_free_out=o[1])
            check(t, want, *o)
        assert torch.equal(t["ctx"], keep[0]) and torch.equal(t["nfree"], keep[1])


@pytest.mark.parametrize("what,status", [("blocks", 1), ("row", 2), ("rows", 4), ("length", 8),
                                         ("new", 8), ("free", 8), ("free_low", 8), ("both", 3),
                                         ("sum", 6)])
def test_what_does_not_fit_places_nothing(what, status):
    ctx, new, bs, rows, mb = [10, 40, 0], [30, 50, 8000], 16, 8200, 512
    t = tensors(ctx, new, bs, mb, 0, rows, 3)
    if what in ("blocks", "both"):
        t["nfree"] -= 1
    if what in ("row", "both"):
        t["bt"] = t["bt"][:, :499].contiguous()
    if what == "rows":
        t["slots"], t["pos"], rows = t["slots"][:8079], t["pos"][:8079], 8079
    if what == "length":
        t["ctx"][1] = -1
    if what == "new":
        t["new"][2] = -5
    if what == "free":
        t["nfree"] += 100
    if what == "free_low":
        t["nfree"].fill_(-1)
    if what == "sum":                       # sums past 32 bits
        t["new"].fill_(2 ** 31 - 1)
        t["nfree"].fill_(0)
        status = 7
    want = expect(t, bs, rows)
    assert want[6] == status
    run(t, bs)
    check(t, want)


def test_optional_outputs_and_several_steps():
    """Steps of one token, in place, without positions and starts, across block borders."""
    import pa_int8

    ctx = [0, 15, 31, 16]
    t = tensors(ctx, [40] * 4, 16, 8, 0, 4, 4)
    t["new"].fill_(1)
    for _ in range(40):
        want = expect(t, 16, 4)
        pa_int8.extend_block_tables(t["bt"], t["ctx"], t["new"], t["free"], t["nfree"], t["slots"],
                                    None, None, t["st"])
        assert t["st"].item() == 0 and t["slots"].tolist() == want[3]
        assert t["bt"].tolist() == want[0] and t["ctx"].tolist() == want[1]
    assert t["nfree"].item() == 0
    want = expect(t, 16, 4)
    run(t, 16)
    assert want[6] in (0, 1)
    check(t, want)


def test_several_calls_captured_into_a_graph():
    """Two steps and a chunk, in place, replayed: each replay goes on from the last one."""
    ctx, bs = [5, 0, 47, 16], 16
    t = tensors(ctx, [80] * 4, bs, 9, 0, 700, 11)
    steps = [[1, 1, 1, 1], [0, 12, 1, 0], [2, 1, 0, 2]]
    news = [torch.tensor(n, dtype=torch.int32, device=DEV) for n in steps]
    outs = [{k: torch.empty_like(t[k]) for k in ("slots", "pos", "cu", "st")} for _ in steps]
    calls = [{**t, **o, "new": n} for o, n in zip(outs, news)]
    start = {k: t[k].clone() for k in ("bt", "ctx", "nfree")}
    for c in calls:                        # (outside a capture first)
        run(c, bs)
    torch.cuda.synchronize()
    for k, v in start.items():
        t[k].copy_(v)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for c in calls:
            run(c, bs)
    for _ in range(3):
        state = [t["bt"].tolist(), t["ctx"].tolist(), int(t["nfree"])]
        g.replay()
        torch.cuda.synchronize()
        for c, n in zip(calls, steps):
            want = plain(state[0], state[1], n, t["free"].tolist(), state[2], 700, bs)
            state = [want[0], want[1], want[2]]
            assert want[6] == 0 and c["st"].item() == 0
            assert c["slots"].tolist() == want[3] and c["pos"].tolist() == want[4]
            assert c["cu"].tolist() == want[5]
        assert t["bt"].tolist() == state[0] and t["ctx"].tolist() == state[1]
        assert t["nfree"].item() == state[2]


def test_refusals():
    import pa_int8

    t = tensors([3, 4], [1, 1], 16, 4, 2, 2, 5)
    args = ["bt", "ctx", "new", "free", "nfree", "slots", "pos", "cu", "st"]

    def call(bs=16, **kw):
        pa_int8.extend_block_tables(*[kw.get(n, t[n]) for n in args], bs)

    for kw, match in [(dict(bt=t["bt"].long()), "int32"), (dict(ctx=t["ctx"][:1]), "num_seqs"),
                      (dict(slots=t["slots"].int()), "int64"), (dict(pos=t["pos"][:1]), "positions"),
                      (dict(cu=t["cu"][:2]), "cu_seqlens"), (dict(st=t["cu"]), "one value"),
                      (dict(free=t["free"].cpu()), "device"), (dict(bs=24), "block_size"),
                      (dict(bs=256), "block_size"), (dict(bt=t["bt"][:, ::2]), "contiguous"),
                      (dict(bt=t["bt"].cpu()), "CUDA")]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    with pytest.raises(RuntimeError, match="overlaps"):   # (an output is no other input)
        pa_int8.extend_block_tables(*[t[n] for n in args], 16, context_lens_out=t["new"])
    with pytest.raises(RuntimeError, match="overlaps"):
        call(st=t["nfree"])
    n = 4097
    z = torch.zeros(n, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="at most 4096"):
        call(bt=torch.zeros(n, 1, dtype=torch.int32, device=DEV), ctx=z, new=z,
             cu=torch.zeros(n + 1, dtype=torch.int32, device=DEV))
