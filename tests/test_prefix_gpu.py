"""Decode attention behind shared prefixes against its definition in 64 bits.

What may differ.  A score is a sum of D products of floats, q times the scale (and log2 e) rounded once: off by at most
e = (D + 4) 2^-24 scale sum |q k|, and each weight by the factor 2^(+-e log2 e) (1 + 2^-21) (the exponential's own error and those
of the rescalings); numerator and denominator together twice that, and every addition 2^-24 of what is added up (at most L + 64
of them in a row).  With weights that sum to one: 2 (exp(e) - 1 + 2^-21 + (L + 64) 2^-24) max |v|.  bfloat16 adds the rounding of
the result, 2^-8 of it, and on the tensor cores that of each weight, 2^-8 max |v|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def prefix():
    from llm_infer_rust_b200.kernels import prefix as m
    return m


def ops():
    from llm_infer_rust_b200.kernels import ops as m
    return m


class Case:
    """A batch on the device.  ``groups``: (rows, shared keys, [own keys of each row]); own keys may be negative (the row sees less
    than the group shares).  Slots of the pool that no row sees hold NaN.  ``other_tokens``: tokens of q between the rows'."""

    def __init__(self, groups, nh, nkv, d, page, dtype, seed=0, other_tokens=0, scramble=False):
        g = torch.Generator().manual_seed(seed + 13 * d + page)
        self.nh, self.nkv, self.d, self.page, self.dtype = nh, nkv, d, page, dtype
        self.scale = d ** -0.5
        lengths, shared_of, tables, place = [], [], [], []
        total = 1 + sum(-(-s // page) + n * 2 + sum(-(-max(0, o) // page) for o in own) for n, s, own in groups)
        order = (torch.randperm(total, generator=g) + 1).tolist()
        copies = []
        for n, shared, own in groups:
            assert len(own) == n
            whole = [order.pop() for _ in range(shared // page)]
            begun = None
            place.append((len(tables), shared))
            for o in own:
                length = shared + o
                mine = [order.pop() for _ in range(max(0, -(-max(length, shared) // page) - len(whole)))]
                if shared % page:
                    if begun is None:
                        begun = mine[0]
                    else:
                        copies.append((begun, mine[0], shared % page))
                tables.append(whole + mine)
                lengths.append(length)
                shared_of.append(shared)
        n = len(tables)
        k = torch.full((total + 1, nkv, page, d), float("nan"))
        v = k.clone()
        for t, length, shared in zip(tables, lengths, shared_of):
            for j in range(max(length, shared)):
                k[t[j // page], :, j % page] = torch.randn(nkv, d, generator=g)
                v[t[j // page], :, j % page] = torch.randn(nkv, d, generator=g)
        for a, b, slots in copies:
            k[b, :, :slots], v[b, :, :slots] = k[a, :, :slots], v[a, :, :slots]
        self.k, self.v = k.to(dtype).to(DEV), v.to(dtype).to(DEV)
        width = max(1, max(len(t) for t in tables)) + 1
        # the batch's rows stand in another order than the groups'
        batch = torch.randperm(n, generator=g).tolist() if scramble else list(range(n))
        table = torch.zeros(n, width, dtype=torch.int32)
        kv_len = torch.zeros(n, dtype=torch.int32)
        for i, t in enumerate(tables):
            table[batch[i], :len(t)] = torch.tensor(t, dtype=torch.int32)
            kv_len[batch[i]] = lengths[i]
        self.table, self.kv_len = table.to(DEV), kv_len.to(DEV)
        self.cu_q = (torch.arange(n + 1, dtype=torch.int32) * (1 + other_tokens)).to(DEV)
        self.rows = torch.tensor(batch, dtype=torch.int32).to(DEV)
        self.groups = torch.tensor(place, dtype=torch.int32).to(DEV)
        self.q = torch.randn(n * (1 + other_tokens), nh * d, generator=g).to(dtype).to(DEV)
        self.hints = dict(most_rows=max(r for r, _, _ in groups), most_shared=max(s for _, s, _ in groups),
                          most_own=max(0, max(max(o) for _, _, o in groups)))
        self.tables, self.lengths, self.batch = tables, lengths, batch

    def run(self, out=None, **hints):
        out = torch.full_like(self.q, 7.0) if out is None else out
        prefix().prefix_attention(self.q, self.k, self.v, out, self.table, self.cu_q, self.kv_len, self.rows, self.groups, self.nh, self.nkv,
                                  self.d, self.page, self.scale, **{**self.hints, **hints})
        return out

    def check(self, out):
        q, k, v = self.q.double().cpu(), self.k.double().cpu(), self.v.double().cpu()
        cu = self.cu_q.tolist()
        per = self.nh // self.nkv
        written = set()
        for i, (t, length) in enumerate(zip(self.tables, self.lengths)):
            token = cu[self.batch[i]]
            written.add(token)
            got = out[token].double().cpu().view(self.nkv, per, self.d)
            if length <= 0:
                assert (got == 0).all()
                continue
            at = torch.arange(length)
            pages = torch.tensor(t)[at // self.page]
            kk, vv = k[pages, :, at % self.page], v[pages, :, at % self.page]          # [L, nkv, d]
            qq = q[token].view(self.nkv, per, self.d)
            s = torch.einsum("hqd,lhd->hql", qq, kk) * self.scale
            want = torch.einsum("hql,lhd->hqd", torch.softmax(s, -1), vv)
            e = (self.d + 4) * 2.0 ** -24 * float(torch.einsum("hqd,lhd->hql", qq.abs(), kk.abs()).max()) * self.scale
            most = float(vv.abs().max())
            tol = 2 * (math.exp(e) - 1 + 2.0 ** -21 + (length + 64) * 2.0 ** -24) * most
            bound = torch.full_like(want, tol)
            if self.dtype == BF16:
                bound += 2.0 ** -8 * most + 2.0 ** -8 * want.abs()
            assert not got.isnan().any(), i
            assert ((got - want).abs() <= bound).all(), (i, float(((got - want).abs() / bound).max()))
        rest = [t for t in range(out.shape[0]) if t not in written]
        assert (out[rest] == 7.0).all()
        ops().check_errors(out.device)


# (groups, nh, nkv, d, page)
CASES = {
    "one row, nothing shared": ([(1, 0, [1])], 4, 2, 16, 16),
    "one row, all shared": ([(1, 33, [0])], 4, 2, 16, 16),
    "two rows, a short prompt": ([(2, 300, [1, 9])], 16, 8, 128, 16),
    "one key": ([(3, 1, [0, 0, 0])], 8, 8, 64, 16),
    "rows that see less than is shared, and nothing": ([(5, 100, [4, -40, 0, -100, -99])], 8, 2, 64, 16),
    "no keys at all": ([(2, 0, [0, 0])], 4, 4, 32, 8),
    "groups of all sizes": ([(1, 17, [3]), (7, 129, [1, 2, 3, 40, 5, 6, 70]), (2, 0, [5, 80]), (12, 64, list(range(1, 13)))], 8, 2, 128, 16),
    "forty rows": ([(40, 257, [1 + i % 7 for i in range(40)])], 8, 2, 128, 16),
    "seventy rows of one head": ([(70, 70, [1 + i % 3 for i in range(70)])], 2, 2, 128, 32),
    "a long prompt": ([(3, 5000, [100, 1, 33])], 8, 2, 128, 16),
    "long answers": ([(2, 31, [1500, 700])], 8, 2, 128, 16),
    "pages of 24": ([(4, 130, [1, 25, 24, 50])], 6, 2, 96, 24),
    "pages of 7": ([(6, 200, [1, 8, 30, 60, 3, 100]), (2, 13, [1, 40])], 8, 2, 128, 7),
    "pages of 40": ([(3, 333, [1, 8, 130])], 8, 2, 64, 40),
    "pages of one": ([(3, 37, [1, 2, 3])], 4, 2, 48, 1),
    "pages of two": ([(3, 75, [1, 2, 30])], 4, 2, 128, 2),
    "pages of 128": ([(3, 300, [1, 2, 130])], 4, 2, 64, 128),
    "heads of two": ([(3, 50, [1, 7, 8])], 4, 2, 2, 16),
    "heads of ten": ([(3, 50, [1, 7, 8])], 4, 2, 10, 16),
    "heads of 80": ([(20, 100, [1 + i for i in range(20)])], 15, 5, 80, 16),
    "heads of 256": ([(9, 190, [1 + 5 * i for i in range(9)])], 8, 2, 256, 16),
    "heads of 512": ([(3, 65, [1, 7, 8])], 4, 2, 512, 16),
    "sixteen query heads": ([(5, 100, [1, 2, 3, 4, 50])], 16, 1, 128, 16),
    "thirty-three query heads": ([(3, 100, [1, 2, 30])], 33, 1, 64, 16),
    "many groups": ([(1 + i % 3, 20 + 7 * i, [1 + j for j in range(1 + i % 3)]) for i in range(45)], 4, 2, 64, 16),
}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(CASES))
def test_against_64_bits(name, dtype):
    groups, nh, nkv, d, page = CASES[name]
    c = Case(groups, nh, nkv, d, page, dtype)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_rows_in_any_order_beside_other_tokens(dtype):
    c = Case([(3, 40, [1, 9, 30]), (4, 100, [2, 2, 2, 60])], 8, 2, 128, 16, dtype, other_tokens=2, scramble=True)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("hints", [dict(most_rows=1, most_shared=0, most_own=0), dict(most_rows=0, most_shared=1 << 20, most_own=1),
                                   dict(most_rows=1000, most_shared=10, most_own=1 << 20)])
def test_hints_do_not_change_what_is_computed(hints, dtype):
    c = Case([(3, 40, [1, 9, 30]), (40, 300, [2 + i for i in range(40)])], 8, 2, 128, 16, dtype)
    c.check(c.run(**hints))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_large_scores_and_values(dtype):
    """Scores in the hundreds: one key takes nearly all of the weight, the others' weights fall below the smallest floats."""
    c = Case([(6, 200, [1, 5, 9, 2, 2, 2])], 8, 2, 64, 16, dtype)
    c.q.mul_(24.0)
    c.v.mul_(64.0)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_the_same_bits_twice_and_beside_another_call(dtype):
    c = Case([(20, 600, [1 + i for i in range(20)]), (3, 50, [1, 2, 3])], 8, 2, 128, 16, dtype)
    first = c.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.full_like(c.q, 7.0) for _ in range(6)]
    for i, o in enumerate(outs):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            c.run(o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_a_captured_call_serves_other_lengths_and_groups(dtype):
    a = Case([(6, 200, [1, 5, 9, 2, 2, 2])], 8, 2, 128, 16, dtype, seed=1)
    b = Case([(6, 77, [0, 30, -5, 1, 3, 40])], 8, 2, 128, 16, dtype, seed=2)
    pool = max(a.k.shape[0], b.k.shape[0])
    width = max(a.table.shape[1], b.table.shape[1])

    def padded(t, shape):
        out = torch.zeros(shape, dtype=t.dtype, device=DEV)
        out[tuple(slice(n) for n in t.shape)] = t
        return out
    for c in (a, b):
        c.k, c.v = (padded(t, (pool,) + tuple(t.shape[1:])) for t in (c.k, c.v))
        c.table = padded(c.table, (6, width))
    a.hints = dict(most_rows=6, most_shared=200, most_own=40)
    a.run()
    torch.cuda.synchronize()
    out = torch.full_like(a.q, 7.0)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    others = torch.full_like(a.q, 7.0)
    for graph, o in zip(graphs, (out, others)):
        with torch.cuda.graph(graph):
            a.run(o)
    want = {}
    for c in (a, b):
        for name in ("q", "k", "v", "table", "kv_len", "groups"):
            want[name] = getattr(a, name)
            if c is not a:
                want[name].copy_(getattr(c, name))
        out.fill_(7.0)
        others.fill_(7.0)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        for _ in range(5):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        c.check(out)
        assert torch.equal(out, others)


def test_a_row_in_front_of_the_first_group_and_no_groups():
    c = Case([(4, 64, [3, 4, 5, 6])], 8, 2, 64, 16, BF16)
    c.groups = torch.tensor([[2, 64]], dtype=torch.int32, device=DEV)      # rows 0 and 1 stand in no group: all their keys are their own
    c.check(c.run())
    c.groups = torch.zeros((0, 2), dtype=torch.int32, device=DEV)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
def test_pages_outside_the_pool_and_rows_longer_than_their_table(dtype, d):
    c = Case([(40, 64, [3 + i for i in range(40)])], 8, 2, d, 16, dtype)
    o = ops()
    good = c.table.clone()
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31):
        for row, at in ((0, 1), (3, 4)):                   # a shared page, an own one
            c.table.copy_(good)
            c.table[row, at] = bad
            c.run()
            with pytest.raises(o.KernelError, match="outside the pool"):
                o.check_errors(c.q.device)
    c.table.copy_(good)
    c.kv_len[5] = 2 ** 31 - 1
    c.run()
    with pytest.raises(o.KernelError, match="outside the pool"):
        o.check_errors(c.q.device)
    c.kv_len[5] = 64 + 8
    c.check(c.run())


def test_nothing_to_do():
    c = Case([(2, 10, [1, 1])], 4, 2, 16, 16, F32)
    c.rows, c.groups = c.rows[:0], c.groups[:0]
    out = torch.full_like(c.q, 7.0)
    c.run(out)
    assert (out == 7.0).all()


NAN_CASES = {"mma": ([(3, 200, [5, 1, 40]), (1, 10, [3])], 8, 2, 64, 16), "tcgen05": ([(40, 2600, [1 + i for i in range(40)])], 32, 8, 128, 16),
             "tcgen05, two tiles": ([(80, 1100, [1 + i for i in range(80)])], 32, 8, 128, 16)}


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", list(NAN_CASES))
def test_a_nan_stays_with_its_row(name, dtype):
    c = Case(*NAN_CASES[name], dtype)
    q = c.q.clone()
    want = c.run()
    bad = [1, 2]
    c.q[1] = float("nan")
    c.q[2, 0] = float("nan")                        # (of one head)
    got = c.run()
    assert got[1].isnan().all() and got[2, :c.d].isnan().all() and not got[2, c.d:].isnan().any()
    c.q.copy_(q)
    got[1], got[2, :c.d] = want[1], want[2, :c.d]
    c.check(got)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["mma", "tcgen05"])
def test_the_output_may_be_where_the_queries_are(name, dtype):
    c = Case(*NAN_CASES[name], dtype, other_tokens=1)
    q, want = c.q.clone(), c.run()
    got = c.run(out=c.q)
    tokens = c.cu_q[:-1].long()
    rest = torch.ones(len(q), dtype=torch.bool, device=DEV)
    rest[tokens] = False
    assert torch.equal(got[tokens], want[tokens]) and torch.equal(got[rest], q[rest])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["mma", "tcgen05"])
def test_calls_on_two_streams_at_once(name, dtype):
    """Every call has memory of its own between its kernels."""
    cases = [Case(*NAN_CASES[name], dtype, seed=s) for s in (0, 1)]
    want = [c.run() for c in cases]
    outs = [[torch.full_like(c.q, 7.0) for _ in range(6)] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for x in range(6):
        for c, out, stream in zip(cases, outs, streams):
            with torch.cuda.stream(stream):
                c.run(out=out[x])
    torch.cuda.synchronize()
    for w, of in zip(want, outs):
        for got in of:
            assert torch.equal(got, w)


# What the tcgen05 kernel is given when it is given everything: (groups, nh, nkv, page), heads of 128 in bfloat16
TCGEN05_CASES = {
    "one key": ([(3, 1, [0, 0, 0])], 8, 8, 16),
    "one row": ([(1, 300, [5])], 4, 2, 16),
    "a block less a key": ([(3, 127, [1, 0, 20])], 8, 2, 16),
    "a block": ([(3, 128, [1, 0, 20])], 8, 2, 16),
    "a block and a key": ([(3, 129, [1, 0, 20])], 8, 2, 16),
    "two blocks and a key": ([(3, 257, [1, 0, 20])], 8, 2, 16),
    "five blocks": ([(12, 640, [1 + i for i in range(12)])], 8, 2, 16),
    "rows that see less than is shared, and nothing": ([(6, 700, [4, -40, 0, -700, -699, -300])], 8, 2, 16),
    "a tile and a row of vectors": ([(33, 400, [1 + i % 5 for i in range(33)])], 8, 2, 16),
    "two tiles": ([(64, 1000, [1 + i % 50 for i in range(64)])], 8, 2, 16),
    "three tiles of two": ([(70, 300, [1 + i % 3 for i in range(70)])], 16, 2, 16),
    "groups of all sizes": ([(1, 17, [3]), (7, 129, [1, 2, 3, 40, 5, 6, 70]), (2, 0, [5, 80]), (40, 640, list(range(1, 41)))], 8, 2, 16),
    "sixteen query heads": ([(9, 500, [1 + i for i in range(9)])], 16, 1, 16),
    "pages of one": ([(4, 150, [1, 2, 3, 4])], 4, 2, 1),
    "pages of four": ([(20, 333, [1 + i for i in range(20)])], 8, 2, 4),
    "pages of 64": ([(20, 333, [1 + i for i in range(20)])], 8, 2, 64),
    "a long prompt": ([(5, 20000, [100, 1, 33, 7, 2])], 8, 1, 16),
}


@pytest.fixture
def always_tcgen05(monkeypatch):
    m = prefix()
    asked = []
    load = m.load_entry_points
    monkeypatch.setattr(m, "load_entry_points", lambda source, *a: asked.append(source) or load(source, *a))
    for name in ("_TENSOR_CORE_BLOCKS", "_TENSOR_CORE_BLOCKS_A_STEP", "_TENSOR_CORE_BLOCKS_OF_GROUPS"):
        monkeypatch.setattr(m, name, 0)
    # (it is asked for from the first vector on; what an item of the other kernel takes stays)
    monkeypatch.setattr(m, "_TENSOR_CORE_VECTORS", 0)
    m._plan.cache_clear()
    yield asked
    m._plan.cache_clear()
    assert "prefix_tcgen05.cu" in asked


@pytest.mark.parametrize("name", list(TCGEN05_CASES))
def test_tcgen05_against_64_bits(name, always_tcgen05):
    groups, nh, nkv, page = TCGEN05_CASES[name]
    c = Case(groups, nh, nkv, 128, page, BF16)
    c.check(c.run())


@pytest.mark.parametrize("hints", [dict(most_rows=1, most_shared=0, most_own=0), dict(most_rows=0, most_shared=1 << 20, most_own=1),
                                   dict(most_rows=1000, most_shared=10, most_own=1 << 20), dict(sharing_groups=1), dict(sharing_groups=0)])
def test_tcgen05_with_other_hints(hints, always_tcgen05):
    c = Case([(3, 40, [1, 9, 30]), (50, 300, [2 + i for i in range(50)]), (7, 1300, [5] * 7)], 8, 2, 128, 16, BF16, other_tokens=1, scramble=True)
    c.check(c.run(**hints))


def test_tcgen05_large_scores(always_tcgen05):
    """Scores in the hundreds, rising along the keys: the reference maximum moves again and again."""
    c = Case([(20, 1500, [1 + i for i in range(20)])], 8, 2, 128, 16, BF16)
    c.q.mul_(24.0)
    c.v.mul_(64.0)
    rise = torch.linspace(0.1, 4.0, c.k.shape[0], device=DEV).to(BF16)
    order = torch.tensor(c.tables[0][:1500 // 16], device=DEV)
    c.k[order] *= rise[:len(order), None, None, None]
    for t in c.tables[1:]:                          # (the begun page is in every row's table)
        assert t[:1500 // 16] == c.tables[0][:1500 // 16]
    c.check(c.run())


def test_tcgen05_the_same_bits_on_other_streams_and_in_a_graph(always_tcgen05):
    c = Case([(20, 600, [1 + i for i in range(20)]), (30, 900, [1 + i for i in range(30)])], 8, 2, 128, 16, BF16)
    first = c.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = [torch.full_like(c.q, 7.0) for _ in range(8)]
    for i, o in enumerate(outs[:6]):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            c.run(o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(outs[6])
        c.run(outs[7])
    for _ in range(3):
        outs[6].fill_(7.0)
        outs[7].fill_(7.0)
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    # the captured call on other lengths and groups: rows move to the first group, lengths shrink
    c.groups.copy_(torch.tensor([[0, 600], [35, 333]], dtype=torch.int32))
    lengths = c.kv_len.tolist()
    c.kv_len[20:35] = torch.tensor([590] * 15, dtype=torch.int32)
    c.kv_len[35:] -= 100
    graph.replay()
    torch.cuda.synchronize()
    got = outs[6].clone()
    # (rows 20 to 34 now read the first group's keys, no further than 590; the others their own from 333 on)
    c.lengths = [lengths[i] if i < 20 else 590 if i < 35 else lengths[i] - 100 for i in range(50)]
    c.tables = [t if i < 20 or i >= 35 else c.tables[0] for i, t in enumerate(c.tables)]
    c.check(got)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["q", "k", "v", "out"])
def test_tensors_off_16_bytes(which, dtype):
    c = Case([(5, 100, [4, -40, 0, -100, 33]), (2, 13, [1, 2])], 8, 2, 128, 16, dtype)

    def off(t):
        there = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
        return there.copy_(t)
    out = torch.full_like(c.q, 7.0)
    if which == "out":
        out = off(out)
    else:
        setattr(c, which, off(getattr(c, which)))
    c.check(c.run(out))


def by_definition(c):
    """Every row's outputs in 64 bits, NaN and infinities as the definition has them, and how far they may be off: as at the top of this
    file, with the largest value of each dim that is no infinity."""
    q, k, v = c.q.double().cpu(), c.k.double().cpu(), c.v.double().cpu()
    per, found = c.nh // c.nkv, []
    for i, (t, length) in enumerate(zip(c.tables, c.lengths)):
        token = c.cu_q.tolist()[c.batch[i]]
        at = torch.arange(length)
        pages = torch.tensor(t)[at // c.page]
        kk, vv = k[pages, :, at % c.page], v[pages, :, at % c.page]
        s = torch.einsum("hqd,lhd->hql", q[token].view(c.nkv, per, c.d), kk) * c.scale
        want = torch.einsum("hql,lhd->hqd", torch.softmax(s, -1), vv)
        sizes = torch.einsum("hqd,lhd->hql", q[token].view(c.nkv, per, c.d).abs(), kk.abs())
        e = (c.d + 4) * 2.0 ** -24 * float(sizes[sizes.isfinite()].max()) * c.scale
        most = vv.abs().masked_fill(vv.isinf(), 0.0).amax(0)[:, None]                   # [nkv, 1, d]
        bound = 2 * (math.exp(e) - 1 + 2.0 ** -21 + (length + 64) * 2.0 ** -24) * most
        if c.dtype == BF16:
            bound = bound + 2.0 ** -8 * most + 2.0 ** -8 * want.abs()
        # (a result below the smallest normal number has the last place of those)
        found.append((token, want, bound + length * torch.finfo(c.dtype).smallest_normal * torch.finfo(c.dtype).eps))
    return found


def agrees(c, out):
    for token, want, bound in by_definition(c):
        got = out[token].double().cpu().view(want.shape)
        assert torch.equal(got.isnan(), want.isnan()), token
        assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()), token
        some = want.isfinite()
        assert ((got - want).abs() <= bound)[some].all(), (token, float(((got - want).abs() / bound)[some].max()))


# (groups, nh, nkv, d, page, dtype): every kernel
ODD_VALUES = {
    "float32": ([(6, 200, [1, 5, 9, 2, 2, 40])], 8, 2, 64, 16, F32),
    "float32, two tiles of vectors": ([(20, 200, [1 + i for i in range(20)])], 8, 2, 128, 16, F32),
    "float32, heads of 30": ([(6, 200, [1, 5, 9, 2, 2, 40])], 8, 2, 30, 16, F32),
    "float32, heads of 512": ([(6, 200, [1, 5, 9, 2, 2, 40])], 4, 2, 512, 16, F32),
    "bfloat16, all sizes": ([(6, 200, [1, 5, 9, 2, 2, 40])], 34, 2, 64, 16, BF16),
    "mma": ([(6, 200, [1, 5, 9, 2, 2, 40])], 8, 2, 64, 16, BF16),
    "tcgen05": ([(40, 2600, [1 + i for i in range(40)])], 32, 8, 128, 16, BF16),
    "tcgen05, two tiles": ([(80, 1100, [1 + i for i in range(80)])], 32, 8, 128, 16, BF16),
}


@pytest.mark.parametrize("name", list(ODD_VALUES))
def test_infinities_among_keys_and_values(name):
    c = Case(*ODD_VALUES[name])
    inf = float("inf")

    def put(cache, row, key, head, dim, value):
        cache[c.tables[row][key // c.page], head, key % c.page, dim] = value
    c.q.view(len(c.q), c.nh, c.d)[..., 3] = c.q.view(len(c.q), c.nh, c.d)[..., 3].abs() + 0.5
    put(c.k, 0, 17, 0, 3, -inf)                      # a shared key that no row's weight falls on
    put(c.k, 5, c.lengths[5] - 2, 0, 3, -inf)        # an own one
    put(c.k, 4, c.lengths[4] - 1, 1, 3, inf)         # one that takes all of the weight: no distribution
    put(c.v, 0, 40, 0, 5, inf)
    put(c.v, 0, 41, 0, 7, -inf)
    put(c.v, 0, 42, 0, 9, inf)
    put(c.v, 0, 43, 0, 9, -inf)                      # (the sum of both is none)
    put(c.v, 3, c.lengths[3] - 1, 1, 0, -inf)
    want = by_definition(c)
    assert want[4][1][1].isnan().all() and want[3][1][1, :, 0].isneginf().all() and want[0][1][0, :, 9].isnan().all() and want[0][1][1].isfinite().all()
    agrees(c, c.run())


@pytest.mark.parametrize("name", [n for n in ODD_VALUES if "mma" not in n and "tcgen05" not in n])
def test_the_largest_and_the_smallest_floats(name):
    """Floats that rounding to 11 bits would carry beyond the largest one, and those whose rest would be lost below the smallest."""
    c = Case(*ODD_VALUES[name])
    largest = torch.finfo(c.dtype).max
    key = (c.tables[0][2], 1, 5)
    c.q.view(len(c.q), c.nh, c.d)[..., 4] = 2.0 ** -124
    c.k[key][4] = largest
    c.v[key][6] = largest
    c.v[key][8] = -largest
    c.v[..., 11] *= 2.0 ** -122
    agrees(c, c.run())


def test_tables_and_caches_beyond_what_the_tensor_core_kernels_count():
    """They count in 32 bits; the all-sizes kernel takes the rest."""
    c = Case([(2, 300, [5, 130])], 16, 8, 64, 128, BF16)
    small = c.table
    c.table = torch.zeros(2, 1 << 23, dtype=torch.int32, device=DEV)          # 2^30 places
    c.table[:, :small.shape[1]] = small
    c.check(c.run())
    # 2^31 rows of keys, the call's pages the last ones
    c = Case([(3, 300, [5, 130, 0])], 16, 8, 16, 128, BF16)
    c.v = c.k
    pages = (1 << 21) + 5
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("64 GiB of keys")
    small, first = c.k, pages - c.k.shape[0]
    c.k = c.v = torch.empty((pages,) + tuple(small.shape[1:]), dtype=BF16, device=DEV)
    c.k[first:] = small
    c.table += first
    out = c.run()
    c.k = c.v = small
    torch.cuda.empty_cache()
    c.check(out)


@pytest.mark.parametrize("sharing", [1, 2, 3, 4, 5, None])
def test_tcgen05_of_the_first_groups_alone(sharing, always_tcgen05):
    """Groups behind those that it is said to serve are the other kernel's, whether they share keys or not."""
    c = Case([(40, 300, [2 + i for i in range(40)]), (3, 700, [1, 9, -200]), (2, 0, [50, 0]), (35, 200, [1 + i for i in range(35)]), (1, 0, [33])],
             8, 2, 128, 16, BF16, other_tokens=1, scramble=True)
    c.check(c.run(sharing_groups=sharing))


@pytest.mark.parametrize("rows", [397, 398, 430])
def test_as_many_rows_as_the_tensor_core_kernels_take_and_more(rows):
    """400 rows and groups together: 397 and 398 rows in two groups, then the all-sizes kernel."""
    first = rows - 50
    c = Case([(first, 150, [1 + i % 40 for i in range(first)]), (50, 33, [1 + i for i in range(50)])], 4, 2, 64, 16, BF16, scramble=True)
    c.check(c.run())


@pytest.mark.parametrize("d", [130, 192, 256, 384, 512])
def test_float32_wide_heads_in_several_groups(d):
    c = Case([(3, 70, [1, 40, 9]), (2, 0, [5, 33]), (20, 130, [1 + i for i in range(20)]), (1, 16, [3])], 8, 2, d, 16, F32, other_tokens=1, scramble=True)
    c.check(c.run())
