"""Forks of requests on the host: pages with several holders, what a fork has to copy, and the rows of a step that share pages."""
import random

import numpy as np
import pytest

from llm_infer_rust_b200.kernels.build import load_host_runtime

rt = load_host_runtime()
Ready = rt.Acquire.Ready


def manager(pages, page_size=4, window=0, slots=8):
    if isinstance(pages, int):
        pages, window = [pages], [window]
    return rt.CacheManager([rt.GroupSpec(page_size, n, w) for n, w in zip(pages, window)], slots)


def hold(m, request, length):
    assert m.grow(request, length)
    m.advance(request, length)


def test_a_page_is_free_again_with_its_last_holder():
    pool = rt.PagePool(3)
    page = pool.alloc()
    pool.share(page)
    pool.share(page)
    assert pool.holders(page) == 3 and pool.free_count() == 2
    assert pool.release(page) and pool.release(page) and pool.is_held(page) and pool.free_count() == 2
    assert pool.release(page) and not pool.is_held(page) and pool.free_count() == 3
    assert not pool.release(page)
    for bad in (0, 2, 4):
        with pytest.raises(Exception):
            pool.share(bad)


def test_a_fork_shares_whole_pages_and_copies_the_begun_one():
    m = manager(10)
    m.open(1)
    hold(m, 1, 10)                                            # pages 10, 9 and half of 8
    got, pages, state = m.fork(1, 2)
    assert got == Ready and pages == [[[8, 7, 2]]] and state == [1, 2]
    assert m.block_table(2, 0) == [10, 9, 7] and m.length(2) == 10 and m.shared_pages(0) == 2 and m.check() == ""
    assert m.fork(2, 3)[:2] == (Ready, [[[7, 6, 2]]]) and m.shared_pages(0) == 2 and m.check() == ""
    hold(m, 1, 13)
    hold(m, 2, 11)
    assert m.block_table(1, 0) == [10, 9, 8, 5] and m.slot_of(2, 0, 10) == 7 * 4 + 2
    assert m.release(1) and m.check() == "" and m.shared_pages(0) == 2
    assert m.release(3) and m.shared_pages(0) == 0
    assert m.release(2) and m.free_pages(0) == 10 and m.check() == ""


def test_a_fork_at_a_page_boundary_copies_nothing_and_one_of_nothing_shares_nothing():
    m = manager(4)
    m.open(1)
    assert m.fork(1, 2) == (Ready, [[]], [1, 2]) and m.length(2) == 0
    hold(m, 1, 8)
    assert m.fork(1, 3)[:2] == (Ready, [[]]) and m.block_table(3, 0) == m.block_table(1, 0)
    hold(m, 3, 9)
    hold(m, 1, 9)
    assert m.block_table(3, 0)[2] != m.block_table(1, 0)[2] and m.check() == ""


def test_pages_that_a_parent_has_but_does_not_use_yet_are_its_own():
    m = manager(6)
    m.open(1)
    hold(m, 1, 5)
    m.grow(1, 12)                                             # (a step that did not come about)
    assert m.fork(1, 2)[1] == [[[5, 3, 1]]] and m.block_table(2, 0) == [6, 3] and m.check() == ""


def test_a_fork_without_room_changes_nothing():
    m = manager(3, slots=2)
    m.open(1)
    hold(m, 1, 9)
    assert m.fork(1, 2)[0] == rt.Acquire.DeferredMemory and not m.has(2) and m.free_state_slots() == 1 and m.check() == ""
    m = manager(9, slots=1)
    m.open(1)
    hold(m, 1, 9)
    assert m.fork(1, 2)[0] == rt.Acquire.DeferredSlots and not m.has(2) and m.shared_pages(0) == 0 and m.check() == ""


def test_forks_that_are_refused():
    m = manager(9)
    m.open(1)
    hold(m, 1, 3)
    with pytest.raises(Exception):
        m.fork(5, 6)                                          # no such parent
    with pytest.raises(Exception):
        m.fork(1, 1)
    assert m.acquire(7, 8, 4) == Ready
    with pytest.raises(Exception, match="promise"):
        m.fork(7, 8)
    assert not m.has(8) and m.check() == ""


def test_windows_share_what_is_live():
    m = manager([20, 20], window=[0, 6])
    m.open(1)
    for n in (4, 8, 12, 14):
        hold(m, 1, n)
    got, pages, _ = m.fork(1, 2)
    assert got == Ready and len(pages[0]) == len(pages[1]) == 1 and m.check() == ""
    assert m.block_table(2, 1)[:2] == [0, 0] and m.first_live_page(2, 1) == m.first_live_page(1, 1)
    free = m.free_pages(1)
    hold(m, 1, 20)                                            # its window leaves the shared page: the child still holds it
    assert m.check() == "" and m.shared_pages(1) == 0
    hold(m, 2, 20)
    assert m.check() == ""
    m.release(1)
    m.release(2)
    assert m.free_pages(0) == m.free_pages(1) == 20 and free < 20 and m.check() == ""


def test_no_page_is_lost_in_random_forks():
    rng = random.Random(5)
    m = manager([60, 40], window=[0, 9], slots=12)
    live, next_id = [], 1
    for _ in range(4000):
        what = rng.random()
        if what < 0.2 and len(live) < 12:
            if m.open(next_id) == Ready:
                live.append(next_id)
            next_id += 1
        elif what < 0.45 and live:
            if m.fork(rng.choice(live), next_id)[0] == Ready:
                live.append(next_id)
            next_id += 1
        elif what < 0.85 and live:
            r = rng.choice(live)
            n = m.length(r) + rng.randint(1, 6)
            if m.grow(r, n):
                m.advance(r, n)
        elif live:
            m.release(live.pop(rng.randrange(len(live))))
        assert m.check() == ""
    for r in live:
        m.release(r)
    assert m.free_pages(0) == 60 and m.free_pages(1) == 40 and m.shared_pages(0) == m.shared_pages(1) == 0 and m.check() == ""


def batch(m, ids, counts=None, **more):
    counts = counts or [1] * len(ids)
    req = rt.BatchRequest()
    req.ids, req.counts, req.tokens = ids, counts, [0] * sum(counts)
    req.want_counts, req.want_index = [1] * len(ids), [0] * len(ids)
    for name, value in more.items():
        setattr(req, name, value)
    for r, c in zip(ids, counts):
        assert m.grow(r, m.length(r) + c)
    layout = rt.plan_batch(m, req)
    out = np.full(layout.total_ints, -7, dtype=np.int32)
    return rt.build_batch(m, req, out), out, req


def groups_of(layout, out):
    rows = out[layout.off_prefix_rows:layout.off_prefix_rows + layout.num_decode].tolist()
    groups = out[layout.off_prefix_groups:layout.off_prefix_groups + 2 * layout.num_prefix_groups].reshape(-1, 2).tolist()
    ends = [g[0] for g in groups[1:]] + [len(rows)]
    return [(sorted(rows[a:b]), keys) for (a, keys), b in zip(groups, ends)]


def test_rows_that_share_pages_are_found():
    m = manager(100, slots=20)
    m.open(1)
    hold(m, 1, 13)                                            # three whole pages
    for c in (2, 3):
        m.fork(1, c)
    m.open(4)
    hold(m, 4, 9)
    m.fork(4, 5)
    for r in (6, 7):
        m.open(r)
        hold(m, r, 30)
    ids = [6, 2, 4, 1, 7, 5, 3]
    plain, _, req = batch(m, ids)
    assert plain.num_prefix_groups == 0
    req.prefix_group = 0
    assert rt.count_prefix_groups(m, req) == (2, 2 * 12 + 1 * 8, 12, 31)
    layout, out, _ = batch(m, ids, prefix_group=0)
    assert layout.num_prefix_groups == 3
    found = groups_of(layout, out)
    assert sorted(found[:2]) == [([1, 3, 6], 12), ([2, 5], 8)] and found[2] == ([0, 4], 0)
    assert (layout.most_prefix_rows, layout.most_prefix_keys, layout.most_own_keys) == (3, 12, 31)
    assert layout.total_ints > plain.total_ints


def test_pages_are_shared_only_as_far_as_all_rows_hold_them():
    m = manager(100)
    m.open(1)
    hold(m, 1, 9)
    m.fork(1, 2)                                              # two pages in common
    hold(m, 1, 17)
    m.fork(1, 3)                                              # four with the first
    layout, out, _ = batch(m, [1, 2, 3], prefix_group=0)
    assert groups_of(layout, out) == [([0, 1, 2], 8), ([], 0)]


def test_prompts_rows_without_a_whole_page_and_steps_without_forks_have_no_groups():
    m = manager(100)
    m.open(1)
    hold(m, 1, 3)
    m.fork(1, 2)                                              # only the begun page, which is copied
    layout, _, _ = batch(m, [1, 2], prefix_group=0)
    assert layout.num_prefix_groups == 0
    m = manager(100)
    m.open(1)
    hold(m, 1, 8)
    m.fork(1, 2)
    layout, _, _ = batch(m, [1, 2], [3, 1], prefix_group=0)   # one of the two brings a portion of a prompt
    assert layout.num_prefix_groups == 0


def test_places_of_a_graph():
    m = manager(100)
    m.open(1)
    hold(m, 1, 8)
    m.fork(1, 2)
    layout, out, _ = batch(m, [1, 2], prefix_group=0, prefix_groups=3, pad_rows_to=4, fixed_table_width=[10])
    assert layout.num_decode == 4 and groups_of(layout, out) == [([0, 1], 8), ([], 0), ([2, 3], 0)]
    empty, _, _ = batch(m, [], prefix_group=0, prefix_groups=3, pad_rows_to=4, fixed_table_width=[10])
    assert empty.total_ints == layout.total_ints
    with pytest.raises(Exception, match="more groups"):
        batch(m, [1, 2], prefix_group=0, prefix_groups=1, pad_rows_to=4, fixed_table_width=[10])


def test_groups_with_a_window_are_not_looked_in():
    m = manager([20, 20], window=[0, 6])
    m.open(1)
    hold(m, 1, 8)
    m.fork(1, 2)
    with pytest.raises(Exception, match="keeps all keys"):
        batch(m, [1, 2], prefix_group=1)


@pytest.mark.parametrize("error", [RuntimeError("the copies fail"), KeyboardInterrupt(), MemoryError("no room for a table")])
def test_no_child_is_left_where_the_copies_fail(error):
    from types import SimpleNamespace
    from llm_infer_rust_b200.engine import Engine
    m = manager([30, 20], window=[0, 9], slots=6)
    m.open(1)
    hold(m, 1, 14)
    free = [m.free_pages(g) for g in range(2)], m.free_state_slots()

    def fails(copies):
        assert len(copies) == 3
        raise error
    engine = SimpleNamespace(cache=SimpleNamespace(manager=m, copy_fork=fails), _rt=rt)
    with pytest.raises(type(error)):
        Engine.fork_request(engine, 1, [2, 3, 4])
    assert m.live_requests() == 1 and ([m.free_pages(g) for g in range(2)], m.free_state_slots()) == free
    assert m.shared_pages(0) == m.shared_pages(1) == 0 and m.check() == ""
    # too few slots for all of them: none is made, and nothing is copied
    engine.cache.copy_fork = lambda copies: pytest.fail("copied")
    with pytest.raises(MemoryError, match="for the 6th; nothing has changed"):
        Engine.fork_request(engine, 1, list(range(2, 9)))
    assert m.live_requests() == 1 and m.shared_pages(0) == 0 and m.check() == ""
    engine.cache.copy_fork = lambda copies: None
    Engine.fork_request(engine, 1, [2, 3, 4])
    assert m.live_requests() == 4 and m.check() == ""


def test_a_row_that_parted_early_takes_the_sharing_from_no_one():
    """Many answers behind a long prompt, and one conversation more that left it after its first page."""
    m = manager(400, slots=20)
    m.open(1)
    hold(m, 1, 5)
    m.fork(1, 2)                                              # one page in common
    hold(m, 1, 103)
    for c in range(3, 13):
        m.fork(1, c)                                          # 25
    layout, out, _ = batch(m, [2, 1] + list(range(3, 13)), prefix_group=0)
    assert groups_of(layout, out) == [(list(range(1, 12)), 100), ([0], 0)]
    req = rt.BatchRequest()
    req.ids, req.counts, req.tokens, req.want_counts, req.want_index = [2, 1, 3], [1] * 3, [0] * 3, [1] * 3, [0] * 3
    req.prefix_group = 0
    assert rt.count_prefix_groups(m, req) == (1, 100, 100, 6)


def test_several_that_parted_early_share_what_they_have():
    m = manager(400, slots=20)
    m.open(1)
    hold(m, 1, 41)
    for c in (2, 3, 4):
        m.fork(1, c)                                          # ten pages
        hold(m, c, 45)                                        # (and a page of its own)
    hold(m, 1, 85)
    for c in range(5, 10):
        m.fork(1, c)                                          # 21
    layout, out, _ = batch(m, list(range(1, 10)), prefix_group=0)
    assert sorted(groups_of(layout, out)) == sorted([([0, 4, 5, 6, 7, 8], 84), ([1, 2, 3], 40), ([], 0)])


def test_random_trees_of_forks_against_all_ways_of_dividing_their_rows():
    from functools import lru_cache
    rng, optimal = random.Random(11), 0
    for turn in range(40):
        m = manager(2000, slots=10)
        m.open(1)
        hold(m, 1, rng.randint(1, 30))
        live = [1]
        while len(live) < 6:
            if rng.random() < 0.5:
                m.fork(rng.choice(live), len(live) + 1)
                live.append(len(live) + 1)
            else:
                r = rng.choice(live)
                hold(m, r, m.length(r) + rng.randint(1, 14))
        tables = [m.block_table(r, 0)[:m.length(r) // 4] for r in live]
        layout, out, _ = batch(m, live, prefix_group=0)
        found = groups_of(layout, out)[:-1] if layout.num_prefix_groups else []

        @lru_cache(None)
        def shared(rows):
            n = 0
            while all(len(tables[r]) > n for r in rows) and len({tables[r][n] for r in rows}) == 1:
                n += 1
            return n

        @lru_cache(None)
        def best(rows):                                       # (all divisions of a set)
            if len(rows) < 2:
                return 0
            lead, rest = rows[0], rows[1:]
            most = 0
            for pick in range(1 << len(rest)):
                mine = (lead,) + tuple(r for i, r in enumerate(rest) if pick >> i & 1)
                most = max(most, (len(mine) - 1) * shared(mine) + best(tuple(r for i, r in enumerate(rest) if not pick >> i & 1)))
            return most
        for rows, keys in found:
            assert len(rows) > 1 and keys == 4 * shared(tuple(rows)) > 0
        assert sorted(r for rows, _ in groups_of(layout, out) for r in rows) == list(range(6)) if found else True
        saved, most = sum((len(rows) - 1) * keys for rows, keys in found) // 4, best(tuple(range(6)))
        assert saved >= 5 * shared(tuple(range(6))) and saved >= 0.8 * most, (turn, saved, most)
        optimal += saved == most
        assert m.check() == ""
    assert optimal >= 35


def test_shared_pages_are_looked_for_where_a_mixer_reads_them_once(tiny):
    import importlib

    import torch

    from llm_infer_rust_b200.cache import plan_cache
    from llm_infer_rust_b200.config import resolve_architecture
    from llm_infer_rust_b200.engine.engine import prefix_group
    from llm_infer_rust_b200.parts import DecoderModel, int8_projections

    def group_of(raw, change=lambda spec: spec):
        arch = resolve_architecture(raw)
        model = DecoderModel(change(arch.model_spec(arch.parse_config(raw))), torch.float32, torch.device("cpu"))
        plan = plan_cache(model, 8, 4)
        found, heads = prefix_group(model, plan)
        assert not heads if found < 0 else plan.groups[found].window is None and heads == [tuple(model.blocks[0].mixer.spec[n] for n in ("num_heads", "num_kv_heads", "head_dim"))]
        return found
    for name in "ABCDE":
        assert group_of(tiny[name]["raw"]) >= 0 and group_of(tiny[name]["raw"], int8_projections) >= 0
    for kit in ("bevuvik", "kefetar", "lufizen", "mukenex", "sigudra", "torinex"):
        made = importlib.import_module(f"{kit}_kit")
        for raw in made.CONFIGS.values():
            assert group_of(getattr(made, "as_given", dict)(raw)) == -1, kit


def test_a_long_row_is_not_what_a_call_is_cut_up_for():
    """The rows' own keys that a step names: not those of one row that shares nothing, where the kernels share all rows' out evenly."""
    from types import SimpleNamespace

    import torch

    from llm_infer_rust_b200.engine import Engine
    m = manager(9000, slots=60)
    m.open(1)
    hold(m, 1, 4004)
    m.fork(1, 2)
    hold(m, 1, 16384)
    for c in range(3, 50):
        m.fork(1, c)
    ids = [1, 2] + list(range(3, 50))
    req = rt.BatchRequest()
    req.ids, req.counts, req.tokens, req.want_counts, req.want_index = ids, [1] * 49, [0] * 49, [1] * 49, [0] * 49
    for dtype, heads, own in ((torch.bfloat16, (16, 8, 128), 2 * -(-(48 + 4005) // 49)), (torch.float32, (16, 8, 128), 4005), (torch.bfloat16, (32, 1, 128), 4005)):
        engine = SimpleNamespace(cache=SimpleNamespace(manager=m, page_sizes=[4]), _rt=rt, _prefix_group=0, _prefix_heads=[heads], dtype=dtype,
                                 _prefix_places=Engine._prefix_places)
        assert Engine._look_for_prefixes(engine, req, None, [m.length(r) + 1 for r in ids]) == (1, 16384, own), dtype
