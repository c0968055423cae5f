"""What attention behind shared prefixes, page copies and log probabilities refuse, where no GPU is needed to say so."""
import ctypes

import pytest
import torch

from llm_infer_rust_b200 import SamplingParams
from llm_infer_rust_b200.kernels import ops, pages, prefix
from llm_infer_rust_b200.kernels.build import load_cuda_library
from llm_infer_rust_b200.kernels.ops import KernelError

I32 = dict(dtype=torch.int32)


def operands(dtype=torch.float32, heads=4, kv_heads=2, dim=16, page=8, n=3):
    cache = torch.zeros(9, kv_heads, page, dim, dtype=dtype)
    return dict(q=torch.zeros(n, heads * dim, dtype=dtype), k_cache=cache, v_cache=cache.clone(), out=torch.zeros(n, heads * dim, dtype=dtype),
                block_table=torch.zeros(n, 4, **I32), cu_q=torch.arange(n + 1, **I32), kv_len=torch.ones(n, **I32), rows=torch.arange(n, **I32),
                groups=torch.zeros(1, 2, **I32), num_heads=heads, num_kv_heads=kv_heads, head_dim=dim, page_size=page, scale=0.25,
                most_rows=n, most_shared=8, most_own=8)


def test_no_path_on_the_cpu():
    with pytest.raises(KernelError, match="CUDA"):
        prefix.prefix_attention(**operands())
    with pytest.raises(KernelError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 8))
    with pytest.raises(KernelError, match="CUDA"):
        pages.PageCopier([torch.zeros(4, 2, 8, 16)])


@pytest.mark.parametrize("change,what", [
    (dict(num_heads=3), "multiple of num_kv_heads"), (dict(num_kv_heads=0), "multiple of num_kv_heads"), (dict(head_dim=15), "even head sizes"),
    (dict(head_dim=514), "even head sizes"), (dict(most_rows=-1), "negative"), (dict(most_own=-1), "negative"), (dict(sharing_groups=-1), "negative")])
def test_sizes_that_are_refused(change, what):
    with pytest.raises(KernelError, match=what):
        prefix.prefix_attention(**{**operands(), **change})


@pytest.mark.parametrize("change,what", [
    (dict(k_cache=torch.zeros(9, 2, 8, 16, dtype=torch.bfloat16)), "share a dtype"), (dict(out=torch.zeros(3, 64, dtype=torch.bfloat16)), "share a dtype"),
    (dict(q=torch.zeros(3, 64, dtype=torch.float16)), "not supported"), (dict(rows=torch.arange(3)), "are int32"),
    (dict(groups=torch.zeros(1, 2)), "are int32"), (dict(v_cache=torch.zeros(8, 2, 8, 16)), "as many pages"),
    (dict(k_cache=torch.zeros(9, 2, 4, 16)), "cache must be"), (dict(q=torch.zeros(3, 32)), "num_heads"), (dict(out=torch.zeros(2, 64)), "num_heads"),
    (dict(block_table=torch.zeros(3, 0, **I32)), "block_table is"), (dict(groups=torch.zeros(2, **I32)), "block_table is"),
    (dict(groups=torch.zeros(1, 3, **I32)), "block_table is"), (dict(rows=torch.zeros(3, 1, **I32)), "block_table is"),
    (dict(q=torch.zeros(64, 3).t()), "non-contiguous"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale")])
def test_operands_that_are_refused(monkeypatch, change, what):
    monkeypatch.setattr(ops, "_cuda", lambda *tensors: None)
    o = {**operands(), **change}
    for name in ("most_rows", "most_shared", "most_own"):
        o.pop(name)
    with pytest.raises(KernelError, match=what):
        prefix._refuse(**o)
    prefix._refuse(**{k: v for k, v in operands().items() if not k.startswith("most")})      # (and nothing else is)


def test_calls_go_where_they_are_served():
    def plan(dtype=torch.bfloat16, heads=32, kv_heads=8, dim=128, page=16, n_rows=64, n_groups=1, most_rows=64, shared=4096, own=100, sharing=1, aligned=True):
        got = prefix._plan(dtype, heads, kv_heads, dim, page, n_rows, n_groups, most_rows, shared, own, sharing, aligned, 148)
        return ["all sizes", "tcgen05", "mma"][0 if got[0] is not None else 1 if got[1] is not None else 2], got[3]
    assert plan()[0] == "tcgen05"
    floats, splits, _, tiles, two, covered, ctas, sms = plan()[1]
    assert (tiles, two, covered, sms) == (1, 1, 256, 148) and 8 * splits + ctas <= 148      # (side by side)
    floats, splits, _, tiles, two, covered, ctas, sms = plan(most_rows=32, n_rows=32)[1]
    assert (tiles, two, covered) == (1, 0, 128) and splits % 2 == 0 and 8 * splits // 2 + ctas <= 148      # one tile: a CTA leaves two parts
    assert plan(most_rows=4)[0] == "mma" and plan(shared=416)[0] == "mma" and plan(dim=64)[0] == "mma"
    assert plan(shared=417)[0] == "tcgen05" and plan(most_rows=8, shared=3489)[0] == "tcgen05" and plan(most_rows=8, shared=3488)[0] == "mma"
    assert plan(most_rows=8, shared=4609)[0] == "mma" and plan(most_rows=8, shared=5793)[0] == "tcgen05"      # (a second step)
    assert plan(page=24)[0] == "mma"
    for other in (dict(dtype=torch.float32), dict(dim=72), dict(heads=17, kv_heads=1), dict(n_rows=400), dict(aligned=False)):
        assert plan(**other)[0] == "all sizes", other
    assert plan(n_rows=399)[0] == "tcgen05"
    # own keys that outweigh the shared ones come behind them, on all SMs or on most
    assert plan(own=1)[1][6] < plan(own=4000)[1][6]
    assert plan(n_groups=4, sharing=3, most_rows=16, shared=4064)[0] == "mma" and plan(n_groups=4, sharing=3, most_rows=16, shared=4097)[0] == "tcgen05"
    # groups that share nothing are no reason to cut the others into fewer splits
    assert plan(n_groups=3)[1][1] == plan(n_groups=3, sharing=1)[1][1] > plan(n_groups=3, sharing=3)[1][1]


@pytest.mark.parametrize("moves,rc", [
    ([(0, 1, 4)], None), ([(0, 1, 4), (2, 1, 4)], -11), ([(0, 1, 4), (1, 2, 4)], -11), ([(3, 3, 4)], -11), ([(0, 9, 4)], -10), ([(9, 1, 4)], -10),
    ([(-1, 2, 4)], -10), ([(0, 2, 5)], -10), ([(0, 2, -1)], -10), ([(0, 2 ** 31 - 1, 1)], -10)])
@pytest.mark.parametrize("before", [0, 20])
def test_moves_are_checked_before_anything_runs(moves, rc, before):
    """``before``: so many good moves in front (the two ways of comparing pages)."""
    if rc is None:
        return                                                     # (a good call would launch)
    entry = load_cuda_library("pages.cu").b200_copy_pages
    entry.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_longlong,
                      ctypes.c_void_p]
    pages_there = 9 + 2 * before
    table = torch.zeros(4, dtype=torch.int64)
    all_moves = [(9 + i, 9 + before + i, 4) for i in range(before)] + [tuple(pages_there if x == 9 and i < 2 else x for i, x in enumerate(m)) for m in moves]
    m = torch.tensor(all_moves, dtype=torch.int32)
    assert entry(m.data_ptr(), len(all_moves), table.data_ptr(), 1, pages_there, 4, 16, 256, None) == rc


def test_c_entry_points_refuse_what_they_cannot_serve():
    lib = load_cuda_library("logprobs.cu")
    none = ctypes.c_void_p()
    some = ctypes.c_void_p(1 << 20)                                # (never followed)

    def logprobs(rows=1, vocab=100, top=0, stride=100, logits=some, tokens=none, chosen=none, entropy=some, ids=none, best=none, err=some):
        return lib.b200_token_logprobs(logits, ctypes.c_longlong(stride), rows, vocab, tokens, top, chosen, entropy, ids, best, err, none)
    assert logprobs(rows=0) == 0
    for bad in (dict(rows=-1), dict(vocab=0), dict(top=-1), dict(top=33), dict(vocab=3, top=4), dict(stride=-1), dict(logits=none),
                dict(entropy=none), dict(err=none), dict(tokens=some), dict(top=1), dict(top=1, ids=some), dict(vocab=2 ** 31 - 1), dict(rows=2 ** 30)):
        assert logprobs(**bad) == -2, bad


def test_entry_points_of_the_attention_refuse_what_they_cannot_serve():
    none, some = ctypes.c_void_p(), ctypes.c_void_p(1 << 20)       # (never followed)
    names = ("q", "k", "v", "out", "scratch", "table", "cu", "lengths", "rows", "groups", "err")
    mma = load_cuda_library("prefix_mma.cu", {"HEAD_DIM": 128})
    tc = load_cuda_library("prefix_tcgen05.cu")
    every = load_cuda_library("prefix_attention.cu", {"HEAD_DIM": 128})

    def call(kind, n_rows=2, n_groups=1, nh=8, nkv=2, page=16, pages=9, scale=0.1, stride=4, last=None, **change):
        p = {**{x: some for x in names}, **change}
        args = [p["q"], p["k"], p["v"]] + ([p["out"]] if kind != "tc" else [])
        args += [p["scratch"], p["table"], stride, p["cu"], p["lengths"], p["rows"], n_rows, p["groups"], n_groups, nh, nkv, page, pages, ctypes.c_float(scale)]
        tail = {"mma": [0, 0, 148, 148], "tc": [2, 1, 0], "every": [1, 1, 1, 1, 128, 148]}[kind] if last is None else last
        entry = {"mma": mma.b200_prefix_attention_mma, "tc": tc.b200_prefix_tcgen05, "every": every.b200_prefix_attention}[kind]
        return entry(*args, *tail, p["err"], none)

    for kind in ("mma", "tc", "every"):
        assert call(kind, n_rows=0) == 0 and call(kind, n_rows=-1) == 0
        for name in names:
            if kind != "tc" or name != "out":
                assert call(kind, **{name: none}) == -2, (kind, name)
        # sizes; tables of more than 2^30 places
        for bad in (dict(nh=0), dict(nkv=0), dict(nh=7), dict(page=0), dict(pages=0), dict(stride=0), dict(stride=2 ** 27), dict(n_groups=-1)):
            assert call(kind, **bad) == (0 if kind == "tc" and "n_groups" in bad else -2), (kind, bad)
    assert call("tc", page=24) == -2
    for kind in ("mma", "tc"):
        assert call(kind, pages=2 ** 27) == -2 and call(kind, q=ctypes.c_void_p((1 << 20) + 8)) == -3
    assert call("mma", nh=34) == -2 and call("mma", n_rows=400) == -2 and call("mma", last=[2, 0, 148, 148]) == -2 and call("mma", last=[0, 0, 149, 148]) == -2
    assert call("tc", scale=0.0) == -2 and call("tc", last=[3, 1, 0]) == -2 and call("tc", last=[0, 1, 1]) == -2
    assert call("every", last=[1, 1, 1, 1, 130, 148]) == -2 and call("every", last=[1, 1, 1, 1, 127, 148]) == -2 and call("every", last=[0, 1, 1, 1, 128, 148]) == -2


@pytest.mark.parametrize("logprobs", [-1, 33])
def test_sampling_params_refuse(logprobs):
    with pytest.raises(ValueError, match="0 to 32"):
        SamplingParams(logprobs=logprobs).normalized()
    assert SamplingParams(logprobs=5).normalized().logprobs == 5 and SamplingParams().normalized().logprobs is None


def test_options_of_the_command_line(capsys):
    from llm_infer_rust_b200 import cli
    args = cli.parse_args(["--model-path", "x", "--answers", "4", "--logprobs", "3"])
    assert (args.answers, args.logprobs) == (4, 3)
    for bad in (["--answers", "0"], ["--answers", "9", "--max-running-req", "8"], ["--logprobs", "33"], ["--logprobs", "-1"]):
        assert cli.main(["--model-path", "x", "--prompt-ids", "1"] + bad) == 2
    assert "--answers" in cli.USAGE and "--logprobs" in cli.USAGE


def test_calls_that_the_tensor_core_kernels_cannot_count():
    def counts(pages=1000, kv_heads=8, page=16, width=100, n_rows=4, n_groups=1, heads=32):
        return prefix._counts(torch.empty(pages, kv_heads, page, 1, device="meta"), torch.empty(n_rows, width, device="meta"), n_rows, n_groups, heads,
                              kv_heads, page)
    assert counts() and counts(pages=2 ** 24 - 1) and not counts(pages=2 ** 24)
    items = 1 + 1 + 4                                          # tiles of 16 vectors, groups, rows
    most = (2 ** 30 - 1) // (8 * items) - 2                    # blocks of a row
    assert counts(width=2 * most) and not counts(width=2 * (most + 1))


def test_shared_keys_are_read_once_where_that_was_measured_to_pay():
    BF16, F32, MiB = torch.bfloat16, torch.float32, 1 << 20

    def pays(mib, rows, groups=2, heads=16, kv_heads=8, dim=128, dtype=BF16, page=16, own=64, least=48 * MiB):
        a_key = 2 * kv_heads * dim * dtype.itemsize
        saved = int(mib * MiB) // a_key
        return prefix.pays(dtype, heads, kv_heads, dim, page, rows, groups, saved, saved // (rows - 1) + rows * own, least)
    assert pays(48, 16) and not pays(47, 16) and pays(48, 2) and pays(512, 48) and not pays(30, 48)
    assert pays(64, 16, heads=64) and not pays(63, 16, heads=64) and pays(64, 16, heads=16, kv_heads=1) and not pays(56, 16, heads=16, kv_heads=1)
    # rows with many keys of their own
    assert not pays(48, 128, own=600) and pays(64, 128, own=600) and not pays(64, 384, own=600) and pays(160, 384, own=600)
    # more rows and groups than the tensor-core kernels take, where decode attention has its own
    for mib in (28, 128, 512, 4096, 1 << 20):
        for own in (1, 64, 600):
            assert not pays(mib, 450, own=own) and not pays(mib, 512, own=own) and not pays(mib, 399, own=own)
    assert pays(512, 398, groups=2) and not pays(512, 398, groups=3)
    # the all-sizes kernel against decode attention's
    assert not pays(128, 64, heads=8, dim=72, own=600) and pays(128, 16, heads=8, dim=72) and not pays(512, 4, dim=320) and pays(512, 64, dim=320, own=16)
    assert pays(32, 450, heads=32, kv_heads=1) and pays(32, 2, dtype=F32) and pays(32, 450, dtype=F32, own=600) and not pays(31, 8, dtype=F32)
    # (pages of no power of two are the all-sizes kernel's in decode attention)
    assert pays(48, 16, page=24) and not pays(512, 450, page=24, own=600)
    # nothing saved, and nothing asked for
    assert not pays(0, 16) and pays(1, 16, least=1, own=1)


def test_groups_that_share_nothing_get_no_ctas_of_the_tcgen05_kernel():
    def served(n_groups, sharing):
        got = prefix._plan(torch.bfloat16, 32, 8, 128, 16, 64, n_groups, 64, 32768, 100, sharing, True, 148)
        assert got[1] is not None
        return got[3][2]
    assert [served(2, 1), served(5, 4), served(3, 3), served(9, 0)] == [1, 4, 3, 1]
    # the entry points take the groups beside the tiles and the vectors, and refuse more groups than there are
    none, some = ctypes.c_void_p(), ctypes.c_void_p(1 << 20)       # (never followed)
    entry = load_cuda_library("prefix_tcgen05.cu").b200_prefix_tcgen05
    for tiles in (1 | 3 << 16, 3 << 16, 1 << 16):
        assert entry(some, some, some, some, some, 4, some, some, some, 2, some, 2, 8, 2, 16, 9, ctypes.c_float(0.1), 2, tiles, 0, some, none) == -2
