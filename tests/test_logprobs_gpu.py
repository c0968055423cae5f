"""Log probabilities, entropy and the most likely tokens against 64 bits.

What may differ.  d = l - m is off by 2^-24 |d|, the exponential's argument d log2 e by as much again, the exponential itself by 2^-22;
weighted with p these are (2 sum p |d| + 4) 2^-24 of the sum s, and its additions come in chains of at most n / 512 + 17 and trees
of 20: with c = n / 512 + 41 a log probability is off by (2 sum p |d| + c) 2^-24 plus the roundings of its own two
subtractions and the logarithm, 3 |log p| 2^-24.  The entropy's sum has the same error of each of its terms:
2 (2 sum p |d| + c) 2^-24 (1 + sum p |d|).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")


def ops():
    from llm_infer_rust_b200.kernels import ops as m
    return m


def check(logits, tokens, top, found):
    ops().check_errors(logits.device)
    rows, vocab = logits.shape
    l = logits.double().cpu()
    m = l.amax(1, keepdim=True)
    p = torch.softmax(l, 1)
    spread = torch.where(p > 0, p * (l - m).abs(), torch.zeros_like(p)).sum(1)
    lp = torch.log_softmax(l, 1)
    c = vocab / 512 + 41
    unit = (2 * spread + c) * 2.0 ** -24

    def near(got, want, row):
        same = got == want                                       # (-inf)
        assert (same | ((got - want).abs() <= unit[row] + 3 * want.abs() * 2.0 ** -24)).all(), (got, want)
    if tokens is not None:
        assert found.logprobs.shape == (rows,) and found.logprobs.dtype == torch.float32
        want = lp.gather(1, tokens.long().cpu()[:, None])[:, 0]
        near(found.logprobs.double().cpu(), want, torch.arange(rows))
    else:
        assert found.logprobs is None
    h = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
    assert ((found.entropy.double().cpu() - h).abs() <= 2 * unit * (1 + spread)).all()
    assert found.top_ids.shape == (rows, top) and found.top_logprobs.shape == (rows, top)
    if top:
        order = torch.sort(logits.cpu(), dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(found.top_ids.cpu().long(), order)
        near(found.top_logprobs.double().cpu(), lp.gather(1, order), torch.arange(rows)[:, None])


def logits_of(rows, vocab, seed=0, apart=0, shift=0, scale=3.0):
    g = torch.Generator().manual_seed(seed + rows + vocab)
    wide = torch.full((rows, vocab + apart + shift), NAN, device=DEV)
    x = wide[:, shift:shift + vocab]
    x.copy_((torch.randn(rows, vocab, generator=g) * scale).to(DEV))
    return x


def given(rows, vocab, seed=0):
    return torch.randint(vocab, (rows,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(DEV)


@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("rows,vocab,apart,shift", [
    (1, 32, 0, 0), (3, 33, 0, 0), (2, 100, 3, 1), (5, 511, 1, 3), (1, 2048, 0, 0), (7, 2049, 0, 2), (1, 8192, 0, 0), (3, 16385, 5, 1),
    (45, 32003, 29, 0), (1, 151936, 0, 0), (9, 151936, 0, 0), (200, 50001, 2, 1), (2, 300001, 0, 0)])
def test_against_64_bits(rows, vocab, apart, shift, top):
    x, t = logits_of(rows, vocab, apart=apart, shift=shift), given(rows, vocab)
    check(x, t, top, ops().token_logprobs(x, t, top=top))


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 7])
def test_tiny_vocabularies(vocab):
    x, t = logits_of(3, vocab), given(3, vocab)
    check(x, t, vocab, ops().token_logprobs(x, t, top=vocab))


def test_without_given_tokens():
    x = logits_of(4, 1000)
    check(x, None, 3, ops().token_logprobs(x, top=3))


@pytest.mark.parametrize("rows", [1, 150])
def test_the_best_stand_anywhere(rows):
    """Rising, falling, all in one thread's elements, all in one vector, all at the ends, all alike, few alike."""
    vocab, top = 50003, 32
    up = torch.arange(vocab, dtype=torch.float32) * 1e-3
    cases = [up, -up, torch.zeros(vocab)]
    for at in (torch.arange(32) * 2048 % 49152 + 3, torch.arange(32) + 20000, torch.arange(32) * 4 + 1,
               torch.cat([torch.arange(16), vocab - 1 - torch.arange(16)])):
        x = torch.randn(vocab, generator=torch.Generator().manual_seed(3))
        x[at] = 9.0 + (torch.arange(32) % 5).float()
        cases.append(x)
    cases.append((torch.randn(vocab, generator=torch.Generator().manual_seed(4)) * 2).round())
    cases.append(torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0))
    for case in cases:
        x = case.to(DEV).expand(rows, vocab).contiguous()
        t = given(rows, vocab)
        check(x, t, top, ops().token_logprobs(x, t, top=top))


@pytest.mark.parametrize("rows", [2, 150])
@pytest.mark.parametrize("left", [1, 2, 20, 33, 4000])
def test_forbidden_tokens(rows, left):
    vocab = 32001
    x = logits_of(rows, vocab)
    allowed = torch.randperm(vocab, generator=torch.Generator().manual_seed(left))[:left].to(DEV)
    y = torch.full_like(x, -INF)
    y[:, allowed] = x[:, allowed]
    t = given(rows, vocab)                      # (hardly any of them allowed: -inf)
    t[0] = int(allowed[0])
    check(y, t, 32, ops().token_logprobs(y, t, top=32))


def test_the_types_lowest_value_as_a_mask():
    x = logits_of(4, 32001)
    x[:, 100:] = torch.finfo(torch.float32).min
    t = given(4, 100)
    check(x, t, 20, ops().token_logprobs(x, t, top=20))


def test_certain_and_undecided_rows():
    x = torch.zeros(3, 151936, device=DEV)
    x[0, 77] = 80.0
    x[1, 5] = 3e38
    t = torch.tensor([77, 5, 9], dtype=torch.int32, device=DEV)
    check(x, t, 2, ops().token_logprobs(x, t, top=2))


@pytest.mark.parametrize("vocab", [40, 151936])
def test_rows_without_a_distribution(vocab):
    x = logits_of(6, vocab)
    x[0, 7] = NAN
    x[1, 9] = INF
    x[2] = -INF
    x[3] = NAN
    x[4, 8:] = NAN
    t = given(6, vocab)
    f = ops().token_logprobs(x, t, top=20)
    ops().check_errors(x.device)
    for r in range(5):
        assert f.logprobs[r].isnan() and f.entropy[r].isnan() and f.top_logprobs[r].isnan().all(), r
    clean = torch.where(x.isnan(), torch.full_like(x, -INF), x)
    order = torch.sort(clean.cpu(), dim=1, descending=True, stable=True).indices[:, :20].int()
    assert torch.equal(f.top_ids[[0, 1, 2]].cpu(), order[[0, 1, 2]])
    assert (f.top_ids[3] == -1).all()
    assert torch.equal(f.top_ids[4, :8].cpu(), order[4, :8]) and (f.top_ids[4, 8:] == -1).all()
    check(x[5:], t[5:], 20, ops().token_logprobs(x[5:], t[5:], top=20))


@pytest.mark.parametrize("bad", [-1, 1000, 2 ** 31 - 1, -2 ** 31])
def test_tokens_outside_the_vocabulary(bad):
    x = logits_of(3, 1000)
    t = torch.tensor([5, bad, 6], dtype=torch.int32, device=DEV)
    f = ops().token_logprobs(x, t, top=2)
    with pytest.raises(ops().KernelError, match="token id"):
        ops().check_errors(x.device)
    assert f.logprobs[1].isnan() and not f.logprobs[[0, 2]].isnan().any() and not f.entropy.isnan().any()


def test_streams_and_graphs():
    x, t = logits_of(5, 40001), given(5, 40001)
    want = ops().token_logprobs(x, t, top=7)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = ops().token_logprobs(x, t, top=7)
    here = ops().token_logprobs(x, t, top=7)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = ops().token_logprobs(x, t, top=7)
    graph.replay()
    torch.cuda.synchronize()
    for f in (other, here, held):
        assert all(torch.equal(a, b) for a, b in zip(f, want))
    x.copy_(logits_of(5, 40001, seed=9))
    t.copy_(given(5, 40001, seed=9))
    graph.replay()
    torch.cuda.synchronize()
    check(x, t, 7, held)


def test_rows_beyond_2_31_elements():
    rows, vocab = 15000, 151936                                  # 9.1 GB
    x = torch.zeros(rows, vocab, device=DEV)
    x[-1] = logits_of(1, vocab)[0]
    t = given(rows, vocab)
    f = ops().token_logprobs(x, t, top=3)
    check(x[-1:], t[-1:], 3, ops().TokenLogprobs(*(a[-1:] for a in f)))


def test_no_rows():
    f = ops().token_logprobs(torch.zeros(0, 100, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), top=4)
    assert f.logprobs.shape == (0,) and f.top_ids.shape == (0, 4)


def test_one_row_for_many_tokens():
    """Rows that are one row again and again, and rows that overlap."""
    x, t = logits_of(1, 5000).expand(7, -1), given(7, 5000)
    check(x, t, 4, ops().token_logprobs(x, t, top=4))
    x = logits_of(1, 5000)[0].as_strided((7, 4000), (130, 1))
    t = given(7, 4000)
    check(x, t, 4, ops().token_logprobs(x, t, top=4))
