"""token_logprobs against the definition in 64 bits, on an MI355X.

Tolerances, before any run: a thread sums up to V / 256 exponentials one after another (a random walk of half
steps of 2^-24: 42 at 460,000 tokens), each within 3 steps (its argument's rounding and exp2's), and the joins add
20: under 2^-17 of the sum, so of log s and, times the largest |x - m| that weighs anything (20), of w / s relative
to 1 + entropy by 2^-16. x - m and the log round at 2^-24 of themselves. Tokens and ranks are equal.
"""

import pytest
import torch

from linuxformer_amd import mk_build
from linuxformer_amd.score import token_logprobs

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def cuda():
    assert torch.cuda.is_available(), "the gpu tests need an MI355X"
    mk_build.load()
    return torch.device("cuda", 0)


def _near(got, ref, tol):
    got = got.double().cpu()
    fine = ref.isfinite()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()])
    off = (got - ref)[fine].abs() - tol * (1 + ref[fine].abs())
    assert not (off > 0).any(), float(off.max())


def _check(x, tokens, top, r):
    """r against the definition: x on the CPU, its values as float32 (-0 is 0)."""
    x = x.float() + 0.0
    N, V = x.shape
    lp = torch.log_softmax(x.double(), 1)
    lp[(x == INF).any(1) | x.isnan().any(1) | (x == -INF).all(1)] = NAN
    ok = (tokens >= 0) & (tokens < V)
    t = tokens.clamp(0, V - 1).long()[:, None]
    _near(r.logprob, torch.where(ok, lp.gather(1, t)[:, 0], torch.where(tokens < 0, 0.0, NAN).double()), 2.0 ** -17)
    p = lp.exp()
    _near(r.entropy, -(p * lp.masked_fill(p == 0, 0)).sum(1), 2.0 ** -16)
    y = x.masked_fill(x.isnan(), INF)  # (in the order a NaN is first; the tests with NaN hold no inf)
    order = torch.sort(y, dim=1, descending=True, stable=True).indices
    rank = (order == t).int().argmax(1)
    nan_token = x.gather(1, t)[:, 0].isnan()
    assert r.rank.cpu().tolist() == torch.where(ok & ~nan_token, rank, -1).tolist()
    k = min(top, V)
    assert r.top_tokens.shape == (N, k) and torch.equal(r.top_tokens.cpu().long(), order[:, :k])
    _near(r.top_logprobs, lp.gather(1, order[:, :k]), 2.0 ** -17)


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("N,V,top", [(1, 1, 1), (3, 7, 64), (1, 8192, 5), (2, 8201, 64), (5, 31999, 20), (1, 459982, 8),
                                     (1300, 500, 3), (2, 100003, 0), (1030, 16411, 1), (7, 65, 64)])
def test_token_logprobs(cuda, N, V, top, dt):
    print(f"[gpu-test] token_logprobs {N}x{V} top {top} {dt}", flush=True)
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(N, V, generator=g)).to(dt)
    tokens = torch.randint(-1, V + 1, (N,), generator=g)
    tokens[0] = x[0].float().argmax()
    _check(x, tokens, top, token_logprobs(x.to(cuda), tokens.to(cuda), top))


ROWS = {
    "ties": lambda V: torch.zeros(V),
    "rising": lambda V: torch.arange(V) / 64.0,
    "falling": lambda V: -torch.arange(V) / 64.0,
    "masked": lambda V: torch.where(torch.arange(V) % 997 == 5, 1.0, -INF),
    "nothing": lambda V: torch.full((V,), -INF),
    "one": lambda V: torch.where(torch.arange(V) == V - 1, 3.0, -INF),
    "lowest": lambda V: torch.full((V,), torch.finfo(F32).min).index_fill(0, torch.tensor([V // 2]), 0.0),
    "far": lambda V: torch.where(torch.arange(V) % 2 == 0, 3.0e4, -3.0e4),
    "zeros": lambda V: torch.where(torch.arange(V) % 3 == 0, -0.0, 0.0),
    "nan": lambda V: torch.arange(V) % 5.0 + torch.where(torch.arange(V) % 4999 == 17, NAN, 0.0),
    "nans": lambda V: torch.full((V,), NAN),
    "inf": lambda V: torch.arange(V) % 7.0 + torch.where(torch.arange(V) == V // 3, INF, 0.0),
}


@pytest.mark.parametrize("parts", [1, 4])
@pytest.mark.parametrize("V", [130, 20001, 40000])
def test_rows_that_go_wrong(cuda, V, parts):
    """Rows whose maximum, order or sum is special, in rows of many parts and of one, the tokens at the start, the
    middle and the end."""
    print(f"[gpu-test] special rows {V} parts {parts}", flush=True)
    copies = 1 if parts > 1 else 100  # (many rows: one part each)
    x = torch.stack([f(V) for f in ROWS.values()]).repeat(copies, 1)
    for dt in (F32, BF):
        y = x.to(dt)
        for i, top in ((0, 64), (V // 2, 20), (V - 1, 1)):
            tokens = torch.full((len(y),), i)
            n = len(ROWS)
            r = token_logprobs(y.to(cuda), tokens.to(cuda), top)
            for a in (0, len(y) - n):
                _check(y[a:a + n], tokens[a:a + n], top, type(r)(*(t[a:a + n] for t in r)))


def test_strides_alignment_types(cuda):
    """Rows of a wider buffer at every alignment (what lies around them is NaN), int32 tokens, columns that are
    not dense, a row past 2^31 elements, no rows."""
    print("[gpu-test] score strides", flush=True)
    g = torch.Generator().manual_seed(0)
    for dt in (BF, F32):
        for lead in range(8):
            x = torch.randn(3, 9001, generator=g).to(dt)
            buf = torch.full((3, 9101 + lead), NAN, dtype=dt, device=cuda)
            view = buf[:, lead:lead + 9001]
            view.copy_(x)
            tokens = torch.tensor([0, 9000, 4500], dtype=torch.int32)
            _check(x, tokens, 10, token_logprobs(view, tokens.to(cuda), 10))
    x = torch.randn(300, 4, generator=g)
    _check(x.T, torch.arange(4), 3, token_logprobs(x.to(cuda).T, torch.arange(4, device=cuda), 3))
    r = token_logprobs(torch.empty(0, 10, device=cuda), torch.empty(0, dtype=torch.int64, device=cuda), 3)
    assert r.logprob.shape == (0,) and r.top_tokens.shape == (0, 3)
    big = torch.empty(2, (1 << 31) + 8, dtype=BF, device=cuda)[:, :9001]
    y = torch.randn(2, 9001, generator=g).to(BF)
    big.copy_(y)
    _check(y, torch.tensor([3, 4]), 5, token_logprobs(big, torch.tensor([3, 4], device=cuda), 5))


@pytest.mark.parametrize("N,V", [(2, 30000), (1100, 700)])
def test_score_graph_and_stream(cuda, N, V):
    """Captured and replayed with eager work between the replays, on a stream of its own: the eager bits."""
    print(f"[gpu-test] score graph {N}x{V}", flush=True)
    x, t = torch.randn(N, V, device=cuda), torch.randint(0, V, (N,), device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = token_logprobs(x, t, 6)
    for _ in range(4):
        graph.replay()
        b = token_logprobs(x, t, 6)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            c = token_logprobs(x, t, 6)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) and torch.equal(u, w) for u, v, w in zip(a, b, c))
        x.normal_()


def test_top_is_read_at_each_call(cuda):
    """A number of alternatives in a tensor that is changed between two calls."""
    x, t, top = torch.randn(3, 100, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda), torch.tensor(2)
    assert token_logprobs(x, t, top=top).top_tokens.shape == (3, 2)
    top.fill_(5)
    assert token_logprobs(x, t, top=top).top_tokens.shape == (3, 5)


def test_long_sums_of_equal_terms(cuda):
    """Rows of one value behind the maximum, whose equal terms round the same way at each addition, in rows of one
    part. Steps of 2^-24 of the sum: a term is within 3.25 (its argument's product and constant at |x - m| <= 1: 1.25;
    exp2: 2), 32 equal terms added one after another within 16.5, their sums, joined without loss, 2, 10 joins of waves
    and lanes: 32 of s. The log moves by as much and rounds by 16 (a step at 12.5), the last difference by 8: 56,
    below 2^-18. w / s is at most 1 and has both sums' errors and 2 roundings, w's terms one more: 70 beside the log's
    48, below 2^-17."""
    print("[gpu-test] score, long sums", flush=True)
    c = torch.arange(1, 17) / 16
    x = torch.zeros(1024, 248320, dtype=BF, device=cuda)
    x[:, 8320:] = -c.repeat(64)[:, None].to(cuda)  # (every thread of 32 elements in turn has met the maximum)
    r = token_logprobs(x, torch.zeros(1024, dtype=torch.int32, device=cuda))
    n, c = 240000, c.double()
    s = 8320 + n * torch.exp(-c)
    ref, entropy = -s.log(), s.log() + n * c * torch.exp(-c) / s
    assert (r.logprob.double().cpu() - ref.repeat(64)).abs().max() <= 2.0 ** -18
    assert (r.entropy.double().cpu() - entropy.repeat(64)).abs().max() <= 2.0 ** -17


@pytest.mark.parametrize("N,V", [(3, 30000), (1100, 70)])
def test_results_are_tensors_of_their_own(cuda, N, V):
    """Each result may be kept, saved, changed in place or weighed with something that learns, whatever becomes of the
    others and of the call's workspace."""
    print(f"[gpu-test] score results {N}x{V}", flush=True)
    r = token_logprobs(torch.randn(N, V, device=cuda), torch.zeros(N, dtype=torch.int32, device=cuda), 5)
    assert all(t._base is None and t.untyped_storage().nbytes() == t.numel() * t.element_size() for t in r)
    w = torch.ones(N, device=cuda, requires_grad=True)
    loss = (w * r.logprob).sum()
    r.rank.add_(1), r.top_tokens.zero_()
    loss.backward()
    assert torch.equal(w.grad, r.logprob)
    r.logprob.mul_(w)
    assert r.logprob.requires_grad


def test_more_rows_than_a_launch_holds(cuda):
    """A launch's threads are counted in 32 bits: rows past 16,777,215 workgroups of 256 go in another."""
    print("[gpu-test] score of many rows", flush=True)
    N = 16_777_300
    x, t = torch.randn(N, 2, device=cuda), torch.randint(0, 2, (N,), dtype=torch.int32, device=cuda)
    r = token_logprobs(x, t, 1)
    lp = torch.log_softmax(x.double(), 1)
    ref = lp.gather(1, t[:, None].long())[:, 0]
    best = x.max(1)
    first = torch.where(x[:, 0] == x[:, 1], 0, best.indices)
    assert ((r.logprob - ref).abs() <= 2.0 ** -17 * (1 + ref.abs())).all()
    entropy = -(lp.exp() * lp).sum(1)
    assert ((r.entropy - entropy).abs() <= 2.0 ** -16 * (1 + entropy)).all()
    assert torch.equal(r.top_tokens[:, 0].long(), first) and torch.equal(r.rank, (t != first).int())
    assert torch.equal(r.top_logprobs[:, 0].isfinite(), torch.ones_like(first, dtype=torch.bool))
    assert torch.equal(torch.where(t == first, r.top_logprobs[:, 0], r.logprob), r.logprob)
