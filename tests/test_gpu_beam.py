"""beam_select against a plain implementation in 64 bits.

Tolerance of the scores: a score is a sum of three float32 terms, each rounded
once, and the log of a float32 sum; with |terms| below 2^5 and sums of at most a
few hundred terms per thread that is under 2^-24 * 2^5 * 16 = 3.1e-5."""
import numpy as np
import pytest
import torch

from quipsharp_b200.beam import beam_select

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 3.1e-5


def plain(logits, scores, n, finished=None, pad=0):
    """Definition on the host: per beam a stable order by logit, then a stable merge by float64 score."""
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    s0 = scores.double().cpu().numpy()
    s0 = np.where(np.isnan(s0), -np.inf, s0)
    B, K, V = x.shape
    out = []
    for b in range(B):
        cand = []
        for k in range(K):
            order = np.argsort(-x[b, k], kind="stable")[:n]
            top = x[b, k].max()
            if finished is not None and bool(finished[b, k]):
                cand += [(s0[b, k] if r == 0 else -np.inf, k, pad) for r in range(n)]
                continue
            with np.errstate(invalid="ignore", divide="ignore"):
                d = np.where(x[b, k] == top, 0.0, x[b, k] - top)
                logp = d - np.log(np.exp(d).sum()) if top != -np.inf else np.full(V, -np.inf)
            cand += [(s0[b, k] + logp[t], k, int(t)) for t in order]
        order = sorted(range(len(cand)), key=lambda i: -cand[i][0])[:n]
        out.append([cand[i] for i in order])
    return (np.array([[c[0] for c in r] for r in out]), np.array([[c[1] for c in r] for r in out]),
            np.array([[c[2] for c in r] for r in out]))


def check(logits, scores, n, finished=None, pad=0):
    got = beam_select(logits, scores, n, finished, pad)
    ws, wp, wt = plain(logits, scores, n, finished, pad)
    s = got[0].double().cpu().numpy()
    assert np.array_equal(np.isneginf(s), np.isneginf(ws))
    fin = np.isfinite(ws)
    scale = np.maximum(1.0, np.abs(ws[fin]) / 32)
    assert (np.abs(s[fin] - ws[fin]) <= TOL * scale).all()
    assert np.array_equal(got[1].cpu().numpy(), wp) and np.array_equal(got[2].cpu().numpy(), wt)


def spread(B, K, V, dtype, seed):
    """Logits whose best candidates are further apart than the rounding of their scores."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K, V, generator=g) * 2
    hot = torch.rand(B, K, V, generator=g).argsort(-1)[..., :min(V, 40)]
    x.scatter_(2, hot, torch.rand(hot.shape, generator=g) * 12 + 4)
    scores = -torch.rand(B, K, generator=g) * 8
    return x.to(dtype).to(DEV), scores.to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [
    (1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 33, 5), (1, 4, 32000, 4), (3, 5, 8191, 10), (2, 8, 50001, 16), (1, 64, 300, 64),
    (5, 1, 4099, 1), (40, 2, 2049, 3), (1, 2, 128003, 64)])
def test_select(B, K, V, n, dtype):
    x, s = spread(B, K, V, dtype, B + V)
    check(x, s, n)


@pytest.mark.parametrize("B,K,V,n", [
    (1, 64, 40000, 64), (2, 9, 30000, 16), (8, 6, 30004, 16), (2, 8, 60000, 17), (1, 1, 128000, 33), (4, 16, 9000, 3)])
def test_lists_of_every_shape(B, K, V, n):
    """Fewer and more chunks than n, beams merged some at a time, more beams than half the warps."""
    check(*spread(B, K, V, torch.float16, 3), n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_token_and_beam(dtype):
    x = torch.zeros(2, 3, 5000, device=DEV, dtype=dtype)  # every logit equal, in every chunk
    s = torch.zeros(2, 3, device=DEV)
    check(x, s, 8)
    x[0, 1, 4000:] = 1
    x[1, :, ::7] = 2
    check(x, s, 8)
    check(torch.full((1, 2, 70000), -0.0, device=DEV, dtype=dtype).index_fill_(2, torch.tensor([5], device=DEV), 0.0),
          s[:1, :2], 6)  # -0 and 0 are equal


def test_masked_vocabularies():
    inf = float("inf")
    x, s = spread(3, 4, 9001, torch.float16, 1)
    x[0, :, 5:] = -inf          # fewer visible tokens than continuations
    x[1, 2] = -inf              # a beam with none
    x[2, 0, 17] = x[2, 0, 8000] = inf
    x[2, 1, ::3] = float("nan")
    x[2, 3] = torch.finfo(torch.float16).min
    check(x, s, 12)
    s[1] = -inf                 # a search with no live beam
    s[0, 0] = float("nan")
    check(x, s, 12)


@pytest.mark.parametrize("n", [1, 4, 9])
def test_finished_beams(n):
    x, s = spread(4, 4, 3000, torch.bfloat16, 2)
    fin = torch.tensor([[1, 0, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [0, 1, 1, 0]], dtype=torch.bool, device=DEV)
    check(x, s, n, fin, pad=77)


def test_large_scores_do_not_lose_the_order_of_logits():
    """At a score of -4000 neighbouring logits round to one score: they rank by logit all the same."""
    x, _ = spread(1, 2, 20000, torch.float32, 3)
    s = torch.tensor([[-4000.0, -4100.0]], device=DEV)
    got = beam_select(x, s, 16)
    order = torch.sort(x[0, 0], descending=True, stable=True)[1][:16]
    assert got[1].unique().tolist() == [0] and torch.equal(got[2][0].long(), order)


def test_many_large_logits_in_few_threads_places():
    """More candidates above the bound than a chunk keeps: the rounds take over."""
    x = torch.randn(1, 1, 16384, device=DEV)
    base = torch.arange(16384, device=DEV)
    x[0, 0, (base // 4) % 256 < 8] += 100.0  # the places of eight threads' pieces
    s = torch.zeros(1, 1, device=DEV)
    got = beam_select(x, s, 64)
    assert torch.equal(got[2][0].long(), torch.sort(x[0, 0], descending=True, stable=True)[1][:64])


def test_strided_and_unaligned_logits():
    x, s = spread(3, 4, 4001, torch.float16, 5)
    wide = torch.full((3, 4, 4100), 60000.0, device=DEV, dtype=torch.float16)  # what surrounds a row must not enter
    for off in (0, 1, 3, 8):
        view = wide[:, :, off:off + 4001]
        view.copy_(x)
        check(view, s, 6)
        wide.fill_(60000.0)
    check(x.transpose(1, 2).contiguous().transpose(1, 2), s, 6)
    check(x[1:2].expand(3, -1, -1), s, 6)


def test_empty_batch_and_other_stream():
    out = beam_select(torch.zeros(0, 3, 50, device=DEV), torch.zeros(0, 3, device=DEV))
    assert [t.shape for t in out] == [(0, 3)] * 3
    x, s = spread(2, 4, 32000, torch.float32, 6)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = beam_select(x, s, 4)
    side.synchronize()
    for a, b in zip(got, beam_select(x, s, 4)):
        assert torch.equal(a, b)


def test_refusals():
    x, s = torch.zeros(2, 3, 50, device=DEV), torch.zeros(2, 3, device=DEV)
    for error, call in (
            (ValueError, lambda: beam_select(x, s, 51)), (ValueError, lambda: beam_select(x, s, 0)),
            (ValueError, lambda: beam_select(x[0], s)), (ValueError, lambda: beam_select(x, s[:1])),
            (TypeError, lambda: beam_select(x.double(), s)), (TypeError, lambda: beam_select(x, s.half())),
            (TypeError, lambda: beam_select(x, s, finished=s)), (RuntimeError, lambda: beam_select(x, s.cpu())),
            (NotImplementedError, lambda: beam_select(torch.zeros(1, 65, 50, device=DEV), torch.zeros(1, 65, device=DEV), 4)),
            (RuntimeError, lambda: beam_select(x.clone().requires_grad_(), s))):
        with pytest.raises(error):
            call()
