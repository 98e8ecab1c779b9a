"""Drafted tokens held against the target's probabilities, against a plain 64-bit form."""
import numpy as np
import pytest
import torch

import plain_q8 as plain
from minfer_b200.kernels import api as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(logits, drafts, cu, draft_logits, accept_u, draw_u, temperature):
    rows = len(draw_u)
    accepted = torch.full((rows,), -7, dtype=torch.int32, device=DEV)
    tokens = torch.full((rows,), -7, dtype=torch.int32, device=DEV)

    def dev(x, dtype):
        return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype).to(DEV)
    K.verify_drafts(logits if torch.is_tensor(logits) else dev(logits, torch.float32), dev(drafts, torch.int32),
                    dev(cu, torch.int32), None if draft_logits is None else
                    (draft_logits if torch.is_tensor(draft_logits) else dev(draft_logits, torch.float32)),
                    dev(accept_u, torch.float32), dev(draw_u, torch.float32), temperature, accepted, tokens)
    return accepted.tolist(), tokens.tolist()


def make(vocab, counts, seed, near=True):
    rng = np.random.RandomState(seed)
    n, rows = sum(counts), len(counts)
    cu = [0] + np.cumsum(counts).tolist()
    logits = (rng.randn(n + rows, vocab) * 2.0).astype(np.float32)
    place = [cu[b] + b + j for b in range(rows) for j in range(counts[b])]
    draft_logits = (logits[place] + 0.7 * rng.randn(n, vocab)).astype(np.float32).reshape(n, vocab)
    noise = rng.gumbel(size=(n, vocab))
    drafts = (draft_logits + noise).argmax(1).astype(np.int32) if n else np.zeros(0, np.int32)
    return logits, drafts, cu, draft_logits, rng.rand(n).astype(np.float32), rng.rand(rows).astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 7, 128, 389, 8192, 8195, 40004])
@pytest.mark.parametrize("counts", [[4], [0], [0, 3, 1, 8, 0], [1] * 70, [25, 0]], ids=str)
@pytest.mark.parametrize("with_logits", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.3])
def test_against_the_plain_form(vocab, counts, with_logits, temperature):
    logits, drafts, cu, dl, u, r = make(vocab, counts, vocab + len(counts))
    got = run(logits, drafts, cu, dl if with_logits else None, u, r, temperature)
    assert got == plain.verify(logits, drafts, cu, dl if with_logits else None, u, r, temperature)


@pytest.mark.parametrize("with_logits", [True, False])
def test_a_vocabulary_of_many_pieces(with_logits):
    logits, drafts, cu, dl, u, r = make(300007, [2, 0, 5], 3)
    got = run(logits, drafts, cu, dl if with_logits else None, u, r, 1.0)
    assert got == plain.verify(logits, drafts, cu, dl if with_logits else None, u, r, 1.0)


@pytest.mark.parametrize("temperature", [2e-6, 1e30])
@pytest.mark.parametrize("with_logits", [True, False])
def test_extreme_temperatures(temperature, with_logits):
    logits, drafts, cu, dl, u, r = make(5000, [3, 3, 0], 3)
    logits[:, 7::3] = -np.inf
    logits[:, 6] = np.finfo(np.float32).min
    got = run(logits, drafts, cu, dl if with_logits else None, u, r, temperature)
    assert got == plain.verify(logits, drafts, cu, dl if with_logits else None, u, r, temperature)


@pytest.mark.parametrize("vocab", [389, 20000])
def test_the_same_distribution_is_always_accepted_and_another_never(vocab):
    logits, drafts, cu, _, u, r = make(vocab, [3, 5], 2)
    place = [0, 1, 2, 4, 5, 6, 7, 8]
    dl = logits[place].copy()
    got, _ = run(logits, drafts, cu, dl, np.minimum(u, 0.999), r, 0.8)
    assert got == [3, 5]
    # a target that rules the drafts out
    for j, x in zip(place, drafts):
        logits[j, x] = -np.inf
    got, tokens = run(logits, drafts, cu, dl, np.zeros_like(u), r, 0.8)
    assert got == [0, 0] and tokens == plain.verify(logits, drafts, cu, dl, np.zeros_like(u), r, 0.8)[1]


def test_ties_go_to_the_lowest_index():
    logits = np.zeros((4, 9000), dtype=np.float32)
    logits[:, [8999, 8500, 40]] = 3.0
    logits[1, 2] = 3.0
    logits[2] = -0.0
    logits[2, 5:] = 0.0
    assert run(logits, [40, 2, 0], [0, 3], None, [0.5] * 3, [0.5], 0.0) == ([3], [40])
    assert run(logits, [40, 40, 0], [0, 3], None, [0.5] * 3, [0.5], 0.0) == ([1], [2])
    assert run(logits, [41, 2, 0], [0, 3], None, [0.5] * 3, [0.5], 0.0) == ([0], [40])


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("what", ["nan", "nothing", "inf"])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_row_that_is_no_distribution(what, at, temperature):
    logits, _, cu, _, u, r = make(8200, [2, 2], 5)
    drafts = np.array([logits[0].argmax(), logits[1].argmax(), logits[3].argmax(), logits[4].argmax()], np.int32)
    u = np.zeros(4, np.float32)
    clean = run(logits, drafts, cu, None, u, r, temperature)
    assert clean[0] == [2, 2]
    if what == "nothing":
        logits[at] = -np.inf
    else:
        logits[at, 8100] = np.nan if what == "nan" else np.inf
    got = run(logits, drafts, cu, None, u, r, temperature)
    if what == "inf" and temperature == 0.0:
        assert got == plain.verify(logits, drafts, cu, None, u, r, temperature)      # the first maximum
    else:
        assert got[0][0] == at and got[1][0] == -1
    assert (got[0][1], got[1][1]) == (clean[0][1], clean[1][1])


def test_drafts_outside_the_vocabulary_and_broken_offsets():
    logits, drafts, cu, dl, u, r = make(389, [3, 2], 5)
    drafts[0], drafts[4] = 389, -1
    for lg in (dl, None):
        for t in (0.0, 1.0):
            got = run(logits, drafts, cu, lg, u, r, t)
            assert got == plain.verify(logits, drafts, cu, lg, u, r, t)
            assert got[0][0] == 0
    got = run(logits, drafts, [0, 6, 5], dl, u, r, 1.0)       # beyond the drafts, then backwards
    assert got == ([0, 0], [-1, -1])


def test_draft_logits_that_are_no_distribution_leave_the_target():
    logits, drafts, cu, dl, u, r = make(500, [2], 5)
    dl[0, 3] = np.nan
    assert run(logits, drafts, cu, dl, u, r, 1.0) == plain.verify(logits, drafts, cu, dl, u, r, 1.0)


@pytest.mark.parametrize("r", [0.0, 0.25, 0.5, 0.99999994])
def test_borders_of_the_running_sum(r):
    """Four equal weights among tokens that are ruled out: sums and borders are exact."""
    logits = np.full((1, 8300), -np.inf, dtype=np.float32)
    for i in (3, 700, 8193, 8299):
        logits[0, i] = 1.5
    want = {0.0: 3, 0.25: 700, 0.5: 8193, 0.99999994: 8299}[r]
    assert run(logits, [], [0, 0], None, [], [r], 0.7) == ([0], [want])


def test_numbers_of_one_and_more_take_the_last_token_that_can_be_drawn():
    logits = np.zeros((1, 300), dtype=np.float32)
    logits[0, 250:] = -np.inf
    assert run(logits, [], [0, 0], None, [], [1.0], 1.0) == ([0], [249])
    assert run(logits, [], [0, 0], None, [], [2.0], 1.0) == ([0], [249])


def test_rows_may_be_strided():
    logits, drafts, cu, dl, u, r = make(777, [2, 4], 3)
    want = run(logits, drafts, cu, dl, u, r, 0.9)
    for pad in (1, 3, 4, 23):
        wide = torch.full((8, 777 + pad), float("nan"), device=DEV)
        wide[:, :777] = torch.tensor(logits).to(DEV)
        wide_d = torch.full((6, 777 + pad), float("nan"), device=DEV)
        wide_d[:, :777] = torch.tensor(dl).to(DEV)
        assert run(wide[:, :777], drafts, cu, wide_d[:, :777], u, r, 0.9) == want
        assert run(wide[:, 1:777], drafts, cu, None, u, r, 0.9) == plain.verify(logits[:, 1:], drafts, cu, None, u, r, 0.9)


def test_frequencies_are_the_targets():
    """Whatever the drafts were drawn from, accepted drafts and drawn tokens together follow the target: the
    first token behind a sequence, over 20,000 sequences, against the target's probabilities (each
    count within 5 standard deviations)."""
    rng = np.random.RandomState(1)
    vocab, n = 6, 20000
    target, draft = rng.randn(vocab).astype(np.float32), rng.randn(vocab).astype(np.float32)
    t = 0.7
    q = plain.softmax(draft, t)
    drafts = rng.choice(vocab, size=n, p=q).astype(np.int32)
    logits = torch.tensor(target).to(DEV).repeat(2 * n, 1)
    dl = torch.tensor(draft).to(DEV).repeat(n, 1)
    acc, tok = run(logits, drafts, np.arange(n + 1), dl, rng.rand(n).astype(np.float32), rng.rand(n).astype(np.float32), t)
    first = np.where(np.array(acc) == 1, drafts, np.array(tok))
    p = plain.softmax(target, t)
    counts = np.bincount(first, minlength=vocab)
    assert (np.abs(counts - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


def test_captured():
    logits, drafts, cu, dl, u, r = make(9001, [4, 2], 9)
    want = run(logits, drafts, cu, dl, u, r, 0.9)
    args = [torch.tensor(x).to(DEV) for x in (logits, drafts, np.array(cu, np.int32), dl, u, r)]
    acc, tok = (torch.zeros(2, dtype=torch.int32, device=DEV) for _ in range(2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.verify_drafts(*args, 0.9, acc, tok)
    for _ in range(2):
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert (acc.tolist(), tok.tolist()) == want
