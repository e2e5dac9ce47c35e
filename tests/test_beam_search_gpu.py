"""Beam search of the own model (jdg_beam_search) against the oracle's forward: the same search on
the CPU, every hypothesis replayed from scratch.  It runs the paged append, the attention behind
the shared prompt, the selection and the reordering together, through the engine.

Two hypotheses whose scores are closer than the measured difference of the logits allows may
change places: a score is a sum of log-probabilities, each off by 2 max|d logit| at most (the
logits agree to LOGIT_TOL of their largest), so candidates nearer than 4 steps LOGIT_TOL max|logit|
are not told apart.  The seeds are such that the CPU search alone meets none."""
import os
import subprocess

import numpy as np
import pytest

from _util import LOGIT_TOL
from oracle.oracle import OwnModel

pytestmark = pytest.mark.gpu


def cpu_search(om, prompt, beams, max_new, eos):
    """(hypotheses best first, smallest gap between the last kept and the first dropped candidate or
    between neighbours, largest |logit|)."""
    def logits(seq):
        om.reset()
        for i, t in enumerate(seq):
            lg = om.forward(int(t), i)
        return lg.astype(np.float64)

    live, gap, top = [(0.0, [], False)], np.inf, 0.0
    for _ in range(max_new):
        cand = []
        for b, (s, seq, done) in enumerate(live):
            if done:
                cand.append((s, b, eos, seq + [eos], True))
                continue
            lg = logits(list(prompt) + seq)
            top = max(top, float(np.abs(lg).max()))
            lp = lg - lg.max()
            lp -= np.log(np.exp(lp).sum())
            for t in np.argsort(-lp, kind="stable")[:beams + 1]:
                cand.append((s + lp[t], b, int(t), seq + [int(t)], int(t) == eos))
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for a, b in zip(cand[:beams], cand[1:beams + 1]):
            gap = min(gap, a[0] - b[0])
        live = [(c[0], c[3], c[4]) for c in cand[:beams]]
    out = []
    for s, seq, _ in live:
        out.append((s, seq[:seq.index(eos) + 1] if eos in seq else seq))
    return out, gap, top


def pair(jd, orc, depth, seed, masks, **over):
    om = OwnModel(orc, orc.config(depth, **over), seed, 0.08, masks)
    return om, jd.Model.seeded(jd.config_from_depth(depth, **over), seed, 0.08, masks)


@pytest.mark.parametrize("depth,seed,n,beams,max_new,eos", [
    (2, 1, 1, 2, 6, -1),     # no prefix at all: the prompt is the first own row
    (2, 3, 7, 4, 9, -1),
    (4, 5, 40, 5, 7, -1),
    (4, 5, 12, 1, 6, -1),    # one beam: greedy
    (8, 2, 21, 8, 5, -1),    # grouped heads (8 over 4), more than 16 queries behind the prefix
    (2, 3, 7, 3, 20, "second"),
])
def test_beam_search_matches_the_oracle(jd, orc, gpu_ctx, depth, seed, n, beams, max_new, eos):
    over = dict(vocab_size=700, seq_len=96)
    om, pm = pair(jd, orc, depth, seed, depth > 2, **over)
    prompt = np.random.default_rng(seed).integers(0, 700, n).astype(np.int32)
    eng = jd.Engine.own(gpu_ctx, pm, max(beams, 2))
    try:
        if eos == "second":  # a token that the search without an end picks: some beams finish early
            eos = cpu_search(om, prompt, beams, 3, -1)[0][1][1][1]
        want, gap, top = cpu_search(om, prompt, beams, max_new, eos)
        assert gap > 1e-6  # the seeds meet no tie
        for _ in range(2):  # a second search finds the engine as the first did
            seqs, scores = eng.beam_search(prompt, beams, max_new, eos)
            if gap > 4 * max_new * 1e-5 * top:
                assert seqs == [s for _, s in want]
            for (w, _), s in zip(want, scores):
                assert abs(w - s) <= 2 * max_new * LOGIT_TOL * top
            assert list(scores) == sorted(scores, reverse=True)
        if beams == 1:
            eng.set_prompt(prompt[None], [n])
            eng.run(1, n - 1 + max_new)
            assert [int(t) for t in eng.history(1, max_new)[0]] == seqs[0]
    finally:
        eng.close()
        om.close()


def test_beam_search_scores_are_the_sequences_own(jd, orc, gpu_ctx):
    """Long search, many beams, graphs replayed: each returned score is its sequence's log-probability
    by the oracle, the sequences differ, and decoding afterwards is as before."""
    om, pm = pair(jd, orc, 4, 11, True, vocab_size=500, seq_len=256)
    prompt = np.random.default_rng(2).integers(0, 500, 60).astype(np.int32)
    eng = jd.Engine.own(gpu_ctx, pm, 20)
    try:
        eng.set_prompt(prompt[None], [60])
        eng.run(1, 60 - 1 + 8)
        before = eng.history(1, 8)[0].tolist()
        seqs, scores = eng.beam_search(prompt, 20, 40)
        assert len({tuple(s) for s in seqs}) == 20 and all(len(s) == 40 for s in seqs)
        for b in (0, 7, 19):
            om.reset()
            total, top, full = 0.0, 0.0, list(prompt) + seqs[b]
            for i, t in enumerate(full[:-1]):
                lg = om.forward(int(t), i).astype(np.float64)
                if i + 1 >= len(prompt):
                    top = max(top, float(np.abs(lg).max()))
                    total += lg[full[i + 1]] - lg.max() - np.log(np.exp(lg - lg.max()).sum())
            assert abs(total - scores[b]) <= 2 * 40 * LOGIT_TOL * top * 1e-2, (b, total, scores[b])
        eng.reset()
        eng.set_prompt(prompt[None], [60])
        eng.run(1, 60 - 1 + 8)
        assert eng.history(1, 8)[0].tolist() == before
    finally:
        eng.close()
        om.close()


def test_beam_search_refusals(jd, orc, gpu_ctx):
    om, pm = pair(jd, orc, 2, 1, False, vocab_size=40, seq_len=32)
    eng = jd.Engine.own(gpu_ctx, pm, 4)
    try:
        for args in (([], 2, 4), ([1, 2], 5, 4), ([1, 2], 0, 4), ([1, 2], 2, 0), ([1, 2], 2, 31), ([1, 40], 2, 4),
                     ([1, -1], 2, 4), ([1, 2], 2, 4, 40)):
            with pytest.raises(jd.JdError) as ei:
                eng.beam_search(*args)
            assert ei.value.code == jd.JD_EINVAL
        assert len(eng.beam_search([1, 2], 2, 30)[0][0]) == 30  # to the last position
    finally:
        eng.close()
        om.close()


def test_command_line_beams(jd, gpu_ctx):
    """`m --beams N` prints the best sequence of the same search."""
    cli = os.path.join(os.path.dirname(jd.LIB_PATH), "m")
    r = subprocess.run([cli, "--depth", "2", "--vocab", "700", "--seed", "4", "--ask", "hello there", "--gen", "9",
                        "--beams", "3", "--print-ids"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    got = [ln for ln in r.stdout.splitlines() if ln.startswith("[ids] generated")][0].split()[2:]
    pm = jd.Model.seeded(jd.config_from_depth(2, vocab_size=700), 4, 0.02, False)
    eng = jd.Engine.own(gpu_ctx, pm, 3)
    try:
        best = eng.beam_search(list(b"hello there"), 3, 9, 257)[0][0]
        assert [int(t) for t in got] == [t for t in best if t != 257]
    finally:
        eng.close()
