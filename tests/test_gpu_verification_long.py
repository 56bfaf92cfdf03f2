"""verify_drafts over rows of more than 2^20 tokens, whose parts are cut again and again, and over rows that several
blocks share with nothing left in them. Weights are multiples of 2^-12 and numbers have few bits, so that every sum
and product is exact in 64 bits in any order, and borders are hit exactly."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from test_gpu_verification import plan_of
from test_step_plan import _desc


def part_of(vocab):
    """Tokens of a part: a multiple of 1024, at most 1024 parts a row."""
    return -(-vocab // (1 << 20)) * 1024


def places(rs, vocab):
    """Tokens beside the borders of parts, of what parts are cut into, of the row; and others."""
    part = part_of(vocab)
    some = {0, 1, vocab - 1, vocab - 2, vocab // part * part, vocab // part * part - 1}
    for p in [0, part, (vocab // part - 1) * part, vocab // part * part] + (rs.randint(0, vocab // part, 5) * part).tolist():
        size = part
        while size > 1024:
            size = -(-size // 16)
            k = rs.randint(1, 16)
            some |= {p + size * k + d for d in (-1, 0, 1)}
            p += size * rs.randint(0, 16)
        some |= {p - 1, p, p + 1, p + 511, p + 512, p + 1023}
    some |= set(rs.randint(0, vocab, 20).tolist())
    return np.array(sorted(t for t in some if 0 <= t < vocab))


def answer(tokens, weights, draw):
    """The first token whose running sum exceeds the draw's share of the whole."""
    run = np.cumsum(weights)
    return int(tokens[np.argmax(run > float(draw) * run[-1])])


def chains(R, vocab):
    """A plan of R chains of two nodes, over short caches."""
    plan, _ = plan_of(np.full(R, 3), np.full(R, 2), np.arange(R)[:, None], np.zeros(0), 16, 2 * R, 2, R)
    return plan


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("vocab,R", [
    ((1 << 20) - 1, 3), (1 << 20, 2), ((1 << 20) + 1, 9), ((1 << 20) + 1, 140), ((1 << 20) + 1027, 5), (3 * (1 << 20) + 77, 4),
    (20_000_003, 5), (300_000_001, 2), (1 << 30, 1)])
def test_rows_of_many_parts(gpu_device, vocab, R, drafts):
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    if drafts and vocab == 1 << 30:
        R = 1
    rs = np.random.RandomState(vocab % 1000 + R)
    at = places(rs, vocab)
    p = rs.randint(0, 33, (2 * R, at.size)) * 2.0 ** -12
    p[:, rs.randint(0, at.size, 8)] = 0.0
    p[:, -1] = 2.0 ** -12                             # the row's last token always has some
    q = rs.randint(0, 25, (2 * R, at.size)) * 2.0 ** -12
    index = torch.from_numpy(at).cuda()
    probs = torch.zeros(2 * R, vocab, device="cuda")
    probs[:, index] = torch.from_numpy(p).float().cuda()
    models = None
    if drafts:
        models = torch.zeros(2 * R, vocab, device="cuda")
        models[:, index] = torch.from_numpy(q).float().cuda()
    plan = chains(R, vocab)
    pick = rs.randint(0, at.size, R)
    tokens = np.zeros(2 * R, np.int64)
    tokens[1::2] = at[pick]
    for turn in range(6):
        uniforms = (rs.randint(0, 64, 2 * R) / 2048 if not drafts else rs.randint(0, 16, 2 * R) / 8).astype(np.float32)
        draws = (rs.randint(0, 1 << 12, R) * 2.0 ** -12).astype(np.float32)
        draws[:1] = [0.0, 1 - 2.0 ** -24, 0.5, 0.25, 0.75, 2.0 ** -12][turn]
        kept, answers = [], []
        for r in range(R):
            a, u = 2 * r, float(uniforms[2 * r])
            chance = p[a, pick[r]]
            good = chance > 0 and (u * q[a, pick[r]] < chance if drafts else u < chance)
            kept.append(2 if good else 1)
            left = p[a + 1] if good else np.maximum(p[a] - q[a], 0.0) if drafts else np.where(np.arange(at.size) == pick[r], 0.0, p[a])
            answers.append(answer(at, left if left.any() else p[a], draws[r]))
        got = verify_drafts(probs, torch.from_numpy(tokens).cuda(), plan, torch.from_numpy(uniforms).cuda(),
                            torch.from_numpy(draws).cuda(), draft_probs=models)
        assert got.kept.tolist() == kept and got.answers.tolist() == answers
    if R >= 4:
        assert 1 in kept


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [32769, 70001, (1 << 20) + 1, 20_000_003])
def test_nothing_left_of_long_rows(gpu_device, vocab):
    """As in short rows, where several blocks share a row's sums."""
    from kv_cache_repair_amd.kernels.verification import verify_drafts

    plan = chains(5, vocab)
    probs = torch.zeros(10, vocab, device="cuda")
    probs[:, 7], probs[:, vocab - 1] = 0.5, 0.5
    tokens = torch.tensor([0, 7] * 5, device="cuda")
    uniforms, draws = torch.full((10,), 0.75, device="cuda"), torch.full((5,), 0.75, device="cuda")
    models = probs.clone()
    models[2, 7] = 0.75                                   # refused, and nothing above the draft's but at the end
    models[4, 7], models[4, vocab - 1] = 0.75, 0.6        # refused, and nothing left: the target's own
    probs[6] = 0.0                                        # no mass at all
    probs[8, 7] = math.nan                                # an entry that does not count
    models[2, vocab - 1] = 0.25
    got = verify_drafts(probs, tokens, plan, uniforms, draws, draft_probs=models)
    assert got.kept.tolist() == [2, 1, 1, 1, 1] and got.answers.tolist() == [vocab - 1, vocab - 1, vocab - 1, -1, vocab - 1]
    assert got.path.tolist() == [0, 1] + [0, -1] * 4
    draws[2] = 0.25
    assert verify_drafts(probs, tokens, plan, uniforms, draws, draft_probs=models).answers[2].item() == 7
    probs.zero_()
    probs[:, 7] = 1.0
    uniforms.fill_(1.0)                                   # outside [0, 1): the child is not kept though it has all of the mass
    got = verify_drafts(probs, tokens, plan, uniforms, draws)
    assert got.kept.tolist() == [1] * 5 and got.answers.tolist() == [7] * 5


@pytest.mark.parametrize("workspace,short", [(None, 0), ((1 << 20) + 8, 0), (1 << 20, 1), (1 << 20, 16)])
def test_refuses_a_workspace_that_does_not_hold(workspace, short):
    from kv_cache_repair_amd import _native

    lib, at = _native.lib(), 1 << 20
    need = lib.kvr_verify_workspace_bytes(4, 40000)
    assert need > 0 and need % 16 == 0 and lib.kvr_verify_workspace_bytes(4, 32768) == 0
    assert lib.kvr_verify_drafts(at, 40000, None, 0, 40000, at, at, at, ctypes.byref(_desc()), at, at, at, workspace,
                                 need - short, None) == -6
