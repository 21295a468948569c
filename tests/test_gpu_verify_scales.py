"""Verification at temperatures next to 0, random numbers outside [0, 1) and large vocabularies, against the rules in 64 bits (test_gpu_verify)."""
import math

import pytest
import torch

from test_gpu_verify import compare, inputs

pytestmark = pytest.mark.gpu


# A weight is 2^(logit log2(e) / T - K).  From |logit| / T = 1e10 or so neighbouring floats are further apart than all that has weight.
@pytest.mark.parametrize("t", [1e-6, 1e-8, 1e-9, 1e-10, 1e-11, 3e-12, 1e-13])
@pytest.mark.parametrize("size", [5.0, 20.0, 30.0, 130.0, 200.0, -5.0, -200.0])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_temperatures_next_to_zero(cuda, t, size, kind):
    """All weight is the largest logit's, whatever its size: it is accepted where it is drafted, and drawn."""
    counts = [5, 9, 1]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, kind, 1500, torch.float32, 31)
    logits = logits - logits.amax(-1, keepdim=True) + size
    logits[1, [7, 1400]] = logits[1].max()            # (two share it)
    for i in (1, 2, 6):
        token[i] = int(logits[i - 1].argmax())
    for draft in (q, None):
        path, count, said = compare(logits, counts, parents, token, draft, [t] * 3, u, u_next, 9, chain=kind == "chain")
        assert int(said[2, 0]) == int(logits[14].argmax())


@pytest.mark.parametrize("vocab", [196000, 256000, 262141, 262144, 262145])
@pytest.mark.parametrize("mode,dtype", [("drawn", torch.float32), ("chosen", torch.bfloat16), ("greedy", torch.float16)])
@pytest.mark.parametrize("kind", ["chain", "tree"])
def test_vocabularies_that_fill_a_cluster(cuda, vocab, mode, dtype, kind):
    """The weights of sixteen blocks' slices fill their shared memory, or just do not fit any more."""
    counts = [4, 7, 1]
    logits, parents, token, q, u, u_next = inputs(cuda, counts, kind, vocab, dtype, 33)
    token[2] = int(logits[1].argmax())
    token[5] = vocab - 1
    logits[4, vocab - 1] = logits[4].max() + 1
    temps = None if mode == "greedy" else [1.0, 0.7, 1.3]
    compare(logits, counts, parents, token, q if mode == "drawn" else None, temps, u, u_next, 7, chain=kind == "chain")


@pytest.mark.parametrize("vocab", [3, 700, 256000])
def test_random_numbers_of_one_and_more(cuda, vocab):
    """They accept no token that has no weight left, and draw like the largest below 1."""
    from poptransformer_b200 import ops
    logits = torch.full((4, vocab), -math.inf, device=cuda)
    p = torch.rand(300, generator=torch.Generator().manual_seed(34)).tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    for k in range(0, 300, 2):
        logits[0, 0], logits[0, 1] = math.log(p[k] + 1e-3), math.log(p[k + 1] + 1e-3)
        said = []
        for u in (1.5, 1.0000002, 1.0):                # (the two tokens are all of p; the third has none)
            _, count, tok, _ = ops.verify_drafts(logits, i32([0, 4]), i32([0, 0, 1, 2]), i32([-1, 0, 0, 0]), max_path=2, temperature=torch.ones(1, device=cuda),
                                                 uniform=torch.full((4,), u, device=cuda), uniform_next=torch.full((1,), u, device=cuda))
            said.append((int(count[0]), int(tok[0, 0])))
        assert all(t in (0, 1) for _, t in said), (k, said)
