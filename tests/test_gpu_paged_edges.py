"""The operators over a paged cache where they are easily wrong: logits so large
that nothing else counts, a key that outweighs all others, far positions, single
tiles, tables and batches that do not fit, lanes that part ways before an
instruction that wants them together."""
import math

import numpy as np
import pytest
import torch

import paged_ref
from test_gpu_paged import Setup, cuda_lib_status, ints

pytestmark = pytest.mark.gpu


# ---- verify -------------------------------------------------------------------------------------------------------

LARGEST = torch.finfo(torch.float32).max
# (largest logit, temperature): where it is +inf; where its neighbours in fp32 lie further
# apart than a weight reaches, or about as far; where nothing below it is finite
TOPS = [(math.inf, 1.0), (math.inf, 1e-6), (math.inf, 1e6), (LARGEST, 1.0), (3e9, 1.0), (2e10, 1.0), (2.2e9, 1.0), (2.2e6, 1e-3),
        (2.2e4, 1e-5), (1500.0, 1e-6), (1060.0, 1e-6), (1.7e7, 1e-3), (-1500.0, 1e-6), (-LARGEST, 1.0)]


@pytest.mark.parametrize("top,temperature", TOPS)
@pytest.mark.parametrize("V", [5, 3001, 40000])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_rows_whose_largest_logits_have_it_all(cuda_lib, top, temperature, V, probs):
    """One or two ids share a row, and the draft is one of them, or is not: what is
    kept and what is drawn are what p = 1, or 1/2 each, gives."""
    from odiengine_b200 import paged

    rng = np.random.default_rng(V)
    B = 8
    logits = (3 * rng.standard_normal((2 * B, V))).astype(np.float32)
    if top < 0:
        logits = np.full_like(logits, -np.inf) if top == -LARGEST else logits + np.float32(2 * top)
    tokens, ua = np.zeros(2 * B, np.int32), np.zeros(2 * B, np.float32)
    for b in range(B):
        ids = rng.choice(V, 3, replace=False)
        logits[2 * b:2 * b + 2, ids[:1 + b % 2]] = top
        tokens[2 * b + 1] = ids[2] if b == 6 else ids[b % 2]
        ua[2 * b] = (0.9, 0.3, 0.999, 0.7)[b % 4]
    un = rng.random(B).astype(np.float32)
    q = torch.softmax(torch.from_numpy(rng.standard_normal((2 * B, V)).astype(np.float32)), -1) if probs else None
    starts = list(range(0, 2 * B + 1, 2))
    got = paged.verify_sampled(torch.from_numpy(logits).cuda(), ints(tokens.tolist()), ints(starts), torch.from_numpy(ua).cuda(),
                               torch.from_numpy(un).cuda(), temperature=temperature, draft_probs=None if q is None else q.cuda(),
                               scratch=paged.verify_scratch(2 * B, B, V))
    want = paged_ref.verify(logits, tokens.tolist(), starts, ua.tolist(), un.tolist(), temperature, None if q is None else q.numpy())
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1], (got, want)
    assert want[0][0] == want[0][2] == 1 and want[0][6] == 0  # p = 1 is kept, p = 0 is not
