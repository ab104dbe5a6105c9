"""CPU checks of masked attention's planner (neuralrs_amd/csrc/masked_attention_plan.hpp)."""
import random

import pytest

import masked_plan

pytestmark = pytest.mark.skipif(not masked_plan.built(),
                                reason="masked_plan_query not built (run __graft_entry__.build())")


def test_the_calls_of_the_gpu_tests_reach_every_kernel():
    reached = {k for s, a in zip(masked_plan.SHAPES, masked_plan.ask(masked_plan.SHAPES))
               for k in masked_plan.kernels(s, a)}
    assert reached == masked_plan.EVERY, (masked_plan.EVERY - reached, reached - masked_plan.EVERY)


def test_scratch_stays_a_few_times_the_outputs():
    """Parts of walks: scratch of the forward (and backward) is at most that of two parts of
    128 rows (and keys) for every workgroup at once, beyond two copies of what is written
    and the rows' own numbers."""
    rng = random.Random(1)
    shapes = []
    for _ in range(3000):
        kv, group = rng.choice([1, 2, 8]), rng.choice([1, 1, 4, 7])
        n = int(2 ** rng.uniform(0, 15))
        shapes.append((int(2 ** rng.uniform(0, 6)), kv * group, kv, rng.choice([n, 1, 100]), n,
                       rng.choice([16, 32, 64, 96, 128])))
    for s, a in zip(shapes, masked_plan.ask(shapes)):
        batch, heads, kv, sq, sk, d = s
        forward, backward = map(int, a.split()[4:])
        q, k = 4 * batch * heads * (sq + 256) * (d + 2), 4 * batch * kv * (sk + 128) * d
        most = 4 * 256 * (d + 2) * 4 * masked_plan.CUS
        assert forward <= 3 * q + 2 * most, s
        assert backward <= 3 * q + 6 * k + 4 * most + 64 * (batch * heads * (sq + 64) + batch * kv * (sk + 64)), s
