"""CPU checks of cross attention's planner (neuralrs_amd/csrc/cross_attention_plan.hpp)."""
import pytest

import cross_plan

pytestmark = pytest.mark.skipif(not cross_plan.built(),
                                reason="cross_plan_query not built (run __graft_entry__.build())")


def test_the_calls_of_the_gpu_tests_reach_every_kernel():
    reached = {k for s, a in zip(cross_plan.SHAPES, cross_plan.ask(cross_plan.SHAPES))
               for k in cross_plan.kernels(s, a)}
    assert reached == cross_plan.EVERY
