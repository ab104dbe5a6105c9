"""NaN and infinities in a key that some rows of a call see and others do not, in the
kernels of many rows: workgroups of 256 rows, and walks in parts whose sums are joined.
Rows that do not see it keep their bits."""
import math

import pytest
import torch

import masked_plan
from test_gpu_masked_plans import Call

pytestmark = pytest.mark.gpu

SHAPES = [(8, 16, 16, 1500, 1500), (32, 32, 32, 700, 1000), (1, 1, 1, 2500, 2500),
          (1, 4, 4, 12000, 12000)]
KERNELS = ["tiles256 {} alone", "tiles256 {} alone", "tiles128 {} shared", "tiles256 {} shared"]
CASES = [(0, 64), (0, 96), (0, 70), (0, 128), (1, 32), (1, 24)] + [
    (no, d) for no in (2, 3) for d in (32, 24, 64, 96, 70, 128)]


@pytest.mark.parametrize("mode", ["plain", "cap"])
@pytest.mark.parametrize("no,d", CASES)
def test_rows_that_do_not_see_it(hip, no, d, mode):
    shape = (*SHAPES[no], d)
    if masked_plan.built():
        width = {24: "32 part", 70: "96 part"}.get(d, f"{d} whole")
        assert KERNELS[no].format(width) in masked_plan.kernels(shape, masked_plan.ask([shape])[0])
    call = Call(hip, shape, mode)
    see = call.visible(0)
    at = shape[4] // 2 - 3
    sees = see[:, at]
    assert bool(sees.any()) and not bool(sees.all())
    touched = see[sees].any(dim=0)  # keys that a row with a bad result sees

    def run():
        call.run(True)
        return [x.clone() for x in (call.out, call.dq, call.dk, call.dv)]

    clean = run()
    n = {"q": shape[3], "k": shape[4]}
    for which, column, bad in (("k", d // 3, math.nan), ("v", d - 1, math.nan), ("k", 0, math.inf),
                               ("v", d // 2, -math.inf)):
        print(f"masked attention {shape} {mode}: {which} is {bad}", flush=True)
        x = getattr(call, which)
        was = x[at, column].clone()
        x[at, column] = bad
        got = run()
        x[at, column] = was
        for i, side in enumerate(("q", "q", "k", "k")):
            other = torch.ones_like(got[i], dtype=torch.bool)
            other[:n[side], :d] = ~(sees if side == "q" else touched)[:, None]
            assert torch.equal(got[i][other], clean[i][other]), (which, bad, i)
        if which == "v" or math.isnan(bad):
            lost = ~torch.isfinite(got[0][:n["q"], :d]).all(dim=1)
            assert torch.equal(lost, sees), (which, bad)
