"""The 64-bit cross attention that the GPU tests compare with: its gradients
against differences of its forward."""
import numpy as np

from attention_ref import backward, forward


def test_gradients_against_differences():
    rng = np.random.default_rng(0)
    q, k, v, g = (rng.standard_normal(s) for s in ((5, 8), (7, 8), (7, 8), (5, 8)))
    grads, _ = backward(q, k, v, g, 0.3)
    h = 1e-6
    for i, x in enumerate((q, k, v)):
        for at in np.ndindex(*x.shape):
            losses = []
            for sign in (1, -1):
                args = [q.copy(), k.copy(), v.copy()]
                args[i][at] += sign * h
                losses.append((forward(*args, 0.3)[0] * g).sum())
            # an f64 difference over 2e-6: about 1e-16 / 1e-6, and h^2
            assert abs((losses[0] - losses[1]) / (2 * h) - grads[i][at]) < 1e-8
