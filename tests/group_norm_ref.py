"""Group norm from its definition in 64 bits, with a bound that goes by how far a group's values lie
from each other and not by how far they lie from zero."""
import numpy as np

from tests import mx4_ref as ref

U = 2.0 ** -24      # half a step of 32 bits relative to the value


def norm(x, n_groups, gamma, beta, eps, act, steps):
    """(results, bound before the result's own rounding) of x [N, pixels, C] (64 bits). `steps`: the
    roundings that a value passes through on its way into its group's sums."""
    n, pixels, C = x.shape
    g = x.reshape(n, pixels, n_groups, C // n_groups)
    # (about a value of the group: the mean of equal values is that value, to the last bit)
    rel = g - g[:, :1, :, :1]
    mean = rel.mean((1, 3), keepdims=True)
    d = rel - mean
    rstd = 1 / np.sqrt((d * d).mean((1, 3), keepdims=True) + eps)
    gamma = np.ones(C) if gamma is None else gamma.astype(np.float64)
    beta = np.zeros(C) if beta is None else beta.astype(np.float64)
    y = (d * rstd).reshape(x.shape) * gamma + beta
    # sums of what values are apart, each off by `steps` roundings of the largest of them; the
    # squares of these likewise, and half of that in the root; then the difference from the mean,
    # the root, its product with gamma, the shift and the sum
    off = steps * U * np.abs(rel).max((1, 3), keepdims=True)
    err = (off * rstd + np.abs(d) * rstd * (steps * U + (off * rstd) ** 2 + 4 * U)).reshape(x.shape)
    err = err * np.abs(gamma) + 2 * U * (np.abs(beta) + np.abs(y))
    return ref.activate(y, act), ref.act_error(y, err, act)
