"""The orthogonalised update from its definition in 64 bits (numpy), and how far a computation whose products have relative rounding u may be off.

A perturbation dX of X passes a step as the derivative of p(X) = c0 X + c1 X X'X + c2 X X'X X'X; its gain in the Frobenius norm is at most
g(s) = |c0| + 3 |c1| s^2 + 5 |c2| s^4 (s: the largest singular value), but that bound multiplies up to thousands over five steps although the gains of the actual iteration
are near one.  The bound used here is therefore measured on the case itself: the definition is evaluated in 64 bits with every factor of every product perturbed by random relative
errors of u (the rounding's model: each factor is off by at most u of itself), and four times the largest of six such runs is allowed.

The linear term is no product of rounded factors, and where |X| is tiny it is all there is: X <- c0 X with c0 rounded to 32 bits (2^-24 of it) and the result rounded to 32 bits (2^-24
of it), after a start rounded once.  `steps` such steps are off by at most (1 + 2^-24)^(2 steps + 1) - 1, that is (2 steps + 1) 2^-24 of the result, which is added."""
import numpy as np

C = (3.4445, -4.7750, 2.0315)


def iterate(u, steps, coefficients, scale, rng=None, eps=0.0):
    def r(a):
        return a if rng is None else a * (1 + eps * rng.uniform(-1, 1, a.shape))
    flip = u.shape[0] > u.shape[1]
    x = u.T if flip else u
    x = x / (np.sqrt(np.sum(x * x)) + 1e-7)
    for k in range(steps):
        c = coefficients[k] if np.ndim(coefficients) == 2 else coefficients
        xr = r(x)
        a = r(xr @ xr.T)
        a = (a + a.T) / 2
        b = r(c[1] * a + c[2] * (a @ a))
        x = c[0] * x + b @ r(x)
    return scale * (x.T if flip else x)


def update(grad, momentum=None, beta=0.95, nesterov=True, steps=5, coefficients=C, scale=1.0):
    """(out, new momentum) of one matrix."""
    m = None
    u = np.float64(grad)
    if momentum is not None:
        m = beta * np.float64(momentum) + u
        u = u + beta * m if nesterov else m
    return iterate(u, steps, coefficients, scale), m, u


def allowance(u, eps, steps=5, coefficients=C, scale=1.0):
    """(Frobenius norm, largest element) that factors rounded to eps may move the result by."""
    rng = np.random.default_rng(0)
    base = iterate(u, steps, coefficients, scale)
    d = [iterate(u, steps, coefficients, scale, rng, eps) - base for _ in range(6)]
    line = (2 * steps + 1) * 2.0 ** -24
    return 4 * max(np.linalg.norm(e) for e in d) + line * np.linalg.norm(base), 4 * max(np.abs(e).max() for e in d) + line * np.abs(base).max()
