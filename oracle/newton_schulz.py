"""CPU oracle of the Newton-Schulz updates -- TEST INFRASTRUCTURE ONLY.

Float64 torch, on the CPU unless given a GPU's matrix.  ``orthogonalise`` follows the definition on singular
values (an SVD, no products); ``by_products`` the iteration, optionally with
every operand and product off by random roundings of given sizes, which says
how far roundings of that size move the result.
"""

import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def polynomial(s, coefficients=COEFFICIENTS, steps=5):
    a, b, c = coefficients
    for _ in range(steps):
        s = s * (a + s * s * (b + s * s * c))
    return s


def orthogonalise(G, coefficients=COEFFICIENTS, steps=5, eps=1e-7):
    X = G.double()
    X = X / (X.square().sum().sqrt() + eps)
    U, S, Vh = torch.linalg.svd(X, full_matrices=False)
    return (U * polynomial(S, coefficients, steps)) @ Vh


def by_products(G, coefficients=COEFFICIENTS, steps=5, eps=1e-7, operand=0.0, product=0.0,
                seed=0):
    """The iteration; operands off by a relative `operand`, products by `product`
    of the sum of their terms' sizes, uniformly at random."""
    gen = torch.Generator(device=G.device).manual_seed(seed)

    def off(x, size, by):
        if size == 0.0:
            return x
        return x + size * by * (2 * torch.rand(x.shape, generator=gen, dtype=torch.float64,
                                               device=G.device) - 1)

    def mm(p, q):
        return off(p @ q, product, p.abs() @ q.abs())

    a, b, c = coefficients
    tall = G.shape[0] > G.shape[1]
    X = G.double().T if tall else G.double()
    X = X / (X.square().sum().sqrt() + eps)
    X = off(X, operand, X.abs())
    for i in range(steps):
        A = mm(X, X.T)
        A = off(A, operand, A.abs())
        B = b * A + c * mm(A, A)
        B = off(B, operand, B.abs())
        X = a * X + mm(B, X)
        if i + 1 < steps:
            X = off(X, operand, X.abs())
    return X.T if tall else X


def muon(W, G, M, lr, mu=0.95, nesterov=True, weight_decay=0.0, scale=None, **ns):
    """(W, M) after a step, float64."""
    M = mu * M.double() + G.double()
    U = G.double() + mu * M if nesterov else M
    s = max(1.0, W.shape[0] / W.shape[1]) ** 0.5 if scale is None else scale
    return (1 - lr * weight_decay) * W.double() - lr * s * orthogonalise(U, **ns), M
