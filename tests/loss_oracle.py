"""Softmax cross entropy and its gradient in 64 bits."""
import numpy as np


def scores(x, w):
    return x @ w.T


def cross_entropy(x, w, targets):
    """(losses, lse), zeros for tokens that do not count."""
    losses, lse = np.zeros(len(x)), np.zeros(len(x))
    some = (targets >= 0) & (targets < len(w))
    z = scores(x[some], w)
    most = z.max(1) if len(z) else np.zeros(0)
    lse[some] = most + np.log(np.exp(z - most[:, None]).sum(1))
    losses[some] = lse[some] - z[np.arange(len(z)), targets[some]]
    return losses, lse


def log_sums(x, w):
    """lse of every token, whatever its target."""
    z = scores(x, w)
    most = z.max(1)
    return most + np.log(np.exp(z - most[:, None]).sum(1))


def gradient(x, w, targets, dlosses):
    """(dX, dW, the probabilities that made them and the rows that count)."""
    some = (targets >= 0) & (targets < len(w))
    z = scores(x[some], w)
    p = np.exp(z - z.max(1, keepdims=True)) if len(z) else z
    p = p / p.sum(1, keepdims=True) if len(z) else p
    p[np.arange(len(z)), targets[some]] -= 1
    p *= dlosses[some][:, None]
    dx = np.zeros_like(x)
    dx[some] = p @ w
    return dx, p.T @ x[some], p, some
