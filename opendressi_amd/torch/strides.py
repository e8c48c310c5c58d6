"""Which strided tensors share memory, by their addresses alone."""
from __future__ import annotations

import math

import torch

_STEPS = 10000  # of a search, which is then given up: its tensors may share memory


def _solvable(terms, target: int) -> bool:
    """Whether sum a z = target with whole numbers 0 <= z <= u, over the terms
    (a, u); True where that would take too long to say."""
    most_of: dict[int, int] = {}
    for a, u in terms:
        most_of[a] = most_of.get(a, 0) + u
    terms = []
    for a, u in sorted(most_of.items()):
        if terms and a % terms[-1][0] == 0 and a // terms[-1][0] - 1 <= terms[-1][1]:
            b, v = terms.pop()  # which makes every step between two of a
            a, u = b, v + a // b * u
        terms.append((a, u))
    terms.reverse()
    most, divisor = [0], [0]  # of what the last terms make
    for a, u in reversed(terms):
        most.append(most[-1] + a * u)
        divisor.append(math.gcd(divisor[-1], a))
    most.reverse()
    divisor.reverse()
    left = _STEPS

    def search(k: int, rest: int) -> bool:
        nonlocal left
        if rest == 0:
            return True
        if rest < 0 or rest > most[k] or rest % divisor[k]:
            return False
        a, u = terms[k]
        for z in range(min(u, rest // a), max(0, -((most[k + 1] - rest) // a)) - 1, -1):
            left -= 1
            if left < 0 or search(k + 1, rest - a * z):
                return True
        return False

    return search(0, target)


def apart(t: torch.Tensor) -> bool:
    """Whether no two of t's elements share memory (and it is soon said)."""
    dims = sorted((s, n - 1) for s, n in zip(t.stride(), t.shape) if n != 1)
    end = 1
    for s, u in dims:
        if s < end:
            break
        end += s * u  # past all that the dimensions up to here span
    else:
        return True
    # two elements at a distance of sum s d = 0, d >= 1 in one dimension and |d| <= u in the others
    for i, (s, u) in enumerate(dims):
        others = dims[:i] + dims[i + 1:]
        if s == 0 or _solvable([(s, u - 1)] + [(a, 2 * v) for a, v in others],
                               sum(a * v for a, v in others) - s):
            return t.numel() == 0
    return True


class _Bytes:
    """Where a tensor's elements lie: `size` bytes from start + sum a z, 0 <= z <=
    u, on, over the terms (a, u). `dense`: they fill what they span."""

    def __init__(self, t: torch.Tensor, dense: bool):
        self.start, self.size, self.dense = t.data_ptr(), t.element_size(), dense
        layout = [(1, t.numel())] if dense else zip(t.stride(), t.shape)
        self.terms = [(self.size * s, n - 1) for s, n in layout if s > 0 and n > 1]
        self.end = self.start + self.size + sum(a * u for a, u in self.terms)

    def meets(self, other: _Bytes) -> bool:
        apart = other.start - self.start
        step = math.gcd(self.size, other.size, apart)  # all addresses' but for one
        within = [(step, b.size // step - 1) for b in (self, other) if b.size > step]
        return _solvable(self.terms + other.terms + within, apart + other.end - other.start - step)


def _interleaved(group: list[_Bytes]) -> bool:
    """Whether they lie apart as columns of one table do: modulo its rows' length."""
    period = math.gcd(*(max(b.terms)[0] for b in group if not b.dense and b.terms))
    if period == 0:
        return False
    parts = sorted((b.start % period, b.size + sum(a * u for a, u in b.terms if a % period))
                   for b in group)
    ends = [at + length for at, length in parts]
    starts = [at for at, _ in parts[1:]] + [parts[0][0] + period]
    return all(end <= start for end, start in zip(ends, starts))


def shared(tensors, dense) -> bool:
    """Whether two of the tensors share memory (or it takes too long to say);
    `dense` says of each whether its elements fill what it spans."""
    spans = sorted((_Bytes(t, d) for t, d in zip(tensors, dense) if t.numel()),
                   key=lambda b: b.start)
    groups, end = [], 0  # of spans that touch
    for b in spans:
        if b.start >= end:
            groups.append([])
        groups[-1].append(b)
        end = max(end, b.end)
    for group in groups:
        if len(group) == 1 or (not all(b.dense for b in group) and _interleaved(group)):
            continue
        for i, a in enumerate(group):
            for b in group[i + 1:]:
                if b.start >= a.end:
                    break
                if a.meets(b):
                    return True
    return False
