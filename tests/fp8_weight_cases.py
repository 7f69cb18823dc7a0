"""Weights whose values lie at the ties between two e4m3 values and next to them, and what they have to become (exact fractions)."""
from fractions import Fraction

import torch

GRID = [float(torch.tensor(i, dtype=torch.uint8).view(torch.float8_e4m3fn)) for i in range(127)]          # 0 to 448


def nearest(x: Fraction) -> float:
    low = max(i for i in range(127) if Fraction(GRID[i]) <= abs(x))
    if low == 126:
        return GRID[126] if x >= 0 else -GRID[126]
    to_low, to_high = abs(x) - Fraction(GRID[low]), Fraction(GRID[low + 1]) - abs(x)
    at = low if to_low < to_high or (to_low == to_high and low % 2 == 0) else low + 1
    return GRID[at] if x >= 0 else -GRID[at]


def nearest_float(x: Fraction) -> float:
    """x > 0 -> the nearest float32 (never a tie here)."""
    guess = torch.tensor(float(x), dtype=torch.float64).float()
    near = [(guess.view(torch.int32) + d).view(torch.float32).item() for d in (-1, 0, 1)]
    return min(near, key=lambda v: abs(Fraction(v) - x))


def weight_at_ties(largest: float) -> torch.Tensor:
    """[128, 128] float32 with that largest magnitude: the ties times the scale, with up to two units in the last place more and less, of both signs."""
    scale = nearest_float(Fraction(largest) / 448)
    ties = torch.tensor([(a + b) / 2 * scale for a, b in zip(GRID[:-1], GRID[1:])], dtype=torch.float64).float()
    rows = []
    for d in (-2, -1, 0, 1, 2):
        v = (ties.view(torch.int32) + d).view(torch.float32)
        rows += [torch.cat([v, torch.zeros(2)]), torch.cat([-v, torch.zeros(2)])]
    w = torch.zeros(128, 128)
    w[:len(rows)] = torch.stack(rows).clamp(-largest, largest)
    w[127, 5] = -largest
    return w


def expected(w: torch.Tensor):
    """(values float32 [128, 128], scale) of one block."""
    scale = nearest_float(max(Fraction(w.abs().max().item()), Fraction(2) ** -100) / 448)
    done = {}
    for v in w.flatten().tolist():
        if v not in done:
            done[v] = nearest(Fraction(v) / Fraction(scale))
    return torch.tensor([done[v] for v in w.flatten().tolist()]).view(w.shape), scale


LARGEST = [448.0, 1.0, 3.0, 0.7, 1e-20, 1e20, 0.1234567, 5.4321, 2.0 ** -120, 3.0e38]
