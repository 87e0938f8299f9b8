"""Shared by the tests of the block operators: the float types, inputs, and how far a result may be off."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {name: torch.finfo(t).eps / 2 for name, t in TYPES.items()}   # a rounding to the type, relative
# the smallest step of the type: what a rounding is off by at most half of where the value is subnormal
TINY = {name: torch.finfo(t).smallest_normal * torch.finfo(t).eps for name, t in TYPES.items()}
U = 2.0 ** -24                                                            # a float32 operation, relative


def tensor(a, kind, device):
    return torch.from_numpy(np.ascontiguousarray(a)).to(TYPES[kind]).to(device)


def numbers(t):
    return t.detach().cpu().double().numpy()


def close(got, want, size, kind, steps):
    """|got - want| within `steps` float32 roundings of `size` (the magnitudes the result is made of) and one rounding
    of the result to its type."""
    got = numbers(got)
    assert got.shape == want.shape
    bound = steps * U * size + HALF_STEP[kind] * (np.abs(want) + steps * U * size) + TINY[kind]
    # a number at or above the type's largest plus half its last step (max * (1 + eps / 4)) rounds to infinity
    slack = steps * U * size
    over = np.abs(want) - slack >= torch.finfo(TYPES[kind]).max * (1 + torch.finfo(TYPES[kind]).eps / 4)
    assert np.array_equal(got[over], np.copysign(np.inf, want[over]))
    got, want, bound = np.where(over, 0, got), np.where(over, 0, want), np.where(over, 0, bound)
    off = np.abs(got - want)
    assert not np.isnan(got).any()
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), (worst, got[worst], want[worst], off[worst], bound[worst])


def row_sum_steps(n):
    """Roundings on the way of one term of a row sum: a lane adds n / 64 terms at most, then six steps across the
    wavefront and at most sixteen across wavefronts."""
    return n / 64 + 24
