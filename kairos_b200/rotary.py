"""Rotary positions: which channels turn, how fast, and how the turn is scaled for contexts longer than trained."""
from __future__ import annotations

import ctypes
import math
from decimal import Context, Decimal, localcontext

import torch

from ._lib import RotaryPlan

LAYOUTS = {'half': 0, 'interleaved': 1}
# Frequencies are computed with 40 decimal digits: a step of the kernels is a fraction of 64 bits that far positions multiply, so
# 64-bit floats would leave 2^-56 turns a position in the fast pairs.
_DIGITS = Context(prec=40)
_TWO_PI = Decimal('6.2831853071795864769252867665590057683943388')
_PER_RADIAN = _DIGITS.divide(Decimal(1 << 64), _TWO_PI)         # of a turn in 64 bits


class Rotary:
    """Plan of a rotary embedding for heads of `head_dim` channels, the first `rot_dim` of which turn.

    layout: 'half' pairs channel i with i + rot_dim / 2 (rotate-half), 'interleaved' pairs 2 i with 2 i + 1.
    scaling: None, or a dict with 'type' and
      'linear'  factor: positions divided by it;
      'ntk'     factor: the base grows by factor^(rot / (rot - 2)), which slows the slowest pair by it;
      'llama3'  factor, original_max, low_freq_factor (1), high_freq_factor (4): pairs with fewer than
                low_freq_factor turns within the trained length original_max are slowed by factor, those with more
                than high_freq_factor keep their speed, linear in the number of turns between;
      'yarn'    factor, original_max, beta_fast (32), beta_slow (1), magnitude (0.1 ln factor + 1): the method of
                Peng et al., "YaRN: efficient context window extension of large language models" (2023): a ramp over
                the pair index between the two, and a magnitude on the turned channels.

    `frequencies` holds the radians per position of every pair (float64).  The kernels take them as 64-bit binary fractions of
    a turn, rounded from 40 digits: an angle is off by 2^-65 turns for each position (2^-32 turns at position 2^33)."""

    def __init__(self, head_dim, rot_dim=None, theta=10000.0, layout='half', scaling=None, device='cuda'):
        rot = head_dim if rot_dim is None else rot_dim
        if not 0 < rot <= head_dim or rot % 2:
            raise ValueError(f'rot_dim must be even and between 2 and the head dimension {head_dim}, got {rot}')
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if not 1 < theta < math.inf:
            raise ValueError(f'theta must be above 1, got {theta}')
        self.head_dim, self.rot_dim, self.layout, self.theta = head_dim, rot, layout, float(theta)
        with localcontext(_DIGITS):
            exact, self.magnitude = self._scaled(rot, float(theta), scaling)
            turns = [round(f * _PER_RADIAN) % (1 << 64) for f in exact]
        self.frequencies = torch.tensor([float(f) for f in exact], dtype=torch.float64)
        signed = [t - (1 << 64) if t >= 1 << 63 else t for t in turns]
        self.steps = torch.tensor(signed, dtype=torch.int64, device=device)
        self.index = self.steps.get_device() if self.steps.is_cuda else -1
        self.plan = RotaryPlan(self.steps.data_ptr(), self.magnitude, rot, LAYOUTS[layout])
        self.plan_ptr = ctypes.addressof(self.plan)

    @staticmethod
    def _scaled(rot, theta, scaling):
        def power(base):          # base^(-2 i / rot) for every pair i
            each, powers = (-2 * base.ln() / rot).exp(), [Decimal(1)]
            while len(powers) < rot // 2:
                powers.append(powers[-1] * each)
            return powers

        freq = power(Decimal(theta))
        if scaling is None:
            return freq, 1.0
        opt = dict(scaling)
        kind, factor = opt.pop('type', None), float(opt.pop('factor', 0.0))
        if not 1 <= factor < math.inf:
            raise ValueError(f'rotary scaling needs a factor of at least 1, got {factor}')
        by = Decimal(factor)

        def take(name, default=None):
            value = opt.pop(name, default)
            if value is None:
                raise ValueError(f'rotary scaling {kind!r} needs {name!r}')
            return float(value)

        def blend(keep):          # keep = 1 and above: the pair's own speed, 0 and below: slowed by the factor
            slow = 1 / by
            return [f if k >= 1 else f * slow if k <= 0 else f * (k + (1 - k) * slow) for f, k in zip(freq, keep)]

        magnitude = 1.0
        if kind == 'linear':
            freq = [f / by for f in freq]
        elif kind == 'ntk':
            freq = power(Decimal(theta) * (by.ln() * rot / max(2, rot - 2)).exp())
        elif kind == 'llama3':
            trained, low, high = take('original_max'), take('low_freq_factor', 1.0), take('high_freq_factor', 4.0)
            if not high > low:
                raise ValueError('rotary scaling: high_freq_factor must be above low_freq_factor')
            rate, offset = Decimal(trained) / _TWO_PI / (Decimal(high) - Decimal(low)), Decimal(low) / (Decimal(high) - Decimal(low))
            freq = blend([rate * f - offset for f in freq])
        elif kind == 'yarn':
            trained, fast, slow = take('original_max'), take('beta_fast', 32.0), take('beta_slow', 1.0)
            magnitude = take('magnitude', 0.1 * math.log(factor) + 1)

            def pair_of(turns):       # the pair that makes so many turns within the trained length
                return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot - 1)
            rate = 1 / max(Decimal(hi - lo), Decimal('1e-3'))
            freq = blend([1 - (i - lo) * rate for i in range(rot // 2)])
        else:
            raise ValueError(f"rotary scaling type must be 'linear', 'ntk', 'llama3' or 'yarn', got {kind!r}")
        if opt:
            raise ValueError(f'rotary scaling {kind!r}: unknown options {sorted(opt)}')
        return freq, magnitude
