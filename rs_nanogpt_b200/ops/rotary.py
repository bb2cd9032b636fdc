"""Rotary positions (kernel: ``csrc/kernels/rotary.cu``).

``rotate`` turns the first ``rot`` elements of every head by the angles of its
row's position, ``rotate_bwd`` is its gradient (the transposed turn). Pair i of
a head is ``(x[i], x[i + rot/2])`` in the ``"half"`` layout and
``(x[2i], x[2i+1])`` in the ``"interleaved"`` one; both turn as the model does
(rs-nanogpt src/model/rope.rs:48-72): ``y1 = x1 cos + x2 sin``,
``y2 = x2 cos - x1 sin``.

``tables`` makes the cos and sin of every position once, in 64 bits, with the
usual rules for contexts longer than the trained one.
"""
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._ext import ext

LAYOUTS = ("half", "interleaved")


@dataclass(frozen=True)
class Scaling:
    """How frequencies change for contexts ``factor`` times the trained one.

    * ``"linear"``  every angle divided by ``factor``
    * ``"ntk"``     the base raised, so that the slowest pair turns ``factor``
      times slower and the fastest keeps its frequency
    * ``"parts"``   pairs that turn more than ``high`` times over
      ``original_len`` positions keep their frequency, those that turn less than
      ``low`` times are slowed down by ``factor``, those between are blended;
      cos and sin are multiplied by ``sharpening = 0.1 ln(factor) + 1``, which
      sharpens the softmax as the context grows. A model that divides q and k
      by their norm after the turn divides the factor away, too: it takes tables
      with ``sharpen=False`` and multiplies the attention's scale by
      ``sharpening ** 2``
    """
    kind: str
    factor: float
    original_len: int = 2048
    low: float = 1.0
    high: float = 32.0

    def __post_init__(self):
        if self.kind not in ("linear", "ntk", "parts"):
            raise ValueError(f"unknown rotary scaling {self.kind!r}: linear, ntk or parts")
        if not self.factor >= 1.0:
            raise ValueError(f"rotary scaling factor must be at least 1, got {self.factor}")
        if self.kind == "parts" and not (self.original_len > 0 and self.low < self.high):
            raise ValueError("rotary scaling by parts needs original_len > 0 and low < high")

    @property
    def sharpening(self) -> float:
        return 0.1 * math.log(self.factor) + 1.0 if self.kind == "parts" else 1.0


def tables(rot: int, positions: int, base: float = 10000.0, scaling: Optional[Scaling] = None,
           device="cuda", sharpen: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, fp32 ``(positions, rot / 2)``, multiplied by the scaling's
    ``sharpening`` unless ``sharpen`` is false. Angles are formed in 64 bits:
    in 32 bits the angle of position 100000 is off by up to 0.004 radians."""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rotary: rot must be even and positive, got {rot}")
    if positions <= 0:
        raise ValueError(f"rotary: positions must be positive, got {positions}")
    mul = scaling.sharpening if scaling is not None and sharpen else 1.0
    if scaling is not None and scaling.kind == "ntk":
        if rot == 2:
            raise ValueError("rotary: ntk scaling needs more than one pair")
        base = base * scaling.factor ** (rot / (rot - 2))
    w = torch.pow(base, -torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    if scaling is not None and scaling.kind == "linear":
        w = w / scaling.factor
    elif scaling is not None and scaling.kind == "parts":
        turns = scaling.original_len * w / (2 * math.pi)
        keep = ((turns - scaling.low) / (scaling.high - scaling.low)).clamp_(0, 1)
        w = w * (keep + (1 - keep) / scaling.factor)
    angle = torch.outer(torch.arange(positions, device=device, dtype=torch.float64), w)
    return (angle.cos() * mul).float(), (angle.sin() * mul).float()


def interleaved(layout: str) -> bool:
    if layout not in LAYOUTS:
        raise ValueError(f"unknown rotary layout {layout!r}: half or interleaved")
    return layout == "interleaved"


def _rotate(q, k, pos, cos, sin, layout, q_out, k_out, back):
    if q_out is None:
        q_out = torch.empty_like(q)
    if k is not None and k_out is None:
        k_out = torch.empty_like(k)
    ext().rotate(q, k, pos, cos, sin, interleaved(layout), back, q_out, k_out)
    return q_out, k_out


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
           layout: str = "half", q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """``q`` (rows, heads, head_dim) and ``k`` (rows, kv heads, head_dim; None
    allowed), bf16, fp16 or fp32, rows and heads at any stride; ``pos`` (rows)
    int32. Elements past ``rot = 2 cos.shape[1]`` pass through. The outputs may
    be the inputs. A row whose position is outside the tables is left as it was
    and reported by ``kernel_status``. Returns (q_out, k_out)."""
    return _rotate(q, k, pos, cos, sin, layout, q_out, k_out, False)


def rotate_bwd(dq: torch.Tensor, dk: Optional[torch.Tensor], pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               layout: str = "half", dq_out: Optional[torch.Tensor] = None, dk_out: Optional[torch.Tensor] = None):
    """Gradients of ``rotate``'s inputs from those of its outputs."""
    return _rotate(dq, dk, pos, cos, sin, layout, dq_out, dk_out, True)
