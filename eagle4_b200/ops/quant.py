"""The 8-bit KV cache: its tensors, formats and the layout of multi-axis rotary positions.

A cache of one attention layer's K (or V) holds, per (slot, kv head), ``head_dim`` 8-bit codes and one fp32 scale;
``code * scale`` is the value a code stands for. A row ``x`` is quantised by itself, as it is written:

    scale = max(max|x| * (1 / QMAX), 2^-60),   code = round(x * (1 / scale))   (to the nearest, ties to even)

``fp8`` codes are float8 e4m3 (QMAX 448: three fraction bits, small elements keep their relative precision), ``int8``
codes are integers (QMAX 127: a uniform step of 1/127 of the row's largest element, about a quarter of e4m3's error on
rows without outliers). A row that holds a NaN or an infinity gets a NaN scale and reads back as NaN. Codes are laid
out ``[slots, kv heads, head dim]`` like the 16-bit cache; scales ``[kv heads, slots]``, so that the scales of one
head's consecutive tokens, which attention reads together, share their sectors.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
SCALE_FLOOR = 2.0 ** -60
KV_DTYPES = {"bf16": None, "fp8": torch.float8_e4m3fn, "int8": torch.int8}  # names of the serving options
MAX_AXES = 4


class QuantKV(NamedTuple):
    """One layer's 8-bit K or V cache: ``data [slots, heads, dim]`` (float8_e4m3fn or int8) and ``scale [heads,
    slots]`` fp32. Takes the place of a 16-bit cache tensor in ``ops.attention``, ``ops.qkv_prepare`` and
    ``ops.kv_commit``."""

    data: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def allocate(cls, slots: int, heads: int, dim: int, code: torch.dtype, device) -> "QuantKV":
        if code not in QMAX:
            raise ValueError(f"8-bit KV caches hold float8_e4m3fn or int8 codes, not {code}")
        if dim % 16 or not 16 <= dim <= 256:
            raise ValueError(f"8-bit KV caches need a head dim that is a multiple of 16 up to 256, got {dim}")
        return cls(torch.zeros(slots, heads, dim, dtype=code, device=device),
                   torch.zeros(heads, slots, dtype=torch.float32, device=device))

    @property
    def shape(self) -> torch.Size:
        return self.data.shape


Cache = Union[torch.Tensor, QuantKV]


def kv_code(kv_dtype: Optional[str]) -> Optional[torch.dtype]:
    """The code type of a serving option (None: the 16-bit cache)."""
    if kv_dtype is None:
        return None
    if kv_dtype not in KV_DTYPES:
        raise ValueError(f"kv_dtype must be one of {sorted(KV_DTYPES)}, got {kv_dtype!r}")
    return KV_DTYPES[kv_dtype]


def new_cache(slots: int, heads: int, dim: int, dtype: torch.dtype, code: Optional[torch.dtype], device) -> Cache:
    """A zeroed K or V cache of one layer: 16-bit (``dtype``), or 8-bit when ``code`` is given."""
    if code is None:
        return torch.zeros(slots, heads, dim, dtype=dtype, device=device)
    return QuantKV.allocate(slots, heads, dim, code, device)


def cache_tensors(caches) -> list:
    """The tensors that a list of caches holds."""
    return [t for c in caches for t in (c if isinstance(c, QuantKV) else (c,))]


def same_form(k_cache: Cache, v_cache: Cache) -> bool:
    """Whether K and V are both 8-bit (True) or both 16-bit (False); a mixed pair is refused."""
    k8 = isinstance(k_cache, QuantKV)
    if k8 != isinstance(v_cache, QuantKV):
        raise TypeError("the K and V caches must both be 16-bit tensors or both QuantKV")
    return k8


def attention_workspace(rows: int, q_heads: int, kv_heads: int, dim: int, max_keys: int, sms: int = 148) -> int:
    """Bytes that ``ops.attention`` over 8-bit caches allocates beside its output while it runs: the partial sums of the
    (row, kv head)s that its blocks' bounds cut, up to one at each bound, and where each block begins."""
    group = q_heads // kv_heads
    blocks = sms * (2 if dim <= 128 and group <= 8 else 1)
    chunks = max(1, -(-max_keys // 128))
    grid = min(rows * kv_heads * chunks, blocks)
    return 4 * (4 * grid + (grid - 1) * min(chunks, -(-blocks // kv_heads)) * group * (dim + 4)) if rows else 0


def rope_layout(cfg, pos: torch.Tensor) -> Tuple[Tuple[int, ...], bool]:
    """How the rows' positions turn the rotary frequencies: ``(sections, interleaved)``.

    ``pos [T]``: one axis turns all of them. ``pos [axes, T]``: ``cfg.rope_sections`` gives each axis a number of
    frequencies: consecutive runs, or with ``cfg.rope_interleaved`` axis ``a > 0`` takes the frequencies ``a``, ``a +
    axes``, ``a + 2 axes``, ... and axis 0 the others."""
    half = cfg.rotary_dim // 2
    if pos.dim() == 1:
        return (half,), False
    if pos.dim() != 2 or not 1 <= pos.shape[0] <= MAX_AXES:
        raise ValueError(f"positions must be [T] or [axes, T] with up to {MAX_AXES} axes, got {tuple(pos.shape)}")
    return _sections(tuple(getattr(cfg, "rope_sections", None) or ()), bool(getattr(cfg, "rope_interleaved", False)),
                     pos.shape[0], half)


@lru_cache(maxsize=64)
def _sections(sections: Tuple[int, ...], interleaved: bool, axes: int, half: int) -> Tuple[Tuple[int, ...], bool]:
    if len(sections) != axes:
        raise ValueError(f"positions of {axes} axes need rope_sections of {axes} entries, got {tuple(sections)}")
    if min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"rope_sections {tuple(sections)} must add up to {half}, half of the rotary dims")
    if interleaved and any(a + axes * (n - 1) >= half for a, n in enumerate(sections) if a and n):
        raise ValueError(f"interleaved rope_sections {tuple(sections)} reach past {half} frequencies")
    return tuple(int(n) for n in sections), interleaved


def rope_axis(half: int, sections: Sequence[int], interleaved: bool) -> torch.Tensor:
    """The axis ``[half]`` (int64) whose position turns each frequency."""
    axes = len(sections)
    if not interleaved or axes == 1:
        return torch.repeat_interleave(torch.arange(axes), torch.tensor(list(sections)))
    j = torch.arange(half)
    a = j % axes
    return torch.where((a > 0) & (j < axes * torch.tensor(list(sections))[a]), a, 0)
