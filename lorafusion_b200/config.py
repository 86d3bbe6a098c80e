"""Routing contract shared by the scheduler and the fused multi-adapter LoRA op.

Same public names, fields and error behaviour as lorafusion's
``lorafusion/ops/config.py`` (AdapterSpec ``:14-26``, TileRoute ``:29-39``,
TileRoutingConfig ``:42-69``), so objects built by either package can be
passed to either package's op.  The op in :mod:`lorafusion_b200.b200_ops`
only relies on the duck-typed attributes (``routes``, ``row_start``,
``row_end``, ``adapter_id``, ``scaling``, ``validate``), which means the
reference's own dataclasses work unchanged as inputs.
"""

from __future__ import annotations

from collections.abc import Mapping
from dataclasses import dataclass, field


@dataclass(frozen=True)
class AdapterSpec:
    """One LoRA adapter: its rank, its alpha and the projection it patches.

    ``scaling`` is ``alpha / rank`` (lorafusion/ops/config.py:24-26).
    """

    adapter_id: int
    rank: int
    alpha: float
    in_features: int
    out_features: int

    @property
    def scaling(self) -> float:
        return self.alpha / self.rank


@dataclass(frozen=True)
class TileRoute:
    """A half-open range ``[row_start, row_end)`` of fused rows owned by one adapter."""

    row_start: int
    row_end: int
    adapter_id: int

    @property
    def num_rows(self) -> int:
        return self.row_end - self.row_start


@dataclass(frozen=True)
class TileRoutingConfig:
    """The routing plan of one fused batch: ordered, contiguous adapter row ranges.

    ``tile_size`` is the packer's bin capacity.  ``num_tiles`` counts
    ``ceil(rows / tile_size)`` per route, which is not the bin count
    (lorafusion/ops/config.py:49-53).
    """

    tile_size: int
    routes: list[TileRoute] = field(default_factory=list)

    def num_tiles(self) -> int:
        ts = self.tile_size
        return sum(-(-r.num_rows // ts) for r in self.routes)

    def validate(self, total_rows: int) -> None:
        """Raise ``ValueError`` unless the routes tile ``[0, total_rows)`` in order.

        Mirrors lorafusion/ops/config.py:55-69: the first route whose start is
        not the previous end reports a gap/overlap; otherwise a mismatch in
        covered rows reports under- or over-coverage.
        """
        expected_start = 0
        covered = 0
        for r in self.routes:
            if r.row_start != expected_start:
                raise ValueError(
                    f"Routing gap/overlap at row {r.row_start}, expected {expected_start}"
                )
            covered += r.row_end - r.row_start
            expected_start = r.row_end
        if covered != total_rows:
            raise ValueError(f"Routing covers {covered} rows, expected {total_rows}")


@dataclass(frozen=True)
class AdapterDropout:
    """Dropout in front of the adapters of one fused call (no counterpart in the reference).

    ``rates``: one rate for all adapters, or a mapping adapter id -> rate that names every adapter of the call;
    ``0 <= rate < 1``, taken to the nearest multiple of 1/65536 (and then below 1; float16 calls take rates up to
    63/64).  ``seed`` and ``offset``, ``0 .. 2**64 - 1``, choose the mask: element ``(t, k)`` of ``x`` is dropped by a
    number that depends on seed, offset, ``t`` and ``k`` alone (Philox 4x32-10), so the forward and the backward that
    get the same object agree on it and nothing of it is stored.  ``t`` is the row's number in the call.  Take another
    offset for every step and every projection whose mask should be its own (:meth:`at`), and on every GPU that has
    rows of the batch (``sharding.local_dropout``).
    """

    rates: float | Mapping[int, float]
    seed: int
    offset: int = 0

    def __post_init__(self) -> None:
        for name in ("seed", "offset"):
            v = getattr(self, name)
            if isinstance(v, bool) or not isinstance(v, int) or not 0 <= v < 1 << 64:
                raise ValueError(f"{name} must be a whole number 0 .. 2**64 - 1, got {v!r}")
        many = isinstance(self.rates, Mapping)
        thresholds = {a: self._threshold(r) for a, r in self.rates.items()} if many else self._threshold(self.rates)
        object.__setattr__(self, "_thresholds", thresholds)  # the rates as they are now

    def at(self, offset: int) -> "AdapterDropout":
        """The same rates and seed with another offset."""
        out = AdapterDropout(0.0, self.seed, offset)
        object.__setattr__(out, "rates", self.rates)
        object.__setattr__(out, "_thresholds", self._thresholds)
        return out

    @staticmethod
    def _threshold(rate: float) -> int:
        t = round(float(rate) * 65536) if 0.0 <= rate < 1.0 else 65536
        if t >= 65536:
            raise ValueError(f"a dropout rate must be at least 0 and below 1 (to 1/65536), got {rate!r}")
        return t

    def threshold(self, adapter_id: int) -> int:
        """65536 times the adapter's rate, a whole number (``KeyError`` for an adapter that the mapping lacks)."""
        t = self._thresholds
        return t if type(t) is int else t[adapter_id]
