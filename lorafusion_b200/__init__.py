"""lorafusion_b200: lorafusion's fused multi-adapter LoRA operator, rebuilt for NVIDIA B200 (sm_100a).

* :mod:`lorafusion_b200.b200_ops` — ``fused_lora_forward`` / ``fused_lora_backward``,
  the drop-in backend (same API as ``lorafusion.ops.mock_ops``).
* :mod:`lorafusion_b200.config` — ``AdapterSpec``, ``TileRoute``, ``TileRoutingConfig``,
  ``AdapterDropout`` (dropout in front of the adapters, its mask never stored).
* :mod:`lorafusion_b200.scheduler` — grouping, bin packing and fused-batch assembly.
* :mod:`lorafusion_b200.coordinator` — ``Coordinator`` (request batch in, results out).
* :mod:`lorafusion_b200.training` — what follows the backward: ``clip_adapter_grads`` and ``AdapterAdamW``, each
  adapter with its own norm, step count and rates.
* :mod:`lorafusion_b200.serving` — trained adapters resident in an ``AdapterBank`` and
  ``fused_lora_forward_rows``, one projection for rows of many requests, an adapter index per row.
* :mod:`lorafusion_b200.quant` — a frozen base weight in 4 bits, ``MX4Weight``, taken by the fused ops in the place of
  a dense one, and its products.
* :mod:`lorafusion_b200.sharding` — row sharding of packed bins across GPUs and the
  gradient all-reduce of adapters that span ranks.
"""

__version__ = "0.1.0"

from lorafusion_b200.config import AdapterDropout, AdapterSpec, TileRoute, TileRoutingConfig  # noqa: F401
