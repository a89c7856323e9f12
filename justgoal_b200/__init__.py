"""B200-native FP8 block-scale MoE layer behind the reference's operator entry point.

`run` / `run_dps` keep the reference solutions' `main.py::run` signature; `MoELayer` is the
handle-based form for other shapes (e.g. the Qwen3-MoE shape) and for expert parallelism;
`HostPipeline` overlaps the host<->device copies of consecutive steps with the forward.
`sort_tokens`, `permute`, `combine`, `restore_1x128`, `swiglu_save` and `route_backward`, with the gradients beside them, are the
operators between and around the GEMMs for training (`train.py`).
They are resolved on first use, which loads libb200moe.so and raises if it is missing (build
it with `python -m justgoal_b200.build`): there is no CPU or PyTorch fallback.
"""
from .inputs import (DEEPSEEK_V3, QWEN3_MOE, TINY_DS, TINY_RENORM, MoEShape, ROUTING_DS,  # noqa: F401
                     ROUTING_RENORM_NAIVE)

_LAZY = {"MoELayer": "main", "HostPipeline": "main", "run": "main", "run_dps": "main", "quantize_1x128": "main",
         "B200MoEError": "_lib",
         **{name: "train" for name in ("TokenOrder", "sort_tokens", "permute", "permute_backward", "restore_1x128", "combine", "combine_backward",
                                       "swiglu_save", "swiglu_backward", "route_backward")}}


def __getattr__(name):
    mod = _LAZY.get(name)
    if mod is None:
        raise AttributeError(f"module 'justgoal_b200' has no attribute {name!r}")
    import importlib
    return getattr(importlib.import_module("." + mod, __name__), name)
