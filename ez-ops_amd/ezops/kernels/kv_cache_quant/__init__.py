from . import kv_cache_quant_hip  # noqa: F401
