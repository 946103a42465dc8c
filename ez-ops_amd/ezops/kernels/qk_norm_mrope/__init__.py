from . import qk_norm_mrope_hip  # noqa: F401
