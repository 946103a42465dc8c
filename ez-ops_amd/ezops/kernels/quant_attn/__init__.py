from . import quant_attn_hip  # noqa: F401
