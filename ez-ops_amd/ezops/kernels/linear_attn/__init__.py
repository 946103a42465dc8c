from . import linear_attn_hip  # noqa: F401
