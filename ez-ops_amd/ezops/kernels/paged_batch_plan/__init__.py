from . import paged_batch_plan_hip  # noqa: F401
