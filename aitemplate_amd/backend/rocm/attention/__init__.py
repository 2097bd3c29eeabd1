from . import mem_eff_attention, paged_attention  # noqa: F401  (registers the rocm.<op>.* hooks)
