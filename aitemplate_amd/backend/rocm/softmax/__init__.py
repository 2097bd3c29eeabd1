from . import token_logprobs  # noqa: F401  (registers the rocm.<op>.* hooks)
