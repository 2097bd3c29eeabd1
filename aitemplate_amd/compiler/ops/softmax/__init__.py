from .token_logprobs import token_logprobs  # noqa: F401
