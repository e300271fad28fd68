"""Drawing the next token: temperature, the k largest logits, the likeliest p, at least min_p, from random numbers of a seed."""
import torch

try:
    from . import float_kernel as K
except ImportError:  # pragma: no cover - this directory first on sys.path
    import float_kernel as K


class Sampler:
    """Called with logits [rows, vocab] (float32 or bfloat16, on the GPU): one token per row, int64.  The random numbers come from a
    generator of its own, one per row and call, so that a seed repeats a run.  See `float_kernel.sample` for what a row keeps."""

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, seed=0):
        self.settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        self.seed, self.generator = seed, None

    def __call__(self, logits):
        if self.generator is None:
            self.generator = torch.Generator(logits.device).manual_seed(self.seed)
        u = torch.rand(logits.shape[0], generator=self.generator, device=logits.device)
        return K.sample(logits, u, **self.settings)
