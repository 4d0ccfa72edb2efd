"""gefen_amd: the Gefen optimizer step, MI355X-native (HIP kernels for gfx950).

``from gefen_amd import Gefen, GefenMuon`` replaces ``from gefen import Gefen, GefenMuon``
(reference __init__.py:1-13); the optimizer classes are loaded lazily.

Beside the optimizers, what a training step does around them: ``linear_cross_entropy``
(the loss of an output matrix with its gradients, without the logits), ``gradient_norm``,
``clip_gradients`` and ``clip_grad_norm_``; and what a layer does beside its matrix products:
``attention``, ``rms_norm`` (with the residual's addition; ``rms_norm_quantized`` with an 8-bit
output) and ``dropout``.
"""

__all__ = ["Gefen", "GefenMuon", "kernels", "linear_cross_entropy", "gradient_norm", "clip_gradients",
           "clip_grad_norm_", "attention", "rms_norm", "rms_norm_quantized", "dropout"]

_OPERATORS = {
    "linear_cross_entropy": "linear_cross_entropy",
    "gradient_norm": "gradient_norm", "clip_gradients": "gradient_norm", "clip_grad_norm_": "gradient_norm",
    "attention": "attention", "rms_norm": "rms_norm", "rms_norm_quantized": "rms_norm", "dropout": "dropout",
}


def __getattr__(name):
    if name == "Gefen":
        from .gefen import Gefen

        return Gefen
    if name == "GefenMuon":
        from .gefen_muon import GefenMuon

        return GefenMuon
    if name in _OPERATORS:
        import importlib

        value = getattr(importlib.import_module("gefen_amd.kernels." + _OPERATORS[name]), name)
        globals()[name] = value  # found directly from now on
        return value
    raise AttributeError("module {!r} has no attribute {!r}".format(__name__, name))
