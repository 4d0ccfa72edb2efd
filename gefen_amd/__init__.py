"""gefen_amd: the Gefen optimizer step, MI355X-native (HIP kernels for gfx950).

``from gefen_amd import Gefen, GefenMuon`` replaces ``from gefen import Gefen, GefenMuon``
(reference __init__.py:1-13); the optimizer classes are loaded lazily.

Beside the optimizers, what a training step does around them: ``linear_cross_entropy``
(the loss of an output matrix with its gradients, without the logits), ``gradient_norm``,
``clip_gradients`` and ``clip_grad_norm_``.
"""

__all__ = ["Gefen", "GefenMuon", "kernels", "linear_cross_entropy", "gradient_norm", "clip_gradients",
           "clip_grad_norm_"]


def __getattr__(name):
    if name == "Gefen":
        from .gefen import Gefen

        return Gefen
    if name == "GefenMuon":
        from .gefen_muon import GefenMuon

        return GefenMuon
    if name in ("linear_cross_entropy", "gradient_norm", "clip_gradients", "clip_grad_norm_"):
        import importlib

        module = "linear_cross_entropy" if name == "linear_cross_entropy" else "gradient_norm"
        value = getattr(importlib.import_module("gefen_amd.kernels." + module), name)
        globals()[name] = value  # found directly from now on
        return value
    raise AttributeError("module {!r} has no attribute {!r}".format(__name__, name))
