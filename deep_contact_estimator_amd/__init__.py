"""deep_contact_estimator_amd -- MI355X-native sliding-window contact-state inference.

Drop-in for the reference's inference path (contact_cnn.forward + the windowed batching
loops); see DESIGN.md and INTEGRATION.md.  Importing the package does not need a GPU or the
built library; using the model does (there is no CPU fallback).
"""
from .contact_cnn import contact_cnn, load_checkpoint          # noqa: F401
from . import synth                                              # noqa: F401

__all__ = ["contact_cnn", "load_checkpoint", "synth"]              # (without contact_bank and ops, which import torch: `import *` works where there is none)


def __getattr__(name):                                             # (only when asked for)
    import importlib
    if name == "ops":
        return importlib.import_module(".ops", __name__)
    if name == "contact_bank":
        return importlib.import_module(".bank", __name__).contact_bank
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
