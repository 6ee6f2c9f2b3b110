"""artemis_amd: the ArTEMIS frame-synthesis hot path (cupy_module/synth.py upstream) as
hand-written MI355X (gfx950) HIP kernels behind a C ABI, with the reference's
``FunctionSynth`` operator interface on top; beside it the encoder's operators (layer norm, windowed attention) and
the AdamW step, from a second library of the same kind."""
from .synth import (FunctionSynth, FunctionSynthFrame, synth, synth_unpadded, synth_strip,  # noqa: F401
                    synth_options, options, offset_radius, suggest_tile_radius, adaptive_state,
                    FunctionChronoHead,
                    chrono_head)
from .encoder_ops import layer_norm, window_attention  # noqa: F401
from .optim import AdamW, adamw_step, adamw_step_8bit, moments_from_8bit  # noqa: F401
from ._lib import version, SynthLibraryError  # noqa: F401

__all__ = ["FunctionSynth", "FunctionSynthFrame", "synth", "synth_unpadded", "synth_strip", "FunctionChronoHead", "chrono_head", "synth_options", "options", "offset_radius", "suggest_tile_radius", "adaptive_state", "version",
           "SynthLibraryError", "layer_norm", "window_attention", "AdamW",
           "adamw_step", "adamw_step_8bit", "moments_from_8bit"]
