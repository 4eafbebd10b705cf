from .api import Engine
from .beam import BeamOptions, Hypothesis, beam_loop
from .generate import GenerationOptions, GenStats, generate_loop
from .model import DecoderModel, load_model, weight_manifest
from .step import StepError, Stepper

__all__ = ["BeamOptions", "Engine", "Hypothesis", "beam_loop", "GenerationOptions", "GenStats", "generate_loop", "DecoderModel", "load_model",
           "weight_manifest", "StepError", "Stepper"]
