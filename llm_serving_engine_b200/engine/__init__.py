from .beam_search import Beam, BeamSearch
from .scheduler import GenerationRequest, Scheduler
from .step import StepContext, StepEntry, StepRunner

__all__ = ["Beam", "BeamSearch", "GenerationRequest", "Scheduler", "StepContext", "StepEntry", "StepRunner"]
