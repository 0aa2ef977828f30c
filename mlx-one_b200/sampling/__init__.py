from .options import BeamResult, GenerationChunk, GenerationResult, TextGenerationOptions

__all__ = ["BeamResult", "GenerationChunk", "GenerationResult", "TextGenerationOptions"]
