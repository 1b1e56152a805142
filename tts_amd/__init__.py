"""tts_amd: MI355X-native Griffin-Lim vocoder (mel -> waveform), a drop-in for the
``mel_to_audio_griffin_lim`` function of the reference's vocoder/mel_audio.py, and the MXFP4 and
block operators its acoustic model is served with."""
from .blocks import MXFP4Tensor, Norm, block_norm, mxfp4_conv1d, mxfp4_linear, mxfp4_quantize
from .vocoder import (GriffinLimPlan, HaloChain, audio_to_mel_db, get_plan, griffin_lim_batch, mel_to_audio,
                      mel_to_audio_griffin_lim)

__all__ = ["GriffinLimPlan", "HaloChain", "MXFP4Tensor", "Norm", "audio_to_mel_db", "block_norm", "get_plan",
           "griffin_lim_batch", "mel_to_audio", "mel_to_audio_griffin_lim", "mxfp4_conv1d", "mxfp4_linear",
           "mxfp4_quantize"]
__version__ = "0.1.0"
