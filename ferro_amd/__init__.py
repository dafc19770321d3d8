"""ferro_amd: MI355X (gfx950) token sampler for ferro - the penalty / top-k / top-p / softmax / draw / argmax /
draft-verification hot path as HIP kernels behind the C ABI of include/ferro_sampler.h."""
from .sampler import (BEAM_KEEP_SLOTS, BF16, F16, F32, PARAMS_DTYPE, Context, DeviceRng, Edits, Rng, Sampler,  # noqa: F401
                      SamplerError, SamplerParams, States, argmax_batch, beam_select, decode_step, device_error, edit_batch,
                      hist_append, hist_fork, logprobs, lookup_draft, params_array, penalize_batch, reorder_states,
                      sample_batch, verify)
