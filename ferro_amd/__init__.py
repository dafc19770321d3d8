"""ferro_amd: MI355X (gfx950) token sampler for ferro - the penalty / top-k / top-p / softmax / draw / argmax /
draft-verification hot path as HIP kernels behind the C ABI of include/ferro_sampler.h."""
from .sampler import (BF16, F16, F32, PARAMS_DTYPE, Context, DeviceRng, Edits, Rng, Sampler, SamplerError, SamplerParams,  # noqa: F401
                      argmax_batch, decode_step, device_error, edit_batch, hist_append, logprobs, lookup_draft, params_array,
                      penalize_batch, sample_batch, verify)
