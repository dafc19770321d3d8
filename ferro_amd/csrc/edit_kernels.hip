// edit_kernels.hip - edited logits written out (fs_edit_batch), and rows edited for the sampling kernels that do not read
// masks and biases themselves.
//
//   out[t] = -inf where bit t of the row's mask is 0, else pen(cap(x[t]) + bias[t]),
//
// cap: the final softcap; pen: the repetition, then the frequency / presence penalties over the row's window (sampler.cpp:
// 11-18 and the extension), every step rounded to fp32 as ferro's sampler rounds its own (so that a row edited here and
// sampled equals one sampled under the edits).
// One workgroup of SK_LT threads per (row, segment of 1024 NL logits): the segment's logits are requested first and stay in
// registers; the window's ids are counted in LDS (16 bits per logit) while they arrive; the mask's words come with one load
// per wave and eight groups, the biases 64 at a time.
// Bound: HBM, V times the type's size read and 4 V written per row: 64 rows of 262144, 18.5 us from bf16 (4.9 TB/s of its
// 90.9 MB; a copy of 4 GiB reaches 4.8), 24.7 from fp32. A single row is a launch and the chain offsets, ids, counts:
// 4.4-5.0 us for 65536 logits. Under a softcap the tanh counts, too: 24 rows of 100003 fp16 under masks, windows of 4096 ids,
// 300 biases each, 16.9 us; the masks alone 5.3, with the cap 11.5, with the windows 9.6, with the biases 7.0.
#include "edit_device.hpp"

#include <type_traits>

namespace fs {

template <int TYPE, int NL>
__global__ __launch_bounds__(SK_LT) void edit_kernel(EditArgs e) {
    constexpr int SEG = SK_LT * NL * 4;
    __shared__ __align__(16) uint32_t cnt[SEG / 2];            // occurrences in the window, 16 bits per logit
    const int tid = threadIdx.x, lane = lane_id();
    const int row = (int)blockIdx.x / e.nseg, seg = (int)blockIdx.x - row * e.nseg;
    const int seg_lo = seg * SEG, V = e.V;
    const int n_in = V - seg_lo < SEG ? V - seg_lo : SEG;
    using L = Logits4<TYPE>;
    const __amdgpu_buffer_rsrc_t rs = L::rsrc(e.logits, (int64_t)row * e.ld + seg_lo, n_in);
    typename L::raw raw[NL];
#pragma unroll
    for (int q = 0; q < NL; ++q) raw[q] = L::load(rs, q * SK_LT + tid);

    // verification windows: the row's stream, and the drafts fed before the row behind its history
    int rec = row, nb = 0;
    const int32_t* pb = nullptr;
    if (e.n_streams > 0) {
        int s0 = 0, s1 = e.n_streams;                          // the largest s with row_off[s] <= row
        while (s1 - s0 > 1) {
            const int m = (s0 + s1) >> 1;
            if (ld_const(e.row_off + m) <= row) s0 = m; else s1 = m;
        }
        rec = s0;
        const int64_t r0 = ld_const(e.row_off + s0);
        pb = e.rows + r0 + 1;
        nb = row - (int)r0;
    }
    fs_row_params p = {0.0f, 0, 1.0f, 0.0f, 1.0f, 0.0f, 0.0f, 0, 0, 0.0f};
    if (e.params) p = ld_const(e.params + rec);
    const EdRow r = ed_row(e.ed, row, rec, e.err);
    const EdBits bits = ed_bits<NL>(r, seg_lo, V);
    const EdList few = ed_list<false>(r);

    const bool rep_on = p.repetition_penalty != 1.0f;
    const bool fp_on = p.frequency_penalty != 0.0f || p.presence_penalty != 0.0f;
    int64_t h0 = 0, na = 0;
    if (e.hist && e.hist_off) {
        h0 = ld_const(e.hist_off + rec);
        na = ld_const(e.hist_off + rec + 1) - h0;
    }
    const int64_t len = na + nb, from = window_begin(len, p);
    const bool pen = e.params && (rep_on || fp_on) && p.repeat_last_n != 0 && from < len;   // uniform
    if (pen) {
        for (int i = tid; i < SEG / 8; i += SK_LT) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        bool ovf = false;
        auto mark = [&](int id) {
            const uint32_t rel = (uint32_t)id - (uint32_t)seg_lo;
            if (rel < (uint32_t)n_in) {
                const uint32_t sh = (rel & 1u) * 16u;
                ovf |= ((atomicAdd(&cnt[rel >> 1], 1u << sh) >> sh) & 0xFFFFu) == 0xFFFFu;
            }
        };
        constexpr int U = 8;                                   // ids in flight per thread
        for (int64_t i0 = from + tid; i0 < na; i0 += U * SK_LT) {
            int id[U];
#pragma unroll
            for (int j = 0; j < U; ++j) id[j] = i0 + j * SK_LT < na ? e.hist[h0 + i0 + j * SK_LT] : -1;
#pragma unroll
            for (int j = 0; j < U; ++j) mark(id[j]);
        }
        for (int64_t i = (from > na ? from - na : 0) + tid; i < nb; i += SK_LT) mark(pb[i]);
        if (ovf) atomicOr(e.err, FS_DEVERR_COUNT_OVERFLOW);
        __syncthreads();
    }

    float x[NL][4];
#pragma unroll
    for (int q = 0; q < NL; ++q) {
        L::floats(raw[q], x[q]);
        if (p.softcap > 0.0f) softcap_vals_unrolled(x[q], p.softcap);
    }
    if (few.nb > 0) ed_add<NL, false>(e.ed, rec, few, nullptr, seg_lo, n_in, [&](int q, int c) -> float& { return x[q][c]; });
    const bool greedy = p.temperature <= 0.0f || p.top_k == 1;
    const uint32_t none = e.any ? 0x7FC00000u : 0xFF800000u;   // the sampling kernels' rows: NaN, never a candidate
    float* out = e.out + (int64_t)row * e.out_ld + seg_lo;
    bool any = false;
#pragma unroll
    for (int q = 0; q < NL; ++q) {
        const int at = (q * SK_LT + tid) * 4;
        if (pen) {
            const uint2 c2 = *reinterpret_cast<const uint2*>(&cnt[at >> 1]);
            if ((c2.x | c2.y) != 0u) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t n = ((c < 2 ? c2.x : c2.y) >> (16 * (c & 1))) & 0xFFFFu;
                    if (n != 0u) {
                        float l = x[q][c];
                        if (rep_on) l = l > 0.0f ? __fdiv_rn(l, p.repetition_penalty) : __fmul_rn(l, p.repetition_penalty);
                        if (fp_on)
                            l = __fsub_rn(l, __fadd_rn(__fmul_rn((float)n, p.frequency_penalty), p.presence_penalty));
                        x[q][c] = l;
                    }
                }
            }
        }
        const uint32_t nib = ed_nibble(bits, q);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[q][c] = ed_keep(x[q][c], nib, c, none);
        if (e.any) {                                           // candidates are above -inf
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const bool is = x[q][c] > -__builtin_huge_valf();
                any |= is && at + c < n_in;
                // (ferro's greedy scan keeps index 0 when its logit is NaN: -inf there loses to any candidate)
                if (!is) x[q][c] = greedy && seg_lo + at + c == 0 ? -__builtin_huge_valf() : __uint_as_float(none);
            }
        }
        if (at + 4 <= n_in) {
            *reinterpret_cast<float4*>(out + at) = make_float4(x[q][0], x[q][1], x[q][2], x[q][3]);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (at + c < n_in) out[at + c] = x[q][c];
        }
    }
    if (e.any) {
        if (__ballot(any) != 0ull && lane == 0) atomicOr(&e.any[row], 1u);
        if (seg == 0 && tid == 0) {
            fs_row_params o = p;
            o.repetition_penalty = 1.0f; o.frequency_penalty = 0.0f; o.presence_penalty = 0.0f;
            o.repeat_last_n = 0; o.penalty_from = 0; o.softcap = 0.0f;
            e.rparams[row] = o;
        }
    }
}

hipError_t launch_edit(int nl, const EditArgs& e, hipStream_t st) {
    auto go = [&](auto type) {
        constexpr int T = decltype(type)::value;
        const dim3 grid((unsigned)((int64_t)e.B * e.nseg)), block(SK_LT);
        if (nl == 8) hipLaunchKernelGGL((edit_kernel<T, 8>), grid, block, 0, st, e);
        else if (nl == 4) hipLaunchKernelGGL((edit_kernel<T, 4>), grid, block, 0, st, e);
        else hipLaunchKernelGGL((edit_kernel<T, 2>), grid, block, 0, st, e);
    };
    if (e.type == FS_F32) go(std::integral_constant<int, FS_F32>{});
    else if (e.type == FS_BF16) go(std::integral_constant<int, FS_BF16>{});
    else go(std::integral_constant<int, FS_F16>{});
    return hipGetLastError();
}

// One wave per row, or per stream of a verification window.
__global__ __launch_bounds__(WAVE) void edit_end_kernel(EditEnd e) {
    const int lane = lane_id();
    int64_t r0 = blockIdx.x, m = 1;
    if (e.n_streams > 0) {
        r0 = ld_const(e.row_off + blockIdx.x);
        m = ld_const(e.row_off + blockIdx.x + 1) - r0;
    }
    int acc = 0;
    bool walking = true;
    for (int64_t c0 = 0; c0 < m; c0 += WAVE) {
        const int64_t i = c0 + lane;
        bool stop = false;
        if (i < m) {
            const int64_t row = r0 + i;
            int tok = e.tok[row];
            if (e.any[row] == 0u) {
                tok = -1;
                e.tok[row] = tok;
                if (e.keep) e.keep[row] = 0;
                const fs_row_params& p = e.rparams[row];
                if (e.kcap > 0 && (p.temperature <= 0.0f || p.top_k == 1)) {
                    if (e.cand_ids) e.cand_ids[row * e.kcap] = -1;
                    if (e.cand_probs) e.cand_probs[row * e.kcap] = 0.0;
                }
            }
            e.any[row] = 0u;
            if (e.n_streams > 0) stop = tok < 0 || (e.eos >= 0 && tok == e.eos) || i + 1 >= m || tok != e.rows[row + 1];
        }
        const uint64_t b = __ballot(stop);
        if (walking) acc = b ? (int)c0 + __ffsll((unsigned long long)b) : (int)(m < c0 + WAVE ? m : c0 + WAVE);
        walking = walking && b == 0ull;
    }
    if (e.n_streams > 0) {
        if (lane == 0 && m > 0) e.accepted[blockIdx.x] = acc;
        if ((int)blockIdx.x == e.n_streams - 1)                // rows behind the last stream's
            for (int64_t row = r0 + m + lane; row < e.B; row += WAVE) e.any[row] = 0u;
    }
}

hipError_t launch_edit_end(const EditEnd& e, hipStream_t st) {
    hipLaunchKernelGGL(edit_end_kernel, dim3((unsigned)(e.n_streams > 0 ? e.n_streams : e.B)), dim3(WAVE), 0, st, e);
    return hipGetLastError();
}

}  // namespace fs
