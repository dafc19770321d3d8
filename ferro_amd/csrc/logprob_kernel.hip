// logprob_kernel.hip - log-probabilities of a row's tokens:
//
//   lp(t) = (x_t - M) / T - log sum_j exp((x_j - M) / T),   x = cap(logit) + bias over the allowed tokens, M = max x,
//
// of one chosen token per row with its rank (1 + the number of larger x), and of the row's n largest (the lower id first
// among equal ones). Tokens that are not allowed, NaN and -inf take no part.
// One workgroup of SK_LT threads per (row, segment of 1024 NL logits), the segment's logits requested at once and kept in
// registers: its maximum, the sum of exponentials (fp32 per lane over at most 64 terms, added in fp64), the logits above
// the chosen one, and its n largest (lane maxima sorted in each wave give a bound that at least n logits reach; those at
// or above it, about 1.5 n, are ranked in LDS). The row's last segment (an L2 ticket) joins them: sums in fp64, sorted
// lists by bitonic merges. One read of the logits, whatever is asked.
// Bound: HBM.
#include "edit_device.hpp"
#include "row_device.hpp"

namespace fs {

constexpr int LP_CAP = 1024;               // candidates a segment ranks in LDS

struct LpShared {
    uint64_t cand[LP_CAP];
    uint64_t wl[SK_NW][LP_TOP];
    double sum[SK_NW];
    float max[SK_NW];
    uint32_t above[SK_NW];
    uint32_t bound[SK_NW];
    uint32_t hist[16];
    uint32_t n, last;
    uint32_t digit, need;
};

// x above -inf (a token that takes part): its composite, else 0
__device__ __forceinline__ uint64_t lp_comp(float x, uint32_t id) {
    return x > -__builtin_huge_valf() ? comp_of(key_of(x), id) : 0ull;
}

// The exact k-th largest composite of a segment (0: it holds fewer), by a radix select over 4-bit digits of the logits in
// the registers. For segments with more than LP_CAP logits at the bound (equal ones). Whole workgroup.
template <int NL>
__device__ __forceinline__ uint64_t lp_kth(const float (&x)[NL][4], int seg_lo, int k, LpShared& s) {
    const int tid = threadIdx.x;
    uint64_t prefix = 0ull;
    int need = k;
#pragma unroll 1
    for (int sh = 60; sh >= 0; sh -= 4) {
        __syncthreads();
        if (tid < 16) s.hist[tid] = 0u;
        __syncthreads();
        const uint64_t hi = sh + 4 >= 64 ? 0ull : (~0ull << (sh + 4));
#pragma unroll
        for (int q = 0; q < NL; ++q)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint64_t cm = lp_comp(x[q][c], (uint32_t)(seg_lo + (q * SK_LT + tid) * 4 + c));
                if (cm != 0ull && (cm & hi) == prefix) atomicAdd(&s.hist[(uint32_t)(cm >> sh) & 15u], 1u);
            }
        __syncthreads();
        if (tid == 0) {
            int d = 15;
            for (; d > 0; --d) {
                const int c = (int)s.hist[d];
                if (c >= need) break;
                need -= c;
            }
            s.digit = (uint32_t)d;
            s.need = (uint32_t)need;
        }
        __syncthreads();
        prefix |= (uint64_t)s.digit << sh;
        need = (int)s.need;
    }
    return prefix;
}

template <int TYPE, int NL, bool TOP>
__global__ __launch_bounds__(SK_LT) void logprob_kernel(LpArgs a) {
    constexpr int SEG = SK_LT * NL * 4;
    __shared__ __align__(16) LpShared s;
    const int tid = threadIdx.x, lane = lane_id(), w = tid / WAVE;
    const int row = (int)blockIdx.x / a.nseg, seg = (int)blockIdx.x - row * a.nseg;
    const int seg_lo = seg * SEG, V = a.V;
    const int n_in = V - seg_lo < SEG ? V - seg_lo : SEG;
    constexpr float NONE = -__builtin_huge_valf();
    using L = Logits4<TYPE>;
    const __amdgpu_buffer_rsrc_t rs = L::rsrc(a.logits, (int64_t)row * a.ld + seg_lo, n_in);
    typename L::raw raw[NL];
#pragma unroll
    for (int q = 0; q < NL; ++q) raw[q] = L::load(rs, q * SK_LT + tid);

    const EdRow r = ed_row(a.ed, row, row, a.err);
    const EdBits bits = ed_bits<NL>(r, seg_lo, V);
    float cap = 0.0f, T = 1.0f;
    if (a.params) {
        cap = ld_const(&a.params[row].softcap);
        T = ld_const(&a.params[row].temperature);
        if (!(T > 0.0f)) T = 1.0f;                             // greedy rows: the distribution itself
    }
    // the chosen token's logit
    const int t = a.tok ? ld_const(a.tok + row) : -1;
    float xt = NONE;
    if (t >= 0 && t < V) {
        float l = L::one(a.logits, (int64_t)row * a.ld + t);
        if (cap > 0.0f) l = softcap_one(l, cap);
        xt = fmaxf(ed_one(r, l, t), NONE);                     // (NaN: -inf)
    }

    float x[NL][4];
#pragma unroll
    for (int q = 0; q < NL; ++q) {
        L::floats(raw[q], x[q]);
        if (cap > 0.0f) softcap_vals(x[q], cap);
    }
    if (r.nb > 0) ed_add<NL>(r, seg_lo, n_in, [&](int q, int c) -> float& { return x[q][c]; });
    float lm = NONE;
    uint32_t above = 0u;
#pragma unroll
    for (int q = 0; q < NL; ++q) {
        const uint32_t nib = ed_nibble(bits, q);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const bool in = (q * SK_LT + tid) * 4 + c < n_in;
            x[q][c] = in ? fmaxf(ed_keep(x[q][c], nib, c, 0xFF800000u), NONE) : NONE;
            above += x[q][c] > xt ? 1u : 0u;
        }
        lm = fmaxf(lm, fmaxf(fmaxf(x[q][0], x[q][1]), fmaxf(x[q][2], x[q][3])));
    }
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    auto addu = [](uint32_t u, uint32_t v) { return u + v; };
    auto addf = [](double u, double v) { return u + v; };
    const float wm = wave_allreduce(lm, fmx);
    if (lane == 0) s.max[w] = wm;
    if (TOP) {
        // kq-th largest lane maximum of each wave; the smallest over the waves counts SK_NW kq >= n distinct logits
        const int kq = (a.n + SK_NW - 1) / SK_NW;
        const uint32_t srt = sort64_desc_u32(lm > NONE ? key_of(lm) : 0u);
        if (lane == kq - 1) s.bound[w] = srt;
        if (tid == 0) s.n = 0u;
    }
    above = wave_allreduce(above, addu);
    if (lane == 0) s.above[w] = above;
    __syncthreads();
    const float M = fmaxf(fmaxf(s.max[0], s.max[1]), fmaxf(s.max[2], s.max[3]));
    double part = 0.0;
    if (M > NONE) {
        float e = 0.0f;
        if (M < __builtin_huge_valf()) {
            const float inv = 1.0f / T;
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) e += __expf((x[q][c] - M) * inv);
        } else {                                               // an infinite maximum: its tokens share the mass
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) e += x[q][c] == M ? 1.0f : 0.0f;
        }
        part = wave_allreduce((double)e, addf);
    }
    if (lane == 0) s.sum[w] = part;
    uint64_t* myl = a.lists + ((int64_t)row * a.nseg + seg) * LP_TOP;
    if (TOP) {
        uint32_t tau = s.bound[0];
#pragma unroll
        for (int q = 1; q < SK_NW; ++q) tau = s.bound[q] < tau ? s.bound[q] : tau;
        const float tf = tau != 0u ? val_of(tau) : -3.402823466e38f;      // (no bound: every token)
#pragma unroll
        for (int q = 0; q < NL; ++q) {
            if (__ballot(fmaxf(fmaxf(x[q][0], x[q][1]), fmaxf(x[q][2], x[q][3])) >= tf) != 0ull) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (x[q][c] >= tf) {
                        const uint32_t at = atomicAdd(&s.n, 1u);
                        if (at < (uint32_t)LP_CAP)
                            s.cand[at] = comp_of(key_of(x[q][c]), (uint32_t)(seg_lo + (q * SK_LT + tid) * 4 + c));
                    }
            }
        }
        __syncthreads();
        uint32_t n = s.n;
        if (n > (uint32_t)LP_CAP) {                            // uniform: equal logits at the bound
            const uint64_t kth = lp_kth(x, seg_lo, a.n, s);
            __syncthreads();
            if (tid == 0) s.n = 0u;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint64_t cm = lp_comp(x[q][c], (uint32_t)(seg_lo + (q * SK_LT + tid) * 4 + c));
                    if (cm != 0ull && cm >= kth) s.cand[atomicAdd(&s.n, 1u)] = cm;     // a.n of them
                }
            __syncthreads();
            n = s.n;
        }
        for (uint32_t c = (uint32_t)tid; c < n; c += SK_LT) {
            const uint64_t me = s.cand[c];
            uint32_t rank = 0u;
            for (uint32_t j = 0; j < n; ++j) rank += s.cand[j] > me ? 1u : 0u;
            if (rank < (uint32_t)a.n) st_agent(&myl[rank], me);
        }
        if (tid < LP_TOP && tid >= (int)(n < (uint32_t)a.n ? n : (uint32_t)a.n)) st_agent(&myl[tid], (uint64_t)0);
    }
    __syncthreads();
    if (tid == 0) {
        LpPart* o = a.part + (int64_t)row * a.nseg + seg;
        const double sum = s.sum[0] + s.sum[1] + s.sum[2] + s.sum[3];
        st_agent(reinterpret_cast<uint64_t*>(&o->sum), (uint64_t)__double_as_longlong(sum));
        st_agent(reinterpret_cast<uint64_t*>(&o->max), ((uint64_t)(s.above[0] + s.above[1] + s.above[2] + s.above[3]) << 32) |
                                                           __float_as_uint(M));
    }
    vm_drain();                                                // the segment's results are out
    __syncthreads();
    if (tid == 0)
        s.last = __hip_atomic_fetch_add(a.ticket + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 (uint32_t)a.nseg - 1u ? 1u : 0u;
    __syncthreads();
    if (s.last == 0u) return;

    // ---- the row's end, by its last segment
    const LpPart* pr = a.part + (int64_t)row * a.nseg;
    const uint64_t* rl = a.lists + (int64_t)row * a.nseg * LP_TOP;
    uint64_t acc = 0ull;
    if (TOP) {                                                 // wave w folds lists w, w + SK_NW, ..., then wave 0 the waves'
        for (int i = w; i < a.nseg; i += SK_NW) {
            const uint64_t b = ld_agent(&rl[(int64_t)i * LP_TOP + WAVE - 1 - lane]);      // ascending
            acc = merge_top64(acc, b);
        }
        s.wl[w][lane] = acc;
        __syncthreads();
    }
    if (w != 0) return;
    if (lane == 0) __hip_atomic_store(a.ticket + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float m = NONE;
    for (int i = lane; i < a.nseg; i += WAVE)
        m = fmaxf(m, __uint_as_float((uint32_t)ld_agent(reinterpret_cast<const uint64_t*>(&pr[i].max))));
    m = wave_allreduce(m, fmx);
    double S = 0.0;
    uint32_t ab = 0u;
    for (int i = lane; i < a.nseg; i += WAVE) {
        const uint64_t e = ld_agent(reinterpret_cast<const uint64_t*>(&pr[i].max));
        const double sum = __longlong_as_double((long long)ld_agent(reinterpret_cast<const uint64_t*>(&pr[i].sum)));
        const float mi = __uint_as_float((uint32_t)e);
        ab += (uint32_t)(e >> 32);
        if (mi > NONE) S += mi == m ? sum : sum * exp(((double)mi - (double)m) / (double)T);
    }
    S = wave_allreduce(S, addf);
    ab = wave_allreduce(ab, addu);
    const double z = log(S);
    auto lp_of = [&](float v) { return v > NONE ? (float)((v == m ? 0.0 : ((double)v - (double)m) / (double)T) - z) : NONE; };
    if (lane == 0) {
        if (a.lp) a.lp[row] = lp_of(xt);
        if (a.rank) a.rank[row] = xt > NONE ? (int)ab + 1 : 0;
    }
    if (TOP) {
#pragma unroll 1
        for (int i = 1; i < SK_NW; ++i) acc = merge_top64(acc, s.wl[i][WAVE - 1 - lane]);
        if (lane < a.n) {
            if (a.ids) a.ids[(int64_t)row * a.n + lane] = acc != 0ull ? (int)comp_id(acc) : -1;
            if (a.top) a.top[(int64_t)row * a.n + lane] = acc != 0ull ? lp_of(val_of(comp_key(acc))) : NONE;
        }
    }
}

hipError_t launch_logprobs(int nl, int type, const LpArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.B * a.nseg)), block(SK_LT);
    auto go = [&](auto t, auto top) {
        constexpr int T = decltype(t)::value;
        constexpr bool P = decltype(top)::value;
        if (nl == 16) hipLaunchKernelGGL((logprob_kernel<T, 16, P>), grid, block, 0, st, a);
        else if (nl == 8) hipLaunchKernelGGL((logprob_kernel<T, 8, P>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((logprob_kernel<T, 4, P>), grid, block, 0, st, a);
    };
    auto by_top = [&](auto t) {
        if (a.n > 0) go(t, std::true_type{});
        else go(t, std::false_type{});
    };
    if (type == FS_F32) by_top(std::integral_constant<int, FS_F32>{});
    else if (type == FS_BF16) by_top(std::integral_constant<int, FS_BF16>{});
    else by_top(std::integral_constant<int, FS_F16>{});
    return hipGetLastError();
}

}  // namespace fs
