// logprob_kernel.hip - log-probabilities of a row's tokens:
//
//   lp(t) = (x_t - M) / T - log sum_j exp((x_j - M) / T),   x = cap(logit) + bias over the allowed tokens, M = max x,
//
// of one chosen token per row with its rank (1 + the number of larger x), and of the row's n largest (the lower id first
// among equal ones). Tokens that are not allowed, NaN and -inf take no part.
// One workgroup of SK_LT threads per (row, part): a part is a run of chunks of 16 KB of logits, read once, the next chunk
// requested before the present one is worked on. Every wave works by itself until its part ends (no barrier in between):
//   - the sum: exponentials of c (x - m), c = log2 e / T and m the wave's largest x so far (the largest term is 1, exactly).
//     A chunk's 16 or 32 terms of a lane are added in fp32, chunks in fp64, and a new m scales the lanes' sums in fp64; a
//     subtraction, a product, an exponential and an addition a logit;
//   - a chunk whose sum is NaN (NaN or infinite logits) is added again with those left out; where the row's largest logit
//     is infinite its tokens are counted instead;
//   - the n largest: a bound, first the n-th of the wave's 64 lane maxima, passes over chunks without a candidate by one
//     compare a lane; the others go to a list in LDS, cut to the 64 largest by register sorts whenever it may overflow, which
//     raises the bound.
// The waves' lists and sums are joined, then the parts' by the row's last one (a ticket).
// Bound: HBM; the arithmetic (about 10 instructions a logit) takes about half of the time of reading 16-bit logits.
#include "edit_device.hpp"
#include "row_device.hpp"

namespace fs {

constexpr int LP_LIST = LP_TOP + 4 * WAVE; // entries of a wave's list: the largest so far and one group of four per lane

struct LpShared {
    uint64_t list[SK_NW][LP_LIST];
    double sum[SK_NW];
    float max[SK_NW];
    uint32_t above[SK_NW];
    uint32_t last;
};

constexpr float LP_NONE = -__builtin_huge_valf(), LP_LOWEST = -3.402823466e+38f;

// LDS stores and loads of one wave in order
__device__ __forceinline__ void lp_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ float lp_max3(float a, float b, float c) {   // (fmaxf quiets its operands first)
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(a) : "v"(a), "v"(b), "v"(c));
    return a;
}

// The n largest of the cnt entries (whole wave): sorted, one per lane, 0 past them; the list keeps them.
__device__ __forceinline__ uint64_t lp_cut(uint64_t* list, int& cnt, int n) {
    const int lane = lane_id();
    lp_wave_sync();
    uint64_t acc = 0ull;
    for (int i = 0; i < cnt; i += WAVE) acc = merge_top64(acc, sort64<false>(i + lane < cnt ? list[i + lane] : 0ull));
    acc = lane < n ? acc : 0ull;
    lp_wave_sync();
    list[lane] = acc;
    cnt = __popcll(__ballot(acc != 0ull));
    return acc;
}

// The tokens at +inf of a row whose largest logit that is, by one workgroup.
template <int TYPE>
__device__ __forceinline__ double lp_infinite(const LpArgs& a, const EdRow& r, int row, float cap, LpShared& s) {
    double e = 0.0;
    for (int i = threadIdx.x; i < a.V; i += SK_LT) {
        float x = Logits4<TYPE>::one(a.logits, (int64_t)row * a.ld + i);
        if (cap > 0.0f) x = softcap_one(x, cap);
        e += ed_lane(r, x, i) == __builtin_huge_valf() ? 1.0 : 0.0;
    }
    e = wave_allreduce(e, [](double u, double v) { return u + v; });
    if (lane_id() == 0) s.sum[threadIdx.x / WAVE] = e;
    __syncthreads();
    return s.sum[0] + s.sum[1] + s.sum[2] + s.sum[3];
}

// NL: groups of four per thread and chunk. TOP: the n largest are asked for.
template <int TYPE, int NL, bool TOP>
__global__ __launch_bounds__(SK_LT, 4) void logprob_kernel(LpArgs a) {
    constexpr int CHUNK = SK_LT * NL * 4;
    __shared__ __align__(16) LpShared s;
    const int tid = threadIdx.x, lane = lane_id(), w = tid / WAVE;
    const int row = (int)blockIdx.x / a.nseg, part = (int)blockIdx.x - row * a.nseg;
    const int V = a.V;
    using L = Logits4<TYPE>;
    // the part's chunks [c0, c1): the row's, dealt evenly
    const int nchunk = (V + CHUNK - 1) / CHUNK;
    const int c0 = (int)((int64_t)nchunk * part / a.nseg), c1 = (int)((int64_t)nchunk * (part + 1) / a.nseg);
    EdRow r = {nullptr, false, nullptr, nullptr, 0};
    ed_mask(r, a.ed, row, a.err);
    const bool masked = r.words || r.closed;
    typename L::raw raw[NL];
    EdBits bits = {~0u, ~0u};
    auto load = [&](int c) {
        const int lo = c * CHUNK, n_in = V - lo < CHUNK ? V - lo : CHUNK;
        const __amdgpu_buffer_rsrc_t rs = L::rsrc(a.logits, (int64_t)row * a.ld + lo, n_in);
#pragma unroll
        for (int q = 0; q < NL; ++q) raw[q] = L::load(rs, q * SK_LT + tid);
        if (masked) bits = ed_bits<NL>(r, lo, V);
    };
    load(c0);
    __builtin_amdgcn_sched_barrier(0);
    ed_bias(r, a.ed, row);
    float cap = 0.0f, T = 1.0f;
    if (a.params) {
        cap = ld_const(&a.params[row].softcap);
        T = ld_const(&a.params[row].temperature);
        if (!(T > 0.0f)) T = 1.0f;                             // greedy rows: the distribution itself
    }
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    const float c2 = (float)(1.4426950408889634 / (double)T);
    // the chosen token's logit
    const int t = a.tok ? ld_const(a.tok + row) : -1;
    float xt = __builtin_huge_valf();
    if (t >= 0 && t < V) {
        float l = L::one(a.logits, (int64_t)row * a.ld + t);
        if (cap > 0.0f) l = softcap_one(l, cap);
        xt = ed_one(r, l, t);
        if (!(xt > LP_NONE)) xt = __builtin_huge_valf();       // takes no part: nothing to count
    }
    const bool has = xt < __builtin_huge_valf();

    float mx = LP_LOWEST;                                      // the wave's largest logit: its sums' reference
    double sum = 0.0;
    uint32_t above = 0u;                                       // the wave's count
    float bound = 0.0f;                                        // TOP: of the wave's candidates
    bool bounded = false;
    int cnt = 0;
#pragma unroll 1
    for (int c = c0; c < c1; ++c) {
        const int lo = c * CHUNK, n_in = V - lo < CHUNK ? V - lo : CHUNK;
        float x[NL][4];
#pragma unroll
        for (int q = 0; q < NL; ++q) L::floats(raw[q], x[q]);
        const EdBits now = bits;
        if (c + 1 < c1) load(c + 1);
        __builtin_amdgcn_sched_barrier(0);
        if (cap > 0.0f) {
#pragma unroll
            for (int q = 0; q < NL; ++q) softcap_vals(x[q], cap);
        }
        if (r.nb > 0) ed_add<NL>(r, lo, n_in, [&](int q, int c_) -> float& { return x[q][c_]; });
        if (masked) {
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                const uint32_t nib = ed_nibble(now, q);
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) x[q][c_] = ed_keep(x[q][c_], nib, c_, 0xFF800000u);
            }
        }
        if (n_in < CHUNK) {
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) x[q][c_] = (q * SK_LT + tid) * 4 + c_ < n_in ? x[q][c_] : LP_NONE;
        }
        float cm = LP_NONE;                                    // the chunk's largest of the lane
        auto lane_max = [&]() {
            cm = LP_NONE;
#pragma unroll
            for (int q = 0; q < NL; ++q) cm = lp_max3(lp_max3(cm, x[q][0], x[q][1]), x[q][2], x[q][3]);
        };
        auto add = [&]() {
            if (__ballot(cm > mx) != 0ull) {
                const float m = wave_allreduce(cm, fmx);
                sum *= exp(((double)mx - (double)m) / (double)T);
                mx = m;
            }
            float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) e[c_] += __builtin_amdgcn_exp2f((x[q][c_] - mx) * c2);
            return (e[0] + e[1]) + (e[2] + e[3]);
        };
        lane_max();
        float e = add();
        if (__ballot(!(e < __builtin_huge_valf()) || cm != cm) != 0ull) {    // NaN or infinite logits
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) x[q][c_] = x[q][c_] == x[q][c_] ? x[q][c_] : LP_NONE;
            lane_max();
            e = fminf(add(), 1e30f);                           // (the tokens at +inf are counted by themselves)
        }
        sum += (double)e;
        if (has && __ballot(cm > xt) != 0ull) {
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) above += (uint32_t)__popcll(__ballot(x[q][c_] > xt));
        }
        if (TOP) {
            if (!bounded) {                                    // n lanes reach the n-th of their maxima
                const uint32_t srt = sort64_desc_u32(cm > LP_NONE ? key_of(cm) : 0u);
                const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)srt, a.n - 1);
                bounded = key != 0u;
                bound = bounded ? val_of(key) : -3.402823466e+38f;
            }
            if (__ballot(cm >= bound) != 0ull) {
#pragma unroll
                for (int q = 0; q < NL; ++q) {
                    if (__ballot(lp_max3(lp_max3(LP_NONE, x[q][0], x[q][1]), x[q][2], x[q][3]) >= bound) != 0ull) {
                        if (cnt > LP_LIST - 4 * WAVE) {
                            const uint64_t acc = lp_cut(s.list[w], cnt, a.n);
                            const uint32_t key = comp_key(read_lane(acc, a.n - 1));
                            // later ids lose to equal values: the next value up
                            if (key != 0u) {
                                bounded = true;
                                bound = val_of(key + 1u);
                            }
                        }
#pragma unroll
                        for (int c_ = 0; c_ < 4; ++c_) {
                            const uint64_t m = __ballot(x[q][c_] >= bound);
                            if (x[q][c_] >= bound)
                                s.list[w][cnt + (int)mbcnt(m)] =
                                    comp_of(key_of(x[q][c_]), (uint32_t)(lo + (q * SK_LT + tid) * 4 + c_));
                            cnt += __popcll(m);
                        }
                    }
                }
            }
        }
    }
    // ---- the part's end
    auto addu = [](uint32_t u, uint32_t v) { return u + v; };
    auto addf = [](double u, double v) { return u + v; };
    sum = wave_allreduce(sum, addf);
    uint64_t acc = 0ull;
    if (TOP) acc = lp_cut(s.list[w], cnt, a.n);                // (and keeps it in the list)
    if (lane == 0) {
        s.sum[w] = sum; s.max[w] = mx; s.above[w] = above;
    }
    __syncthreads();
    // a sum S relative to m, relative to M >= m instead
    auto to = [&](double S, float m, float M) {
        return m == M || !(M < __builtin_huge_valf()) ? S : S * exp(((double)m - (double)M) / (double)T);
    };
    float M = fmaxf(fmaxf(s.max[0], s.max[1]), fmaxf(s.max[2], s.max[3]));
    double S = wave_allreduce(lane < SK_NW ? to(s.sum[lane & (SK_NW - 1)], s.max[lane & (SK_NW - 1)], M) : 0.0, addf);
    uint32_t ab = s.above[0] + s.above[1] + s.above[2] + s.above[3];
    if (TOP && w == 0) {
#pragma unroll 1
        for (int i = 1; i < SK_NW; ++i) acc = merge_top64(acc, s.list[i][WAVE - 1 - lane]);
    }
    if (a.nseg > 1) {                                          // uniform
        LpPart* pr = a.part + (int64_t)row * a.nseg;
        uint64_t* rl = a.lists + (int64_t)row * a.nseg * LP_TOP;
        if (w == 0) {
            if (TOP) st_agent(&rl[(int64_t)part * LP_TOP + lane], acc);
            if (lane == 0) {
                uint64_t* o = reinterpret_cast<uint64_t*>(pr + part);
                st_agent(o, (uint64_t)__double_as_longlong(S));
                st_agent(o + 1, ((uint64_t)__float_as_uint(M) << 32) | ab);
            }
            vm_drain();                                        // the part's results are out
            if (lane == 0)
                s.last = __hip_atomic_fetch_add(a.ticket + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                         (uint32_t)a.nseg - 1u ? 1u : 0u;
        }
        __syncthreads();
        if (s.last == 0u) return;
        // ---- the row's end, by its last part
        if (tid == 0) __hip_atomic_store(a.ticket + row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (TOP) {                                             // wave w folds lists w, w + SK_NW, ..., then wave 0 the waves'
            acc = 0ull;
            for (int i = w; i < a.nseg; i += SK_NW)
                acc = merge_top64(acc, ld_agent(&rl[(int64_t)i * LP_TOP + WAVE - 1 - lane]));      // ascending
            s.list[w][lane] = acc;
        }
        M = LP_LOWEST;
        S = 0.0;
        ab = 0u;
        for (int i = lane; i < a.nseg; i += WAVE) {            // (a lane's parts, one after another)
            const uint64_t* o = reinterpret_cast<const uint64_t*>(pr + i);
            const uint64_t e = ld_agent(o + 1);
            const double Si = __longlong_as_double((long long)ld_agent(o));
            const float m = __uint_as_float((uint32_t)(e >> 32)), both = fmaxf(m, M);
            S = to(S, M, both) + to(Si, m, both);
            M = both;
            ab += (uint32_t)e;
        }
        const float all = wave_allreduce(M, fmx);
        S = to(S, M, all);
        M = all;
        S = wave_allreduce(S, addf);
        ab = wave_allreduce(ab, addu);
        if (TOP) {
            __syncthreads();
            if (w == 0) {
#pragma unroll 1
                for (int i = 1; i < SK_NW; ++i) acc = merge_top64(acc, s.list[i][WAVE - 1 - lane]);
            }
        }
    }
    if (!(M < __builtin_huge_valf())) {                        // uniform
        __syncthreads();
        S = lp_infinite<TYPE>(a, r, row, cap, s);
    }
    if (w != 0) return;
    const double z = log(S);                                   // (no token takes part: not used)
    auto lp_of = [&](float v) {
        return v > LP_NONE ? (float)((v == M ? 0.0 : ((double)v - (double)M) / (double)T) - z) : LP_NONE;
    };
    if (lane == 0) {
        bool part_of = t >= 0 && t < V;
        float v = LP_NONE;
        if (part_of) {                                         // (+inf counts too: xt stands for "nothing to count" above)
            v = L::one(a.logits, (int64_t)row * a.ld + t);
            if (cap > 0.0f) v = softcap_one(v, cap);
            v = ed_lane(r, v, t);
            part_of = v > LP_NONE;
        }
        if (a.lp) a.lp[row] = part_of ? lp_of(v) : LP_NONE;
        if (a.rank) a.rank[row] = part_of ? (has ? (int)ab + 1 : 1) : 0;
    }
    if (TOP && lane < a.n) {
        if (a.ids) a.ids[(int64_t)row * a.n + lane] = acc != 0ull ? (int)comp_id(acc) : -1;
        if (a.top) a.top[(int64_t)row * a.n + lane] = acc != 0ull ? lp_of(val_of(comp_key(acc))) : LP_NONE;
    }
}

hipError_t launch_logprobs(int type, const LpArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)a.B * a.nseg)), block(SK_LT);
    auto go = [&](auto t, auto top) {
        constexpr int T = decltype(t)::value;
        hipLaunchKernelGGL((logprob_kernel<T, LP_NL(T), decltype(top)::value>), grid, block, 0, st, a);
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
