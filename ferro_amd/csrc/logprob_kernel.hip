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
//   - the n largest: a bound that n of the wave's 64 lane maxima so far reach (bisected with a compare a step; sorting them
//     takes six times the instructions) passes over chunks without a candidate by one compare a lane; of the others the
//     groups of four with a candidate go to a list in LDS as they are. The list is cut to the n largest tokens by register
//     sorts where it may overflow.
// At the end of a part its waves write out their tokens at or above the best of their bounds (about 2.5 n in a part). The
// row's last part (a ticket; a row's parts share an XCD and its L2) joins the parts' sums, takes a bound from 256 maxima
// of groups of lanes that the parts publish, and ranks the tokens that reach it (about 1.2 n).
// A chunk's mask is read a chunk ahead of its logits, whose groups of four without an allowed token are not read (the
// part's first chunk is requested whole, at once).
// Bound: HBM; the arithmetic (about 10 instructions a logit) takes about half of the time of reading 16-bit logits.
#include "edit_device.hpp"
#include "row_device.hpp"

namespace fs {

constexpr int LP_GROUPS = 256;             // groups of four in a wave's list
constexpr int LP_JOIN = 1024;              // entries that are ranked at once
constexpr int LP_GROWN = 16;               // groups in a list since its bound was taken, after which it is taken again

struct LpShared {
    float4 gval[SK_NW][LP_GROUPS];
    int gid[SK_NW][LP_GROUPS];             // the id of a group's first token
    uint64_t kept[SK_NW][LP_TOP];          // what a cut left: sorted, 0 past the entries
    uint64_t join[LP_JOIN];
    uint64_t top[LP_TOP];
    uint32_t rank[SK_LT];
    double sum[SK_NW];
    float max[SK_NW];
    float bound[SK_NW];
    uint32_t above[SK_NW];
    int cnt[SK_NW];
    uint32_t n, last;
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

// A key that n of the wave's 64 K keys reach, and about a quarter more at most where they differ; n reach `lo` already.
// Bisected: K compares a step.
template <int K>
__device__ __forceinline__ uint32_t lp_nth(const uint32_t (&key)[K], uint32_t lo, int n) {
    uint32_t hi = key[0];
#pragma unroll
    for (int u = 1; u < K; ++u) hi = key[u] > hi ? key[u] : hi;
    hi = wave_max(hi);
    if (n == 1) return hi > lo ? hi : lo;
    uint32_t step = hi > lo ? hi - lo : 0u;                    // the n-th largest lies in [lo, lo + step]
#pragma unroll 1
    while (step > 0u) {
        const uint32_t up = (step >> 1) + (step & 1u);
        int c = 0;
#pragma unroll
        for (int u = 0; u < K; ++u) c += __popcll(__ballot(key[u] >= lo + up));
        if (c >= n) {
            lo += up;
            step -= up;
            if (c <= n + n / 4) break;
        } else {
            step = up - 1u;
        }
    }
    return lo;
}

// What the wave keeps of its list of g groups and an earlier cut: its n largest tokens at or above the bound, sorted, one
// per lane, 0 past them (also in s.kept).
__device__ __forceinline__ uint64_t lp_cut(LpShared& s, int& g, bool& cut, float bound, int n) {
    const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
    lp_wave_sync();
    uint64_t acc = cut ? s.kept[w][lane] : 0ull;
#pragma unroll 1
    for (int i = 0; i < 4 * g; i += WAVE) {                    // sixteen groups at a time
        const int at = (i + lane) >> 2;
        const float x = at < g ? reinterpret_cast<const float*>(&s.gval[w][at])[lane & 3] : LP_NONE;
        acc = merge_top64(acc, sort64<false>(x >= bound ? comp_of(key_of(x), (uint32_t)(s.gid[w][at] + (lane & 3))) : 0ull));
    }
    acc = lane < n ? acc : 0ull;
    lp_wave_sync();
    s.kept[w][lane] = acc;
    g = 0;
    cut = true;
    return acc;
}

// Lanes whose logits a part publishes the largest of.
__device__ __forceinline__ int lp_group(int nseg) {
    return nseg <= 4 ? 4 : nseg <= 8 ? 8 : nseg <= 16 ? 16 : nseg <= 32 ? 32 : 64;
}

// The n largest of the cnt distinct entries in[0, cnt), sorted to s.top, which is zero before. Whole workgroup, after a
// barrier; ends with one.
__device__ __forceinline__ void lp_rank(const uint64_t* in, int cnt, LpShared& s, int n) {
    if (cnt <= SK_LT) {
        sk_rank(in, s.rank, cnt, [&](uint32_t r, uint64_t c) { if (r < (uint32_t)n) s.top[r] = c; });
    } else {
        for (int c = threadIdx.x; c < cnt; c += SK_LT) {
            const uint64_t me = in[c];
            uint32_t r = 0u;
            for (int j = 0; j < cnt; ++j) r += in[j] > me ? 1u : 0u;
            if (r < (uint32_t)n) s.top[r] = me;
        }
    }
    __syncthreads();
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

// The kernel's argument list as a struct: the argument segment follows the same layout rules
struct LpKernargs {
    const void* logits;
    int64_t ld;
    int B, V, nseg, n;
    LpArgs a;
};

// NL: groups of four per thread and chunk. TOP: the n largest are asked for.
template <int TYPE, int NL, bool TOP>
__global__ __launch_bounds__(SK_LT, 4) void logprob_kernel(const void* logits, int64_t ld, int B, int V, int nseg, int n,
                                                           LpArgs a_) {
    constexpr int CHUNK = SK_LT * NL * 4;
    __shared__ __align__(16) LpShared s;
    const int tid = threadIdx.x, lane = lane_id(), w = tid / WAVE;
    // a row's parts are consecutive workgroups of one index class mod XCDS, as in the small-k kernel
    const int j = (int)(blockIdx.x / (unsigned)XCDS);
    const int q_row = __builtin_amdgcn_readfirstlane(j / nseg);
    const int part = j - q_row * nseg;
    const int row = (int)(blockIdx.x % (unsigned)XCDS) + XCDS * q_row;
    if (row >= B) return;
    using L = Logits4<TYPE>;
    // the part's chunks [c0, c1): the row's, dealt evenly
    const int nchunk = (V + CHUNK - 1) / CHUNK;
    const int c0 = (int)((int64_t)nchunk * part / nseg), c1 = (int)((int64_t)nchunk * (part + 1) / nseg);
    typename L::raw raw[NL];
    auto load = [&](int c, bool skip, const EdBits& bits) {
        const int lo = c * CHUNK, n_in = V - lo < CHUNK ? V - lo : CHUNK;
        const __amdgpu_buffer_rsrc_t rs = L::rsrc(logits, (int64_t)row * ld + lo, n_in);
#pragma unroll
        for (int q = 0; q < NL; ++q) {
            int at = q * SK_LT + tid;
            if (skip) at = ed_nibble(bits, q) != 0u ? at : 0x07ffffff;       // (past the buffer: no read, zeros)
            raw[q] = L::load(rs, at);
        }
    };
    EdBits bits = {~0u, ~0u}, next = bits;                     // of the chunk in raw; of the one after it
    load(c0, false, bits);
    __builtin_amdgcn_sched_barrier(0);
    const __attribute__((address_space(4))) char* kseg =       // (as in the small-k kernel: no argument is read earlier)
        (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(kseg) : : "memory");
    const LpArgs& a = *(const LpArgs*)(kseg + offsetof(LpKernargs, a));
    (void)a_;
    EdRow r = {nullptr, false, nullptr, nullptr, 0};
    ed_mask(r, a.ed, row, a.err);
    const bool masked = r.words || r.closed;
    if (masked) {
        bits = ed_bits<NL>(r, c0 * CHUNK, V);
        if (c0 + 1 < c1) next = ed_bits<NL>(r, (c0 + 1) * CHUNK, V);
    }
    ed_bias(r, a.ed, row);
    const EdList few = ed_list(r);
    const int t = a.tok ? ld_const(a.tok + row) : -1;
    float cap = 0.0f, T = 1.0f;
    if (a.params) {
        cap = ld_const(&a.params[row].softcap);
        T = ld_const(&a.params[row].temperature);
        if (!(T > 0.0f)) T = 1.0f;                             // greedy rows: the distribution itself
    }
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    const float c2 = (float)(1.4426950408889634 / (double)T);
    // the chosen token's logit (NaN: it takes no part), and what the others are compared with
    float xv = __builtin_nanf("");
    if (t >= 0 && t < V) {
        xv = L::one(logits, (int64_t)row * ld + t);
        if (cap > 0.0f) xv = softcap_one(xv, cap);
        xv = ed_one(r, few, xv, t);
        xv = xv > LP_NONE ? xv : __builtin_nanf("");
    }
    const bool has = xv < __builtin_huge_valf();               // (none is larger than +inf)

    float mx = LP_LOWEST;                                      // the wave's largest logit: its sums' reference
    double sum = 0.0;
    uint32_t above = 0u;                                       // the wave's count
    // TOP: the bound of new candidates; what n logits of the wave reach; the lane's largest logit
    float bound = LP_LOWEST, reach = LP_LOWEST, lm = LP_NONE;
    int g = 0, bound_at = -LP_GROWN;                           // groups in the list, and when the bound was taken
    bool cut = false;
    if (TOP) {
        if (tid == 0) s.n = 0u;
        if (tid < LP_TOP) s.top[tid] = 0ull;
    }
#pragma unroll 1
    for (int c = c0; c < c1; ++c) {
        const int lo = c * CHUNK, n_in = V - lo < CHUNK ? V - lo : CHUNK;
        float x[NL][4];
#pragma unroll
        for (int q = 0; q < NL; ++q) L::floats(raw[q], x[q]);
        const EdBits now = bits;
        bits = next;
        if (c + 1 < c1) load(c + 1, masked, bits);
        if (masked && c + 2 < c1) next = ed_bits<NL>(r, (c + 2) * CHUNK, V);
        __builtin_amdgcn_sched_barrier(0);
        if (cap > 0.0f) {
#pragma unroll
            for (int q = 0; q < NL; ++q) softcap_vals(x[q], cap);
        }
        if (r.nb > 0) ed_add<NL>(r, &few, lo, n_in, [&](int q, int c_) -> float& { return x[q][c_]; });
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
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) e[c_] += __builtin_amdgcn_exp2f((x[q][c_] - mx) * c2);
                __builtin_amdgcn_sched_barrier(0);             // (all exponentials at once need more registers)
            }
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
        if (has && __ballot(cm > xv) != 0ull) {
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) above += (uint32_t)__popcll(__ballot(x[q][c_] > xv));
        }
        if (TOP) {
            lm = fmaxf(lm, cm);
            const bool any = __ballot(cm >= bound) != 0ull;
            if (any && g - bound_at >= LP_GROWN) {
                const uint32_t key[1] = {key_of(lm)};
                uint32_t from = wave_min(key[0]);              // (every lane reaches it)
                from = reach > LP_LOWEST && from < key_of(reach) ? key_of(reach) : from;
                const uint32_t nth = lp_nth(key, from, n);
                const float b = nth > 0x007FFFFFu ? val_of(nth) : LP_LOWEST;
                bound = fmaxf(bound, b);
                reach = fmaxf(reach, b);
                bound_at = b > LP_LOWEST ? g : bound_at;
            }
            if (any) {
#pragma unroll
                for (int q = 0; q < NL; ++q) {
                    const bool mine = lp_max3(lp_max3(LP_NONE, x[q][0], x[q][1]), x[q][2], x[q][3]) >= bound;
                    const uint64_t m = __ballot(mine);
                    if (m != 0ull) {
                        if (mine) {
                            const int at = g + (int)mbcnt(m);
                            s.gval[w][at] = make_float4(x[q][0], x[q][1], x[q][2], x[q][3]);
                            s.gid[w][at] = lo + (q * SK_LT + tid) * 4;
                        }
                        g += __popcll(m);
                        if (g > LP_GROUPS - WAVE) {
                            const uint32_t key = comp_key(read_lane(lp_cut(s, g, cut, bound, n), n - 1));
                            if (key != 0u) {
                                reach = val_of(key);
                                bound = val_of(key + 1u);      // later ids lose to equal values: the next value up
                            }
                            bound_at = 0;
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
    if (lane == 0) {
        s.sum[w] = sum; s.max[w] = mx; s.above[w] = above; s.bound[w] = reach;
    }
    __syncthreads();
    // a sum S relative to m, relative to M >= m instead
    auto to = [&](double S, float m, float M) {
        return m == M || !(M < __builtin_huge_valf()) ? S : S * exp(((double)m - (double)M) / (double)T);
    };
    float M = fmaxf(fmaxf(s.max[0], s.max[1]), fmaxf(s.max[2], s.max[3]));
    double S = wave_allreduce(lane < SK_NW ? to(s.sum[lane & (SK_NW - 1)], s.max[lane & (SK_NW - 1)], M) : 0.0, addf);
    uint32_t ab = s.above[0] + s.above[1] + s.above[2] + s.above[3];
    float best = LP_LOWEST;
    if (TOP) {                                                 // the wave's tokens that reach the best of the bounds
        best = fmaxf(fmaxf(s.bound[0], s.bound[1]), fmaxf(s.bound[2], s.bound[3]));
        uint64_t* out = nseg > 1 ? a.lists + (((int64_t)row * nseg + part) * SK_NW + w) * LP_TOP : &s.join[w * LP_TOP];
        int cnt = 0;
        bool fits = !cut;
        for (int i = lane; fits && i - lane < 4 * g; i += WAVE) {
            const float x = i < 4 * g ? reinterpret_cast<const float*>(&s.gval[w][i >> 2])[i & 3] : LP_NONE;
            const uint64_t m = __ballot(x >= best);
            fits = cnt + __popcll(m) <= LP_TOP;
            if (fits && x >= best) out[cnt + (int)mbcnt(m)] = comp_of(key_of(x), (uint32_t)(s.gid[w][i >> 2] + (i & 3)));
            cnt += __popcll(m);
        }
        if (!fits) {                                           // a list that was cut, or equal logits at the bound
            const uint64_t e = lp_cut(s, g, cut, best, n);
            cnt = __popcll(__ballot(e != 0ull));
            if (lane < cnt) out[lane] = e;
        }
        // the largest logits of the part's groups of `size` lanes: 256 in a row of up to 64 parts
        if (nseg > 1) {
            uint32_t top = lm > LP_NONE ? key_of(lm) : 0u;
            auto both = [](uint32_t u, uint32_t v) { return u > v ? u : v; };
            top = both(top, xor_lane32<1>(top));
            top = both(top, xor_lane32<2>(top));
            if (nseg > 4) top = both(top, xor_lane32<4>(top));
            if (nseg > 8) top = both(top, xor_lane32<8>(top));
            if (nseg > 16) top = both(top, xor_lane32<16>(top));
            if (nseg > 32) top = both(top, xor_lane32<32>(top));
            const int size = lp_group(nseg);
            if (lane % size == 0) a.part[(int64_t)row * nseg + part].key[(w * WAVE + lane) / size] = top;
        }
        if (lane == 0) s.cnt[w] = cnt;
        if (lane == 0 && nseg > 1) a.part[(int64_t)row * nseg + part].cnt[w] = cnt;
    }
    if (nseg > 1) {                                            // uniform
        LpPart* pr = a.part + (int64_t)row * nseg;
        if (tid == 0) {
            pr[part].sum = S;
            pr[part].above = ab;
            pr[part].max = M;
            pr[part].bound = best;
        }
        vm_drain();                                            // the wave's results are in the L2
        if (TOP) __syncthreads();
        if (tid == 0)
            s.last = __hip_atomic_fetch_add(a.ticket + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) ==
                     (uint32_t)nseg - 1u ? 1u : 0u;
        __syncthreads();
        if (s.last == 0u) return;
        // ---- the row's end, by its last part
        if (tid == 0) a.ticket[row] = 0u;
        const bool is = lane < nseg;
        const double si = is ? pr[lane].sum : 0.0;
        const float mi = is ? pr[lane].max : LP_LOWEST, bi = is ? pr[lane].bound : LP_LOWEST;
        const uint32_t ai = is ? pr[lane].above : 0u;
        if (TOP) {
            // per = SK_LT / (waves' lists, rounded up) threads for each list; its first entries with its length
            constexpr int U = 4;
            const int lists = nseg * SK_NW;
            int per = 1;
            while (2 * per * lists <= SK_LT) per *= 2;
            const int l = tid / per, k0 = tid % per;
            const uint64_t* rl = a.lists + ((int64_t)row * lists + l) * LP_TOP;
            uint64_t e[U] = {0ull, 0ull, 0ull, 0ull};
            int len = 0;
            if (l < lists) {
                len = pr[l / SK_NW].cnt[l % SK_NW];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (k0 + u * per < LP_TOP) e[u] = rl[k0 + u * per];
            }
            const int kp = SK_LT / lp_group(nseg);             // keys of a part
            uint32_t key[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = u * WAVE + lane;
                key[u] = i < nseg * kp ? pr[i / kp].key[i % kp] : 0u;
            }
            best = wave_allreduce(bi, fmx);
            const uint32_t least = lp_nth(key, key_of(best), n);
            auto join = [&](uint64_t c, bool in) {
                if (in && comp_key(c) >= least) {
                    const uint32_t at = atomicAdd(&s.n, 1u);
                    if (at < (uint32_t)LP_JOIN) s.join[at] = c;
                }
            };
#pragma unroll
            for (int u = 0; u < U; ++u) join(e[u], k0 + u * per < len);
            for (int k = k0 + U * per; k < len; k += per) join(rl[k], true);
            __syncthreads();
            if (s.n > (uint32_t)LP_JOIN) {                     // equal logits at the bound: one wave sorts the lists
                if (w == 0) {
                    uint64_t acc = 0ull;
                    for (int i = 0; i < lists; ++i) {
                        const int c = pr[i / SK_NW].cnt[i % SK_NW];
                        acc = merge_top64(acc, sort64<false>(
                            lane < c ? a.lists[((int64_t)row * lists + i) * LP_TOP + lane] : 0ull));
                    }
                    s.top[lane] = lane < n ? acc : 0ull;
                }
                __syncthreads();
            } else {
                lp_rank(s.join, (int)s.n, s, n);
            }
        }
        M = wave_allreduce(mi, fmx);
        S = wave_allreduce(to(si, mi, M), addf);
        ab = wave_allreduce(ai, addu);
    } else if (TOP) {                                          // the waves' lists close up
        __syncthreads();
        int base = 0, all = 0;
#pragma unroll
        for (int q = 0; q < SK_NW; ++q) {
            base += q < w ? s.cnt[q] : 0;
            all += s.cnt[q];
        }
        uint64_t* list = s.join + SK_NW * LP_TOP;
        if (lane < s.cnt[w]) list[base + lane] = s.join[w * LP_TOP + lane];
        __syncthreads();
        lp_rank(list, all, s, n);
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
        if (a.lp) a.lp[row] = lp_of(xv);
        if (a.rank) a.rank[row] = xv > LP_NONE ? (has ? (int)ab + 1 : 1) : 0;
    }
    if (TOP && lane < n) {
        const uint64_t acc = s.top[lane];
        if (a.ids) a.ids[(int64_t)row * n + lane] = acc != 0ull ? (int)comp_id(acc) : -1;
        if (a.top) a.top[(int64_t)row * n + lane] = acc != 0ull ? lp_of(val_of(comp_key(acc))) : LP_NONE;
    }
}

hipError_t launch_logprobs(int type, const LpArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((int64_t)XCDS * a.nseg * (((int64_t)a.B + XCDS - 1) / XCDS))), block(SK_LT);
    auto go = [&](auto t, auto top) {
        constexpr int T = decltype(t)::value;
        hipLaunchKernelGGL((logprob_kernel<T, LP_NL(T), decltype(top)::value>), grid, block, 0, st, a.logits, a.ld, a.B,
                           a.V, a.nseg, a.n, a);
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
