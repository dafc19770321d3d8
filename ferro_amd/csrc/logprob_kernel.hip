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
//     subtraction, a product, an exponential and an addition a logit. Where a term is 1, a lane's terms are added in fp64:
//     beside a 1, fp32 loses what a near-certain token's log-probability consists of (1 and e^-18 in one lane: 0 for
//     -1.5e-8). 1024 rows of 151936 bf16 with heavy tails, 3.5 such chunks of 19: 62.3 us with fp32 alone, 62.8 so, 64.8
//     with every term in fp64;
//   - a chunk whose sum is NaN (NaN or infinite logits) is added again with NaN left out; once the largest logit is
//     infinite its tokens are counted instead;
//   - the n largest: a bound that n of the wave's 64 lane maxima so far reach (bisected with a compare a step; sorting them
//     takes six times the instructions) passes over chunks without a candidate by one compare a lane; of the others the
//     groups of four with a candidate go to a list in LDS as they are. The list is cut to the n largest tokens by register
//     sorts where it may overflow.
// At the end of a part its waves write out their sums and their tokens at or above the best of their bounds (about 2.5 n in
// a part). One wave of the row's last part (a ticket per part; a row's parts share an XCD and its L2. With one per wave the
// atomics on a line took longer than the reading: 64 rows of 262144 16.8 -> 33.8 us) joins the sums, takes a bound from 256
// maxima of groups of lanes that the waves publish, and sorts the tokens that reach it (about 1.2 n) in registers.
// A chunk's mask is read a chunk ahead of its logits, whose groups of four without an allowed token are not read (the
// part's first chunk is requested whole, at once).
// Bound: HBM, and for 16-bit logits nearly as much the arithmetic (about 10 instructions a logit: four fifths of a busy CU's
// cycles). 1024 rows of 151936 bf16: 57.1 us for the chosen token's alone, 62.9 with n 1 (4.9 TB/s of 311 MB). 64 rows of
// 262144 fp32: 14.8 us, 20.8 with n 5, 24.1 with n 20, and 25.6 with n 20 under masks and biases: the lists and the row's end,
// a chain behind the last read. One row of 65536 with n 5: 8.7 us, of which the read is about 1.
#include "edit_device.hpp"
#include "row_device.hpp"

namespace fs {

constexpr int LP_GROUPS = 256;             // groups of four in a wave's list
constexpr int LP_GROWN = 16;               // groups in a list since its bound was taken, after which it is taken again

struct LpShared {
    float4 gval[SK_NW][LP_GROUPS];         // (the row's end gathers its tokens here)
    int gid[SK_NW][LP_GROUPS];             // the id of a group's first token
    uint64_t kept[SK_NW][LP_TOP];          // what a cut left: sorted, 0 past the entries
    float bound[SK_NW];
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
    const EdList few = ed_list<false>(r);
    const int t = a.tok ? ld_const(a.tok + row) : -1;
    float cap = 0.0f, T = 1.0f;
    if (a.params) {
        cap = ld_const(&a.params[row].softcap);
        T = ld_const(&a.params[row].temperature);
        if (!(T > 0.0f)) T = 1.0f;                             // greedy rows: the distribution itself
    }
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    // Where fp32 holds neither log2 e / T nor what a difference past its range comes to, the terms' arguments are fp64. (T
    // infinite: a c that takes every finite difference to 0, and -inf to -inf)
    const double c2d = fmax(1.4426950408889634 / (double)T, 1e-300);
    const float c2 = (float)c2d;
    const bool far = !(T >= 0x1p-100f && T <= 0x1p100f);
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
        if (few.nb > 0) ed_add<NL, false>(a.ed, row, few, nullptr, lo, n_in, [&](int q, int c_) -> float& { return x[q][c_]; });
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
        auto add = [&]() {                                     // the lane's terms
            if (__ballot(cm >= mx) != 0ull || far) {           // one of them is 1 (the first chunk, and few others)
                float m = wave_allreduce(cm, fmx);
                if (__ballot(m > mx) != 0ull) {
                    if (__ballot(sum != 0.0) != 0ull)
                        sum *= m < __builtin_huge_valf() ? exp(((double)mx - (double)m) / (double)T) : 0.0;
                    mx = m;
                }
                m = mx;
                asm volatile("" : "+v"(m));                    // (differences shared with the other branch are spilled)
                double d[2] = {0.0, 0.0};
                if (far) {
#pragma unroll
                    for (int q = 0; q < NL; ++q) {
#pragma unroll
                        for (int c_ = 0; c_ < 4; ++c_)
                            d[c_ & 1] += (double)__builtin_amdgcn_exp2f((float)(((double)x[q][c_] - (double)m) * c2d));
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    return d[0] + d[1];
                }
                if constexpr (NL > 4) {
                    // a lane's logits by their place in the group: eight terms in fp64 only where one of them is 1 (1024 rows
                    // of 151936 bf16: 62.8 us; with all in fp64 64.2, as in the shorter chunks of fp32 rows, where that is
                    // the faster: 64 rows of 262144 25.6 us, by place 25.9)
#pragma unroll
                    for (int c_ = 0; c_ < 4; ++c_) {
                        float most = lp_max3(x[0][c_], x[1][c_], x[2][c_]);
#pragma unroll
                        for (int q = 3; q < NL; q += 2) most = lp_max3(most, x[q][c_], x[q + 1 < NL ? q + 1 : q][c_]);
                        if (__ballot(most == m) != 0ull) {
#pragma unroll
                            for (int q = 0; q < NL; ++q) {
                                d[q & 1] += (double)__builtin_amdgcn_exp2f((x[q][c_] - m) * c2);
                                if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                            }
                        } else {
                            float e[2] = {0.0f, 0.0f};
#pragma unroll
                            for (int q = 0; q < NL; ++q) {
                                e[q & 1] += __builtin_amdgcn_exp2f((x[q][c_] - m) * c2);
                                if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                            }
                            d[c_ & 1] += (double)(e[0] + e[1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < NL; ++q) {
#pragma unroll
                        for (int c_ = 0; c_ < 4; ++c_) d[c_ & 1] += (double)__builtin_amdgcn_exp2f((x[q][c_] - m) * c2);
                        __builtin_amdgcn_sched_barrier(0);     // (all exponentials at once need more registers)
                    }
                }
                return d[0] + d[1];
            }
            float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < NL; ++q) {
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) e[c_] += __builtin_amdgcn_exp2f((x[q][c_] - mx) * c2);
                __builtin_amdgcn_sched_barrier(0);
            }
            return (double)((e[0] + e[1]) + (e[2] + e[3]));
        };
        lane_max();
        double e = add();
        if (__ballot(!(e < __builtin_huge_val()) || cm != cm) != 0ull) {    // NaN or infinite logits
#pragma unroll
            for (int q = 0; q < NL; ++q)
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) x[q][c_] = x[q][c_] == x[q][c_] ? x[q][c_] : LP_NONE;
            lane_max();
            e = add();
            if (!(mx < __builtin_huge_valf())) {
                float ones = 0.0f;
#pragma unroll
                for (int q = 0; q < NL; ++q)
#pragma unroll
                    for (int c_ = 0; c_ < 4; ++c_) ones += x[q][c_] == mx ? 1.0f : 0.0f;
                e = (double)ones;
            }
        }
        sum += e;
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
    // ---- the wave's end
    auto addu = [](uint32_t u, uint32_t v) { return u + v; };
    auto addf = [](double u, double v) { return u + v; };
    const int lists = nseg * SK_NW, me = part * SK_NW + w;
    char* rw = a.rows + (int64_t)row * (int64_t)lp_row_bytes(nseg);
    uint32_t* ticket = a.ticket + (int64_t)row * LP_LINE;
    double* p_sum = reinterpret_cast<double*>(rw);
    float* p_max = reinterpret_cast<float*>(p_sum + lists);
    uint32_t* p_above = reinterpret_cast<uint32_t*>(p_max + lists);
    float* p_bound = reinterpret_cast<float*>(p_above + lists);
    int* p_cnt = reinterpret_cast<int*>(p_bound + lists);
    uint32_t* p_key = reinterpret_cast<uint32_t*>(p_cnt + lists);
    uint64_t* rl = a.lists + (int64_t)row * lists * LP_TOP;
    sum = wave_allreduce(sum, addf);
    if (TOP) {                                                 // the wave's tokens that reach the best of the part's bounds
        if (lane == 0) s.bound[w] = reach;
        __syncthreads();
        reach = fmaxf(fmaxf(s.bound[0], s.bound[1]), fmaxf(s.bound[2], s.bound[3]));
        uint64_t* out = rl + me * LP_TOP;
        int cnt = 0;
        bool fits = !cut;
#pragma unroll 1
        for (int i = 0; fits && i < g; i += WAVE) {
            const bool in = i + lane < g;
            const float4 v = in ? s.gval[w][i + lane] : make_float4(LP_NONE, LP_NONE, LP_NONE, LP_NONE);
            const uint32_t id = in ? (uint32_t)s.gid[w][i + lane] : 0u;
            const float y[4] = {v.x, v.y, v.z, v.w};
            uint64_t m[4];
            int all = cnt;
#pragma unroll
            for (int c_ = 0; c_ < 4; ++c_) {
                m[c_] = __ballot(y[c_] >= reach);
                all += __popcll(m[c_]);
            }
            fits = all <= LP_TOP;
            if (fits) {
#pragma unroll
                for (int c_ = 0; c_ < 4; ++c_) {
                    if (y[c_] >= reach) out[cnt + (int)mbcnt(m[c_])] = comp_of(key_of(y[c_]), id + (uint32_t)c_);
                    cnt += __popcll(m[c_]);
                }
            }
        }
        if (!fits) {                                           // a list that was cut, or equal logits at the bound
            const uint64_t e = lp_cut(s, g, cut, reach, n);
            cnt = __popcll(__ballot(e != 0ull));
            if (lane < cnt) out[lane] = e;
        }
        uint32_t top = lm > LP_NONE ? key_of(lm) : 0u;
        auto both = [](uint32_t u, uint32_t v) { return u > v ? u : v; };
        top = both(top, xor_lane32<1>(top));
        top = both(top, xor_lane32<2>(top));
        if (nseg > 4) top = both(top, xor_lane32<4>(top));
        if (nseg > 8) top = both(top, xor_lane32<8>(top));
        if (nseg > 16) top = both(top, xor_lane32<16>(top));
        if (nseg > 32) top = both(top, xor_lane32<32>(top));
        const int lg = lp_group(nseg);
        if ((lane & ((1 << lg) - 1)) == 0) p_key[((me << 6) + lane) >> lg] = top;
        if (lane == 0) {
            p_cnt[me] = cnt;
            p_bound[me] = reach;
        }
    }
    uint32_t turn = 0u;
    if (lane == 0) {
        p_sum[me] = sum;
        p_max[me] = mx;
        p_above[me] = above;
    }
    vm_drain();                                                // the wave's results are in the L2
    __syncthreads();
    if (w != 0) return;
    if (lane == 0) turn = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (read_lane(turn, 0) != (uint32_t)nseg - 1u) return;
    // ---- the row's end, by its last part's first wave
    if (lane == 0) *ticket = 0u;
    constexpr int LL = LP_PARTS * SK_NW / WAVE;                // waves' results per lane
    double si[LL];
    float mi[LL], bi[LL];
    uint32_t key[LL], ab = 0u;
    int len[LL];
#pragma unroll
    for (int u = 0; u < LL; ++u) {
        const int i = u * WAVE + lane;
        const bool in = i < lists;
        si[u] = in ? p_sum[i] : 0.0;
        mi[u] = in ? p_max[i] : LP_LOWEST;
        ab += in ? p_above[i] : 0u;
        if (TOP) {
            bi[u] = in ? p_bound[i] : LP_LOWEST;
            len[u] = in ? p_cnt[i] : 0;
            key[u] = i < (lists << 6) >> lp_group(nseg) ? p_key[i] : 0u;
        }
    }
    // TOP: the tokens' lists. Half a wave reads a list, sixteen lists in flight; the first of them behind the sums
    constexpr int U = 8, ROOM = sizeof(s.gval) / sizeof(uint64_t);
    static_assert(4 * U * WAVE <= ROOM, "a batch fits behind what has to be sorted first");
    const int half = lane >> 5, pos = lane & 31;
    int* at = s.gid[0];                                        // [LP_PARTS * SK_NW] lists: number, length
    uint64_t* join = reinterpret_cast<uint64_t*>(&s.gval[0][0]);
    uint32_t least = 0u;
    int k = 0, to[U];
    uint64_t e[U];
    auto fetch = [&](int i0, int skip) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + 2 * u + half;
            to[u] = i < k ? at[i] : 0;
            e[u] = pos + skip < (to[u] & 255) ? rl[(to[u] >> 8) * LP_TOP + pos + skip] : 0ull;
        }
    };
    if (TOP) {
        float best = LP_LOWEST;
#pragma unroll
        for (int u = 0; u < LL; ++u) best = fmaxf(best, bi[u]);
        best = wave_allreduce(best, fmx);
        least = lp_nth(key, key_of(best), n);
        // of waves whose largest logit reaches the bound (about 17 of 64 for n = 20; reading all of them took 3 us)
#pragma unroll
        for (int u = 0; u < LL; ++u) {
            const bool in = len[u] > 0 && key_of(mi[u]) >= least;
            const uint64_t m = __ballot(in);
            if (in) at[k + (int)mbcnt(m)] = ((u * WAVE + lane) << 8) | len[u];
            k += __popcll(m);
        }
        lp_wave_sync();
        fetch(0, 0);
    }
    float M = LP_LOWEST;
#pragma unroll
    for (int u = 0; u < LL; ++u) M = fmaxf(M, mi[u]);
    M = wave_allreduce(M, fmx);
    double S = 0.0;
#pragma unroll
    for (int u = 0; u < LL; ++u) {                             // relative to the row's maximum
        if (u * WAVE >= lists) break;                          // uniform
        S += mi[u] == M ? si[u] : M < __builtin_huge_valf() ? si[u] * exp(((double)mi[u] - (double)M) / (double)T) : 0.0;
    }
    S = wave_allreduce(S, addf);
    ab = wave_allreduce(ab, addu);
    const double z = log(S);                                   // (no token takes part: not used)
    auto lp_of = [&](float v) {
        if (!(v > LP_NONE) || (v < M && !(M < __builtin_huge_valf()))) return LP_NONE;
        return (float)((v == M ? 0.0 : ((double)v - (double)M) / (double)T) - z);
    };
    if (lane == 0) {
        if (a.lp) a.lp[row] = lp_of(xv);
        if (a.rank) a.rank[row] = xv > LP_NONE ? (has ? (int)ab + 1 : 1) : 0;
    }
    if (TOP) {
        // the tokens that reach the bound, gathered in LDS
        int cnt = 0;
        uint64_t acc = 0ull;
        bool sorted = false;
        auto gather = [&]() {                                  // (0: no token; the bound is above it)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = comp_key(e[u]) >= least;
                const uint64_t m = __ballot(in);
                if (in) join[cnt + (int)mbcnt(m)] = e[u];
                cnt += __popcll(m);
            }
        };
#pragma unroll 1
        for (int i0 = 0; i0 < k; i0 += 2 * U) {
            if (i0 > 0) fetch(i0, 0);
            gather();
            bool more = false;                                 // lists of more than 32
#pragma unroll
            for (int u = 0; u < U; ++u) more |= (to[u] & 255) > 32;
            if (__ballot(more) != 0ull) {
                fetch(i0, 32);
                gather();
            }
            lp_wave_sync();
            const bool last = i0 + 2 * U >= k;
            if (last && !sorted && cnt <= WAVE) {              // ranks: an eighth of a sort's instructions
                const uint64_t c = lane < cnt ? join[lane] : 0ull;
                int r = 0;
#pragma unroll 4
                for (int i = 0; i < cnt; ++i) r += join[i] > c ? 1 : 0;
                lp_wave_sync();
                join[lane] = 0ull;
                lp_wave_sync();
                if (c != 0ull) join[r] = c;
                lp_wave_sync();
                acc = join[lane];
            } else if (last || cnt > 2 * U * WAVE) {
#pragma unroll 1
                for (int i = 0; i < cnt; i += WAVE)
                    acc = merge_top64(acc, sort64<false>(i + lane < cnt ? join[i + lane] : 0ull));
                cnt = 0;
                sorted = true;
                lp_wave_sync();
            }
        }
        if (lane < n) {
            if (a.ids) a.ids[(int64_t)row * n + lane] = acc != 0ull ? (int)comp_id(acc) : -1;
            if (a.top) a.top[(int64_t)row * n + lane] = acc != 0ull ? lp_of(val_of(comp_key(acc))) : LP_NONE;
        }
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
