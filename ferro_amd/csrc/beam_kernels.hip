// beam_kernels.hip - beam search: histories and model states that follow their beams (the selection: logprob_kernel.hip,
// beam_device.hpp).
#include "sampler_device.hpp"
#include "sampler_launch.hpp"

#include <type_traits>

namespace fs {

// ------------------------------------------------------------------------------------------------ histories
// Beam j of stream s (row s n + j) gets the history of the stream's beam parent[s n + j] and the token behind it.
// One launch where the rows' offsets fit a workgroup's LDS: every workgroup sums the lengths itself (three dependent loads a
// row, from the L2) and copies an equal share of the new ids, four per thread at a time, whose rows it finds by bisection among
// those of its share. More rows: a launch for the offsets first, which the copying one then reads. The new ids are stored past
// the caches (256 histories of 32768 ids: 14.2 -> 13.1 us).
// Bound: latency for few ids (4.5 us for 4 histories of 300, 6.2 for 512 of 2048), then HBM: 256 of 32768 13.3 us (4.9 TB/s of
// 65 MB). In two launches latency throughout: 4096 of 16 and of 500 ids 18.5 and 19.3 us, 16384 29.6 and 56 (its 55 MB: 11.6).
constexpr int FK_T = 256;
// Rows whose offsets are kept in LDS. 1032 rows of 500 ids with 512, 1024, 2048: 12.8, 12.9, 7.2 us, 1024 12.3, 6.9, 7.2; but 16384
// 60, 56, 63 (the offsets' launch takes FK_PER rows per thread).
constexpr int FK_ROWS = 1024;
constexpr int FK_STEP = FK_T * 4;          // ids a workgroup copies at a time
constexpr int FK_U = 4;                    // of these in flight
// Workgroups per CU. 512 histories of 2048 ids with 1, 2, 4, 8, 16: 12.5, 9.1, 7.4, 6.2, 6.2 us; 256 of 32768 25.5, 17.3, 14.1,
// 13.3, 13.7.
constexpr int FK_PER_CU = 8;

struct ForkRow {
    int64_t at, len;                                           // its parent's ids
    int add;                                                   // 1: a token behind them
};
// (without branches: several rows' loads are in flight together)
struct ForkFrom {
    int64_t r0;
    int rows, p;
};
__device__ __forceinline__ ForkFrom fork_from(const ForkArgs& a, int o) {
    const int s = o / a.n;
    ForkFrom f;
    f.r0 = a.row_off ? a.row_off[s] : (int64_t)s * a.n;
    f.rows = a.row_off ? (int)(a.row_off[s + 1] - f.r0) : a.n;
    f.p = a.parent[o];
    return f;
}
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, const ForkFrom& f, bool& bad) {
    const bool on = f.p >= 0 && f.p < f.rows;
    bad |= f.p >= f.rows;
    const int64_t* off = a.hist_off + f.r0 + (on ? f.p : 0);
    ForkRow r;
    r.at = off[0];
    r.len = off[on ? 1 : 0] - r.at;
    r.add = on && a.tok ? 1 : 0;
    return r;
}

constexpr int FK_PER = FK_ROWS / FK_T;     // rows per thread of a scan

// The rows' new offsets by NT threads, FK_PER consecutive rows per thread at most at a time: each(row, its first id, its length,
// its parent's first id). Returns the end. Whole workgroup.
template <int NT, class Each>
__device__ __forceinline__ int64_t fork_scan(const ForkArgs& a, bool& bad, Each each) {
    __shared__ int64_t wave[NT / WAVE];
    const int tid = threadIdx.x, lane = lane_id(), w = tid / WAVE, R = a.S * a.n;
    int64_t carry = 0;
#pragma unroll 1
    for (int c = 0; c < R; c += NT * FK_PER) {
        const int left = R - c < NT * FK_PER ? R - c : NT * FK_PER, per = (left + NT - 1) / NT;
        ForkFrom from[FK_PER];
        ForkRow f[FK_PER];
        int64_t mine = 0;
#pragma unroll
        for (int q = 0; q < FK_PER; ++q) {                     // (past the last row: the last one again)
            const int o = tid * per + q;
            if (q < per) from[q] = fork_from(a, c + (o < left ? o : left - 1));
        }
#pragma unroll
        for (int q = 0; q < FK_PER; ++q) {
            if (q < per) f[q] = fork_row(a, from[q], bad);
            if (q >= per || tid * per + q >= left) f[q] = {0, 0, 0};
        }
#pragma unroll
        for (int q = 0; q < FK_PER; ++q) mine += f[q].len + f[q].add;
        const int64_t sum = (int64_t)wave_scan_f64((double)mine);  // inclusive (ids are counted exactly)
        if (lane == WAVE - 1) wave[w] = sum;
        __syncthreads();
        int64_t at = carry + sum - mine;
#pragma unroll
        for (int i = 0; i < NT / WAVE; ++i) {
            at += i < w ? wave[i] : 0;
            carry += wave[i];
        }
#pragma unroll
        for (int q = 0; q < FK_PER; ++q) {
            if (q < per && tid * per + q < left) each(c + tid * per + q, at, f[q].len + f[q].add, f[q].at);
            at += f[q].len + f[q].add;
        }
        __syncthreads();
    }
    return carry;
}

constexpr int FK_OFF = 1024;               // threads of the offsets' launch
__global__ __launch_bounds__(FK_OFF) void fork_offsets_kernel(ForkArgs a) {
    bool bad = false;
    const int64_t end = fork_scan<FK_OFF>(a, bad, [&](int o, int64_t v, int64_t, int64_t) { a.out_off[o] = v; });
    if (threadIdx.x == 0) {
        a.out_off[(int64_t)a.S * a.n] = end;
        if (end > a.out_cap) atomicOr(a.err, FS_DEVERR_HIST_APPEND);
    }
    if (bad) atomicOr(a.err, FS_DEVERR_PARENT);
}

typedef int i32x4a __attribute__((ext_vector_type(4), aligned(4)));    // (histories begin at any id)

template <bool SELF>
__global__ __launch_bounds__(FK_T, 8) void fork_kernel(ForkArgs a) {
    __shared__ int64_t s_off[SELF ? FK_ROWS + 1 : 1], s_at[SELF ? FK_ROWS : 1];
    __shared__ int s_row[2];
    const int tid = threadIdx.x, R = a.S * a.n;
    bool bad = false;
    int64_t end;
    if (SELF) {
        end = fork_scan<FK_T>(a, bad, [&](int o, int64_t v, int64_t, int64_t from) {
            s_off[o] = v;
            s_at[o] = from;
        });
        if (tid == 0) s_off[R] = end;
        __syncthreads();
        if (blockIdx.x == 0) {
            for (int o = tid; o <= R; o += FK_T) a.out_off[o] = s_off[o];
            if (tid == 0 && end > a.out_cap) atomicOr(a.err, FS_DEVERR_HIST_APPEND);
            if (bad) atomicOr(a.err, FS_DEVERR_PARENT);
        }
    } else {
        end = a.out_off[R];
    }
    auto off = [&](int o) { return SELF ? s_off[o] : a.out_off[o]; };
    if (end > a.out_cap) end = a.out_cap;                      // (ids past it are not written)
    // this workgroup's share of the ids, in whole steps
    const int64_t steps = (end + FK_STEP - 1) / FK_STEP, share = (steps + gridDim.x - 1) / gridDim.x * FK_STEP;
    const int64_t b = share * blockIdx.x, e = b + share < end ? b + share : end;
    if (b >= e) return;
    auto row_of = [&](int64_t i, int lo, int hi) {             // the last row of [lo, hi] that begins at or before id i
        while (lo < hi) {
            const int m = (lo + hi + 1) >> 1;
            if (off(m) <= i) lo = m; else hi = m - 1;
        }
        return lo;
    };
    int r0, r1;
    if (SELF) {                                                // the rows of the share's first and last id
        for (int o = tid; o < R; o += FK_T) {
            if (s_off[o] <= b && b < s_off[o + 1]) s_row[0] = o;
            if (s_off[o] < e && e <= s_off[o + 1]) s_row[1] = o;
        }
        __syncthreads();
        r0 = s_row[0];
        r1 = s_row[1];
    } else {
        r0 = row_of(b, 0, R - 1);
        r1 = row_of(e - 1, r0, R - 1);
    }
#pragma unroll 1
    for (int64_t i0 = b; i0 < e; i0 += FK_U * FK_STEP) {
        i32x4a v[FK_U];
        int from[FK_U];                                        // 4: four of one history; else how many ids there are
#pragma unroll
        for (int u = 0; u < FK_U; ++u) {
            const int64_t i = i0 + u * FK_STEP + tid * 4;
            from[u] = -1;
            if (i < e) {
                const int r = row_of(i, r0, r1);
                const int64_t base = off(r), len = off(r + 1) - base - (a.tok ? 1 : 0);
                bool bad2 = false;
                const int64_t src = SELF ? s_at[r] : fork_row(a, fork_from(a, r), bad2).at;
                from[u] = i + 4 <= e && i - base + 4 <= len ? 4 : 0;
                if (from[u] == 4) v[u] = *reinterpret_cast<const i32x4a*>(a.hist + src + (i - base));
            }
        }
#pragma unroll
        for (int u = 0; u < FK_U; ++u) {
            const int64_t i = i0 + u * FK_STEP + tid * 4;
            if (from[u] == 4) __builtin_nontemporal_store(v[u], reinterpret_cast<i32x4a*>(a.out + i));
            if (from[u] == 0) {                                // a history's end, or the share's: one at a time
                for (int64_t j = i; j < i + 4 && j < e; ++j) {
                    const int r = row_of(j, r0, r1);
                    const int64_t base = off(r), len = off(r + 1) - base - (a.tok ? 1 : 0);
                    bool bad2 = false;
                    const int64_t src = SELF ? s_at[r] : fork_row(a, fork_from(a, r), bad2).at;
                    a.out[j] = j - base < len ? a.hist[src + (j - base)] : a.tok[r];
                }
            }
        }
    }
}

hipError_t launch_hist_fork(const ForkArgs& a, int cus, hipStream_t st) {
    const int64_t R = (int64_t)a.S * a.n;
    const int64_t want = (a.out_cap + FK_STEP - 1) / FK_STEP, most = FK_PER_CU * (int64_t)cus;
    const dim3 grid((unsigned)(want < 1 ? 1 : want < most ? want : most)), block(FK_T);
    if (R <= FK_ROWS) {
        hipLaunchKernelGGL(fork_kernel<true>, grid, block, 0, st, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(fork_offsets_kernel, dim3(1), dim3(FK_OFF), 0, st, a);
    hipLaunchKernelGGL(fork_kernel<false>, grid, block, 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ states
// Row (s, j) of every state gets what row (s, parent[s n + j]) of the source held. A thread takes columns, VB bytes at one
// place of a row, of all of a stream's rows: it loads the column of every row that goes somewhere, then stores them, so a
// stream's rows may change places among themselves in the same buffer, and a row that goes to several is read once.
// The columns of all states and streams are dealt evenly to a grid that fills the device once, in tiles of K columns per
// thread: the streams' lengths are read on the device, 64 streams at a time, and a scan over them gives each workgroup its
// tiles; which rows go where is worked out once per 64 streams, in LDS. All workgroups walk through all states, unless those are
// alike (a model's layers) and a workgroup has few tiles: it then takes one state. (One state by one, 20 of 64 KB of one stream
// 8.7 -> 4.9 us, 32 of 16 streams 14.4 -> 7.6, 16 caches of 64 rows with four tiles each 87 -> 84; with ten each, 20 states of
// 64 MB, 209 -> 221: many states at once are not good for the memory.)
// Stores go past the caches, loads do not (a source may be read again): 16 caches of 64 rows 87.1 -> 80.8 us with stores so; with
// loads so, too, no more.
// Bound: HBM: those caches 79 us (4.7 TB/s of 373 MB), 16 caches of 16 prompts opened into four beams each 223 us (4.8 TB/s of
// 1064 MB, four fifths of them stores), one small state 4.6. Past 32 beams the walk over 64 rows and columns of 8 bytes: 64 rows of
// eight caches of 0.5 MB a row in place by 4, 8, 16, 32, 64 beams 47, 44, 42, 48, 71 us (206 to 256 MB), from one prompt into 8,
// 32, 64 beams 50, 51, 60 (273 to 302 MB).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int VB>
using StateVec = std::conditional_t<VB == 16, u32x4, std::conditional_t<VB == 8, u32x2, std::conditional_t<VB == 4, uint32_t,
                 std::conditional_t<VB == 2, uint16_t, uint8_t>>>>;

constexpr int ST_T = 256;
template <int VB, int NB, int K>
__global__ __launch_bounds__(ST_T) void reorder_states_kernel(StateArgs a_) {
    using Vec = StateVec<VB>;
    constexpr uint32_t TILE = ST_T * K;
    __shared__ unsigned long long to[WAVE][NB];                // the rows that a stream's source row i goes to
    // (indexed records: read from the argument segment, not from a copy)
    const __attribute__((address_space(4))) char* kseg =
        (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
    const StateArgs& a = *(const StateArgs*)kseg;
    (void)a_;
    const int tid = threadIdx.x, lane = lane_id();
    const uint32_t G = a.alike ? gridDim.x / a.n_states : gridDim.x;
    const int k0 = a.alike ? (int)(blockIdx.x % a.n_states) : 0, k1 = a.alike ? k0 + 1 : a.n_states;
    uint32_t turn = a.alike ? blockIdx.x / a.n_states : blockIdx.x;    // this workgroup's next tile, counted from a state's first
#pragma unroll 1
    for (int s0 = 0; s0 < a.S; s0 += WAVE) {
        const int ns = a.S - s0 < WAVE ? a.S - s0 : WAVE;
        const int from = lane < ns && a.from ? a.from[s0 + lane] : 0;
        const int till = lane < ns && a.len ? a.len[s0 + lane] : 0x7fffffff;
        if (s0 > 0) __syncthreads();
        for (int i = tid; i < ns * NB; i += ST_T) to[i / NB][i % NB] = 0ull;
        __syncthreads();
        for (int i = tid; i < ns * a.n; i += ST_T) {
            const int s = i / a.n, j = i - s * a.n, p = a.parent[(int64_t)s0 * a.n + i];
            if (p >= a.n_src) {
                if (blockIdx.x == 0) atomicOr(a.err, FS_DEVERR_PARENT);
            } else if (p >= 0) {
                atomicOr(&to[s][p], 1ull << j);
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int k = k0; k < k1; ++k) {
            const fs_state& z = a.z[k];
            const bool same = z.d_src == z.d_dst;
            const uint32_t per = (uint32_t)z.pos_bytes / VB;
            int lo = 0, hi = 1;
            if (z.positions > 0) {
                lo = from > 0 ? from : 0;
                hi = till < z.positions ? till : z.positions;
            }
            const uint32_t used = lane < ns && hi > lo ? (uint32_t)(hi - lo) : 0u;
            const uint32_t cols = per * used * (uint32_t)z.blocks, tiles = (cols + TILE - 1u) / TILE;
            const uint32_t incl = wave_incl_scan_u32(tiles);
            const uint32_t total = (uint32_t)read_lane((int)incl, WAVE - 1);
            const bool packed = z.src_pos == z.pos_bytes && z.dst_pos == z.pos_bytes;
#pragma unroll 1
            for (; turn < total; turn += G) {
                const int s = __popcll(__ballot(incl <= turn));    // the tile's stream
                const uint32_t first = s > 0 ? (uint32_t)read_lane((int)incl, s - 1) : 0u;
                const uint32_t n_col = (uint32_t)read_lane((int)cols, s), n_pos = (uint32_t)read_lane((int)used, s);
                const int p0 = read_lane(lo, s);
                const unsigned long long mine = lane < NB ? to[s][lane] : 0ull;
                const char* src0 = (const char*)z.d_src + (int64_t)(s0 + s) * a.n_src * z.src_row + (int64_t)p0 * z.src_pos;
                char* dst0 = (char*)z.d_dst + (int64_t)(s0 + s) * a.n * z.dst_row + (int64_t)p0 * z.dst_pos;
                auto goes = [&](int i) {                       // (in place a row that stays does not move)
                    const uint64_t m = read_lane((uint64_t)mine, i);
                    return same ? m & ~(1ull << i) : m;
                };
                const uint32_t run = packed ? per * n_pos : per;   // columns that lie side by side
                int64_t so[K], d_o[K];
                bool on[K];
#pragma unroll
                for (int c = 0; c < K; ++c) {
                    uint32_t col = (turn - first) * TILE + c * ST_T + tid;
                    on[c] = col < n_col;
                    col = on[c] ? col : 0u;
                    const uint32_t at = col / run, off = col - at * run;
                    const uint32_t block = packed ? at : at / n_pos, pos = packed ? 0u : at - block * n_pos;
                    so[c] = (int64_t)block * z.src_block + (int64_t)pos * z.src_pos + (int64_t)off * VB;
                    d_o[c] = (int64_t)block * z.dst_block + (int64_t)pos * z.dst_pos + (int64_t)off * VB;
                }
                Vec v[NB][K];
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    if (goes(i) != 0ull)
#pragma unroll
                        for (int c = 0; c < K; ++c)
                            if (on[c]) v[i][c] = *reinterpret_cast<const Vec*>(src0 + i * z.src_row + so[c]);
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    for (uint64_t m = goes(i); m; m &= m - 1) {
                        char* d = dst0 + (__ffsll((unsigned long long)m) - 1) * z.dst_row;
#pragma unroll
                        for (int c = 0; c < K; ++c)
                            if (on[c]) __builtin_nontemporal_store(v[i][c], reinterpret_cast<Vec*>(d + d_o[c]));
                    }
            }
            turn -= total;
        }
    }
}

hipError_t launch_reorder_states(int vb, StateArgs a, int64_t cols, int cus, hipStream_t st) {
    const int rows = a.n_src > a.n ? a.n_src : a.n;
    auto go = [&](auto v, auto nb, auto k) {                    // (tiles: an upper bound, the states' positions all in use)
        constexpr int VB = decltype(v)::value, NB = decltype(nb)::value, K = decltype(k)::value;
        const int64_t want = (cols + ST_T * K - 1) / (ST_T * K) + (int64_t)a.n_states * a.S, most = 8 * (int64_t)cus;
        int64_t n = want < most ? want : most;
        a.alike &= want <= 4 * most ? 1 : 0;
        if (a.alike) n = (n + a.n_states - 1) / a.n_states * a.n_states;
        const dim3 grid((unsigned)n), block(ST_T);
        hipLaunchKernelGGL((reorder_states_kernel<VB, NB, K>), grid, block, 0, st, a);
    };
    // Columns per thread: as many as keep enough loads in flight, where few rows do not. The caches above with 1, 2, 4 columns,
    // in place by 4 beams: 54, 52, 47 us; by 8: 48, 44, 56; by 16 (1, 2): 42, 44; into other buffers by 4: 96, 100, 89; by 8:
    // 96, 85, 99; by 16 (1, 2): 84, 86. By 64 beams with columns of 4, 8, 16 bytes: 63, 71, 48 in place, 100, 126, 93 into other
    // buffers, 64, 60, 63 from one prompt; in place by 33: 43, 35, 36 (state_bytes in sampler_kernels.hip takes 8).
    auto by_rows = [&](auto v) {
        constexpr int VB = decltype(v)::value;
        if (rows <= 4) go(v, std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
        else if (rows <= 8) go(v, std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
        else if (rows <= 16) go(v, std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
        else if (rows <= 32) go(v, std::integral_constant<int, 32>{}, std::integral_constant<int, 1>{});
        else go(std::integral_constant<int, (VB > 8 ? 8 : VB)>{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
    };
    if (vb == 16) by_rows(std::integral_constant<int, 16>{});
    else if (vb == 8) by_rows(std::integral_constant<int, 8>{});
    else if (vb == 4) by_rows(std::integral_constant<int, 4>{});
    else if (vb == 2) by_rows(std::integral_constant<int, 2>{});
    else by_rows(std::integral_constant<int, 1>{});
    return hipGetLastError();
}

}  // namespace fs
