// beam_kernels.hip - beam search: the selection over a stream's beams and tokens, histories and model states that follow
// their beams.
#include "edit_device.hpp"

namespace fs {

// ------------------------------------------------------------------------------------------------ selection
// Row r of a stream has the score a_r; its token t is the candidate
//
//   c(r, t) = a_r + (x_t - M) / T - log sum_j exp((x_j - M) / T),   x = cap(logit) + bias over the allowed tokens, M = max x.
//
// One workgroup per row makes the row's sum (fp64, relative to each lane's largest logit so far) and its n largest tokens but
// eos (a sorted list per wave, one entry per lane: 64 logits are sorted and merged into it where one of them reaches its n-th);
// eos's logit is kept by itself. One wave per stream then takes the n best of the rows' lists.
constexpr int BM_T = 256;
constexpr int BM_NW = BM_T / WAVE;
constexpr float BM_NONE = -__builtin_huge_valf();

// The stream of a row: the largest s with row_off[s] <= row.
__device__ __forceinline__ int bm_stream(const BeamArgs& a, int row) {
    if (!a.row_off) return row / (a.R / a.S);
    int s0 = 0, s1 = a.S;
    while (s1 - s0 > 1) {
        const int m = (s0 + s1) >> 1;
        if (ld_const(a.row_off + m) <= row) s0 = m; else s1 = m;
    }
    return s0;
}

__device__ __forceinline__ double bm_score(const BeamRow& r, float x) {
    if (!(x > BM_NONE) || (x < r.M && !(r.M < __builtin_huge_valf()))) return -__builtin_huge_val();
    return r.a + ((x == r.M ? 0.0 : ((double)x - (double)r.M) / (double)r.T) - r.z);
}

template <int TYPE>
__global__ __launch_bounds__(BM_T) void beam_rows_kernel(BeamArgs a) {
    __shared__ uint64_t lists[BM_NW][WAVE];
    __shared__ double sums[BM_NW];
    __shared__ float maxs[BM_NW], s_eos;
    const int tid = threadIdx.x, lane = lane_id(), w = tid / WAVE, row = (int)blockIdx.x, V = a.V, n = a.n;
    const float score = a.score ? ld_const(a.score + row) : 0.0f;
    BeamRow* out = a.rows + row;
    if (!(score > BM_NONE)) {                                  // a dead beam: its row is not read
        if (tid == 0) {
            out->cnt = 0;
            out->eos = BM_NONE;
        }
        return;
    }
    const int rec = bm_stream(a, row);
    const EdRow r = ed_row(a.ed, row, rec, a.err);
    float cap = 0.0f, T = 1.0f;
    if (a.params) {
        cap = ld_const(&a.params[rec].softcap);
        T = ld_const(&a.params[rec].temperature);
        if (!(T > 0.0f)) T = 1.0f;
    }
    if (tid == 0) s_eos = BM_NONE;
    __syncthreads();
    using L = Logits4<TYPE>;
    const __amdgpu_buffer_rsrc_t rs = L::rsrc(a.logits, (int64_t)row * a.ld, V);
    float m = BM_NONE;
    double sum = 0.0;
    uint64_t acc = 0ull, bound = 0ull;
#pragma unroll 1
    for (int g = 0; g * 4 < V; g += BM_T) {
        float x[4];
        L::floats(L::load(rs, g + tid), x);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            const int t = (g + tid) * 4 + c;
            float v = c == 0 ? x[0] : c == 1 ? x[1] : c == 2 ? x[2] : x[3];
            if (t < V) {
                if (cap > 0.0f) v = softcap_one(v, cap);
                v = ed_lane(r, v, t);
            }
            const bool on = t < V && v > BM_NONE;
            if (on) {
                if (v > m) {
                    sum = v < __builtin_huge_valf() && m > BM_NONE ? sum * exp(((double)m - (double)v) / (double)T) : 0.0;
                    m = v;
                }
                sum += v == m ? 1.0 : exp(((double)v - (double)m) / (double)T);
                if (t == a.eos) s_eos = v;
            }
            const uint64_t e = on && t != a.eos ? comp_of(key_of(v), (uint32_t)t) : 0ull;
            if (__ballot(e > bound) != 0ull) {
                acc = merge_top64(acc, sort64<false>(e));
                bound = read_lane(acc, n - 1);
            }
        }
    }
    // the wave's, then the row's sum and list
    auto fmx = [](float u, float v) { return fmaxf(u, v); };
    auto add = [](double u, double v) { return u + v; };
    const float wm = wave_allreduce(m, fmx);
    auto onto = [&](double s, float from, float to) {          // a sum relative to another maximum
        if (!(from > BM_NONE)) return 0.0;
        return from == to ? s : to < __builtin_huge_valf() ? s * exp(((double)from - (double)to) / (double)T) : 0.0;
    };
    sum = wave_allreduce(onto(sum, m, wm), add);
    lists[w][lane] = acc;
    if (lane == 0) {
        sums[w] = sum;
        maxs[w] = wm;
    }
    __syncthreads();
    if (w != 0) return;
    float M = BM_NONE;
    for (int i = 0; i < BM_NW; ++i) M = fmaxf(M, maxs[i]);
    double Z = 0.0;
    for (int i = 0; i < BM_NW; ++i) Z += onto(sums[i], maxs[i], M);
    for (int i = 1; i < BM_NW; ++i) acc = merge_top64(acc, lists[i][WAVE - 1 - lane]);
    const int cnt = __popcll(__ballot(lane < n && acc != 0ull));
    a.lists[(int64_t)row * BM_TOP + lane] = acc;
    if (lane == 0) {
        out->a = (double)score;
        out->z = M > BM_NONE ? log(Z) : 0.0;
        out->M = M;
        out->T = T;
        out->eos = s_eos;
        out->cnt = cnt;
    }
}

// A candidate of a stream: its score as an ordered integer (0: none), its row in the stream and its token.
__device__ __forceinline__ uint64_t bm_key(double c) {
    if (!((float)c > BM_NONE)) return 0ull;
    const uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

__global__ __launch_bounds__(WAVE) void beam_join_kernel(BeamArgs a) {
    __shared__ uint64_t key[2 * BM_TOP];                       // the best so far in order, then a row's
    __shared__ int from[2 * BM_TOP], token[2 * BM_TOP];
    __shared__ float value[2 * BM_TOP];
    __shared__ int first[BM_TOP], place[BM_TOP];
    const int lane = lane_id(), s = (int)blockIdx.x, n = a.n;
    const int64_t r0 = a.row_off ? a.row_off[s] : (int64_t)s * (a.R / a.S);
    const int64_t r1 = a.row_off ? a.row_off[s + 1] : r0 + a.R / a.S;
    const int rows = (int)(r1 - r0);
    key[lane] = 0ull;
    from[lane] = -1;
    token[lane] = -1;
    value[lane] = BM_NONE;
#pragma unroll 1
    for (int r = 0; r < rows; ++r) {
        const BeamRow br = a.rows[r0 + r];
        uint64_t k = 0ull;
        int t = -1;
        float v = BM_NONE;
        if (lane < br.cnt) {
            const uint64_t e = a.lists[(r0 + r) * BM_TOP + lane];
            const double c = bm_score(br, val_of(comp_key(e)));
            k = bm_key(c);
            t = k ? (int)comp_id(e) : -1;
            v = k ? (float)c : BM_NONE;
        }
        __syncthreads();
        const int f = k ? r : -1;
        key[BM_TOP + lane] = k;
        const uint64_t k0 = key[lane];
        const int f0 = from[lane], t0 = token[lane];
        const float v0 = value[lane];
        __syncthreads();
        int p0 = lane, p = 0;                                  // places: the earlier rows' first among equal scores
        for (int i = 0; i < BM_TOP; ++i) {
            p0 += key[BM_TOP + i] > k0 ? 1 : 0;
            p += key[i] >= k ? 1 : 0;
        }
        p += lane;                                             // (a row's list is in order)
        __syncthreads();
        if (p0 < BM_TOP) { key[p0] = k0; from[p0] = f0; token[p0] = t0; value[p0] = v0; }
        if (p < BM_TOP) { key[p] = k; from[p] = f; token[p] = t; value[p] = v; }
        __syncthreads();
    }
    const bool live = lane < n && key[lane] != 0ull;
    // ended hypotheses
    if (a.done || a.done_parent || a.done_score) {
        if (lane < n) {
            if (a.done_parent) a.done_parent[(int64_t)s * n + lane] = -1;
            if (a.done_score) a.done_score[(int64_t)s * n + lane] = BM_NONE;
        }
        __syncthreads();
        int done = 0;
        if (a.eos >= 0) {
            for (int b = 0; b < rows; b += WAVE) {
                const int r = b + lane;
                const double c = r < rows ? bm_score(a.rows[r0 + r], a.rows[r0 + r].eos) : -__builtin_huge_val();
                const uint64_t k = bm_key(c);
                int before = 0, ahead = 0;                     // better candidates; those of them that end, too
                for (int i = 0; i < n; ++i) before += key[i] > k ? 1 : 0;
                for (int i = 0; i < rows; ++i) {
                    const uint64_t o = bm_key(bm_score(a.rows[r0 + i], a.rows[r0 + i].eos));
                    ahead += o > k || (o == k && i < r) ? 1 : 0;
                }
                const bool in = k != 0ull && before + ahead < n;
                if (in) {
                    if (a.done_parent) a.done_parent[(int64_t)s * n + ahead] = r;
                    if (a.done_score) a.done_score[(int64_t)s * n + ahead] = (float)c;
                }
                done += __popcll(__ballot(in));
            }
        }
        if (a.done && lane == 0) a.done[s] = done;
    }
    // places of the new beams
    int slot = lane;
    if (a.keep_slots) {
        const int p = live ? from[lane] : -1;
        first[lane] = WAVE;
        __syncthreads();
        if (p >= 0 && p < n) atomicMin(&first[p], lane);
        __syncthreads();
        const bool stays = p >= 0 && p < n && first[p] == lane;
        const bool free_ = lane < n && first[lane] == WAVE;    // (of the slot `lane`)
        const uint64_t fm = __ballot(free_), lm = __ballot(lane < n && !stays);
        if (free_) place[mbcnt(fm)] = lane;
        __syncthreads();
        if (lane < n) slot = stays ? p : place[mbcnt(lm)];
    }
    if (lane < n) {
        const int64_t o = (int64_t)s * n + slot;
        a.parent[o] = live ? from[lane] : -1;
        a.tok[o] = live ? token[lane] : -1;
        a.out_score[o] = live ? value[lane] : BM_NONE;
    }
}

hipError_t launch_beam_select(int type, const BeamArgs& a, hipStream_t st) {
    if (a.R > 0) {
        const dim3 grid((unsigned)a.R), block(BM_T);
        if (type == FS_F32) hipLaunchKernelGGL(beam_rows_kernel<FS_F32>, grid, block, 0, st, a);
        else if (type == FS_BF16) hipLaunchKernelGGL(beam_rows_kernel<FS_BF16>, grid, block, 0, st, a);
        else hipLaunchKernelGGL(beam_rows_kernel<FS_F16>, grid, block, 0, st, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a.S), dim3(WAVE), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ histories
// Beam j of stream s (row s n + j) gets the history of the stream's beam parent[s n + j] and the token behind it.
struct ForkRow {
    int64_t at, len;                                           // its parent's ids
    int add;                                                   // 1: a token behind them
};
__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int64_t o, bool& bad) {
    const int64_t s = o / a.n;
    const int64_t r0 = a.row_off ? a.row_off[s] : s * a.n, rows = a.row_off ? a.row_off[s + 1] - r0 : a.n;
    const int p = a.parent[o];
    ForkRow f = {0, 0, 0};
    bad |= p >= rows;
    if (p < 0 || p >= rows) return f;
    f.at = a.hist_off[r0 + p];
    f.len = a.hist_off[r0 + p + 1] - f.at;
    f.add = a.tok ? 1 : 0;
    return f;
}

// One workgroup: the new offsets.
constexpr int FK_T = 256;
__global__ __launch_bounds__(FK_T) void fork_offsets_kernel(ForkArgs a) {
    __shared__ int64_t part[FK_T];
    const int tid = threadIdx.x;
    const int64_t R = (int64_t)a.S * a.n, per = (R + FK_T - 1) / FK_T;
    const int64_t b = tid * per < R ? tid * per : R, e = b + per < R ? b + per : R;
    bool bad = false;
    int64_t sum = 0;
    for (int64_t o = b; o < e; ++o) {
        const ForkRow f = fork_row(a, o, bad);
        sum += f.len + f.add;
    }
    part[tid] = sum;
    __syncthreads();
    int64_t at = 0;
    for (int i = 0; i < tid; ++i) at += part[i];
    for (int64_t o = b; o < e; ++o) {
        const ForkRow f = fork_row(a, o, bad);
        a.out_off[o] = at;
        at += f.len + f.add;
    }
    if (tid == FK_T - 1) {
        a.out_off[R] = at;
        if (at > a.out_cap) atomicOr(a.err, FS_DEVERR_HIST_APPEND);
    }
    if (bad) atomicOr(a.err, FS_DEVERR_PARENT);
}

__global__ __launch_bounds__(FK_T) void fork_copy_kernel(ForkArgs a) {
    const int64_t o = blockIdx.x;
    bool bad = false;
    const ForkRow f = fork_row(a, o, bad);
    const int64_t to = a.out_off[o];
    for (int64_t i = threadIdx.x; i < f.len + f.add; i += FK_T)
        if (to + i < a.out_cap) a.out[to + i] = i < f.len ? a.hist[f.at + i] : a.tok[o];
}

hipError_t launch_hist_fork(const ForkArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(fork_offsets_kernel, dim3(1), dim3(FK_T), 0, st, a);
    if (a.S > 0) hipLaunchKernelGGL(fork_copy_kernel, dim3((unsigned)((int64_t)a.S * a.n)), dim3(FK_T), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------ states
// Row (s, j) of every state gets what row (s, parent[s n + j]) of the source held. A thread takes one column, VB bytes at one
// place of a row, of all of a stream's rows: it loads the column of every row that is a parent of a row that moves, then
// stores them, so a stream's rows may change places among themselves in the same buffer.
template <int VB>
using StateVec = std::conditional_t<VB == 16, uint4, std::conditional_t<VB == 8, uint2, std::conditional_t<VB == 4, uint32_t,
                 std::conditional_t<VB == 2, uint16_t, uint8_t>>>>;

constexpr int ST_T = 256;
template <int VB, int NB>
__global__ __launch_bounds__(ST_T) void reorder_states_kernel(StateArgs a) {
    using Vec = StateVec<VB>;
    __shared__ uint64_t to[NB];                                // the rows that source row i goes to
    const int s = (int)blockIdx.y;
    const fs_state& z = a.z[blockIdx.z];
    const int tid = threadIdx.x;
    int lo = 0, hi = 1;
    if (z.positions > 0) {
        lo = a.from ? a.from[s] : 0;
        hi = a.len ? a.len[s] : z.positions;
        lo = lo > 0 ? lo : 0;
        hi = hi < z.positions ? hi : z.positions;
        if (lo >= hi) return;
    }
    const uint32_t per = (uint32_t)(z.pos_bytes / VB), used = (uint32_t)(hi - lo);
    const uint32_t cols = per * used * (uint32_t)z.blocks;
    const uint32_t col = blockIdx.x * ST_T + tid;
    if (blockIdx.x * ST_T >= cols) return;
    const bool same = z.d_src == z.d_dst;
    if (tid < NB) to[tid] = 0ull;
    __syncthreads();
    if (tid < a.n) {
        const int p = a.parent[(int64_t)s * a.n + tid];
        if (p >= a.n_src) atomicOr(a.err, FS_DEVERR_PARENT);
        else if (p >= 0 && !(same && p == tid)) atomicOr((unsigned long long*)&to[p], 1ull << tid);
    }
    __syncthreads();
    if (col >= cols) return;
    const uint32_t at = col / per, off = col - at * per;
    const uint32_t block = at / used, pos = at - block * used + (uint32_t)lo;
    const char* src = (const char*)z.d_src + (int64_t)s * a.n_src * z.src_row + block * z.src_block + pos * z.src_pos +
                      (int64_t)off * VB;
    char* dst = (char*)z.d_dst + (int64_t)s * a.n * z.dst_row + block * z.dst_block + pos * z.dst_pos + (int64_t)off * VB;
    Vec v[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
        if (to[i] != 0ull) v[i] = *reinterpret_cast<const Vec*>(src + i * z.src_row);
#pragma unroll
    for (int i = 0; i < NB; ++i)
        for (uint64_t m = to[i]; m; m &= m - 1)
            *reinterpret_cast<Vec*>(dst + (__ffsll((unsigned long long)m) - 1) * z.dst_row) = v[i];
}

hipError_t launch_reorder_states(int vb, const StateArgs& a, int n_states, int64_t tiles, hipStream_t st) {
    const dim3 grid((unsigned)tiles, (unsigned)a.S, (unsigned)n_states), block(ST_T);
    const int rows = a.n_src > a.n ? a.n_src : a.n;
    auto go = [&](auto v) {
        constexpr int VB = decltype(v)::value;
        if (rows <= 8) hipLaunchKernelGGL((reorder_states_kernel<VB, 8>), grid, block, 0, st, a);
        else if (rows <= 16) hipLaunchKernelGGL((reorder_states_kernel<VB, 16>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((reorder_states_kernel<(VB > 8 ? 8 : VB), 64>), grid, block, 0, st, a);
    };
    if (vb == 16) go(std::integral_constant<int, 16>{});
    else if (vb == 8) go(std::integral_constant<int, 8>{});
    else if (vb == 4) go(std::integral_constant<int, 4>{});
    else if (vb == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    return hipGetLastError();
}

}  // namespace fs
