// beam_kernels.hip - beam search: histories and model states that follow their beams (the selection: logprob_kernel.hip,
// beam_device.hpp).
#include "sampler_device.hpp"
#include "sampler_launch.hpp"

#include <type_traits>

namespace fs {

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
