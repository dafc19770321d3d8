// edit_device.hpp - masks of allowed tokens and biases on a segment of logits held in registers: thread t of SK_LT holds
// logits (q * SK_LT + t) * 4 .. + 3 of its segment for q < NL, as in the small-k and mid-k kernels.
#ifndef FERRO_EDIT_DEVICE_HPP
#define FERRO_EDIT_DEVICE_HPP

#include "sampler_device.hpp"
#include "sampler_launch.hpp"

#include <type_traits>

namespace fs {

// A row's mask and biases. words NULL: every token is allowed; closed: none is (a mask index past the last mask).
struct EdRow {
    const uint32_t* words;
    bool closed;
    const int32_t* ids;                    // nb biases
    const float* val;
    int64_t nb;
};
// row: the logits row
__device__ __forceinline__ void ed_mask(EdRow& r, const EdArgs& ed, int row, int32_t* err) {
    r.words = nullptr;
    r.closed = false;
    if (!ed.mask) return;
    const int m = ed.mask_of ? ld_const(ed.mask_of + row) : row;
    r.closed = m >= ed.n_masks;
    if (r.closed && threadIdx.x == 0) atomicOr(err, FS_DEVERR_MASK);
    if (m >= 0 && !r.closed) r.words = ed.mask + (int64_t)m * ed.mask_ld;
}
// rec: its record
__device__ __forceinline__ void ed_bias(EdRow& r, const EdArgs& ed, int rec) {
    r.nb = 0;
    if (!ed.bias_off) return;
    const int64_t b = ld_const(ed.bias_off + rec);
    r.nb = ld_const(ed.bias_off + rec + 1) - b;
    r.ids = ed.bias_ids + b;
    r.val = ed.bias + b;
}
__device__ __forceinline__ EdRow ed_row(const EdArgs& ed, int row, int rec, int32_t* err) {
    EdRow r = {nullptr, false, nullptr, nullptr, 0};
    ed_mask(r, ed, row, err);
    ed_bias(r, ed, rec);
    return r;
}
// One logit, by one lane: a bit of the mask, a bisection of the biases. For the paths that read a row again.
__device__ __forceinline__ float ed_lane(const EdRow& r, float l, int id) {
    if (r.nb > 0) {
        int64_t lo = 0, hi = r.nb;                             // the first bias whose id is at least id
        while (lo < hi) {
            const int64_t m = (lo + hi) >> 1;
            if (r.ids[m] < id) lo = m + 1; else hi = m;
        }
        for (; lo < r.nb && r.ids[lo] == id; ++lo) l = __fadd_rn(l, r.val[lo]);
    }
    return r.closed || (r.words && ((r.words[id >> 5] >> (id & 31)) & 1u) == 0u) ? __builtin_nanf("") : l;
}

// A wave's share of the segment's mask: 32 NL words, word q * 8 + j of which covers lanes 8 j .. 8 j + 7 of group q. Lane l
// holds words l and, with NL = 16, 64 + l: one coalesced load of 4 bytes per eight groups, and a permute gives a lane its
// four bits (a load per group and lane would double the kernel's memory instructions).
struct EdBits {
    uint32_t a, b;
};
template <int NL>
__device__ __forceinline__ EdBits ed_bits(const EdRow& r, int seg_lo, int V) {
    EdBits m = {~0u, ~0u};
    if (r.closed) m.a = m.b = 0u;
    if (!r.words) return m;
    const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
    const int nw = ((V + 31) >> 5) - (seg_lo >> 5);            // words from the segment's first on
    const uint32_t* p = r.words + (seg_lo >> 5);
    const int at = (lane >> 3) * (SK_LT / 8) + w * 8 + (lane & 7);
    m.a = at < nw ? p[at] : 0u;
    if (NL > 8) m.b = at + SK_LT < nw ? p[at + SK_LT] : 0u;
    return m;
}
// the lane's four bits of group q (whole wave)
__device__ __forceinline__ uint32_t ed_nibble(const EdBits& m, int q) {
    const int lane = lane_id();
    const uint32_t word = (uint32_t)__builtin_amdgcn_ds_bpermute(((q & 7) * 8 + (lane >> 3)) * 4, (int)(q < 8 ? m.a : m.b));
    return (word >> (4 * (lane & 7))) & 15u;
}
// x where bit c of the nibble is set, else the bits of `no`
__device__ __forceinline__ float ed_keep(float x, uint32_t nibble, int c, uint32_t no) {
    const uint32_t on = (uint32_t)((int32_t)(nibble << (31 - c)) >> 31);
    return __uint_as_float((__float_as_uint(x) & on) | (no & ~on));
}

// The first of a row's biases whose id is at least `id` (whole wave, uniform): 64 probes at a time.
__device__ __forceinline__ int64_t ed_lower(const EdRow& r, int id) {
    int64_t lo = 0, hi = r.nb;
    while (hi - lo > WAVE) {
        const int64_t step = (hi - lo + WAVE - 1) / WAVE, at = lo + lane_id() * step;
        const int n = __popcll(__ballot(at < hi && r.ids[at] < id));
        hi = lo + n * step < hi ? lo + n * step : hi;
        lo += n > 0 ? (n - 1) * step : 0;
        if (n == 0) return lo;
    }
    return lo + __popcll(__ballot(lo + lane_id() < hi && r.ids[lo + lane_id()] < id));
}
// A row's biases requested early, with the logits, and used when those are there: the first 64 of them in every wave, one
// per lane, or, where the workgroup shares them (SHARE) and there are more, the first SK_LT, one per thread.
struct EdList {
    int64_t nb;
    int id;
    float val;
};
template <bool SHARE>
__device__ __forceinline__ EdList ed_list(const EdRow& r) {
    EdList l = {r.nb, 0x7fffffff, 0.0f};
    const int i = SHARE && r.nb > WAVE ? (int)threadIdx.x : lane_id();
    if (i < r.nb) {
        l.id = r.ids[i];
        l.val = r.val[i];
    }
    return l;
}
// Adds the biases of record rec to the wave's logits of the segment, one after another in list order (equal ids add up):
// each is held by one lane, and the wave gives it to the lane whose logit it is, group by group (with all groups in one
// loop, or with a branch per lane, the kernels spilled their logits). x(q, c): the lane's logits. share: 2 SK_LT words of
// LDS that nothing uses before the workgroup's next barrier (SHARE; 256 mixed rows with 100 biases each: 91.9 -> 90.0 us).
template <int NL, bool SHARE, class X>
__device__ __forceinline__ void ed_add(const EdArgs& ed, int rec, const EdList& list, uint32_t* share, int seg_lo, int n_in,
                                       X x) {
    const int lane = lane_id(), w = (int)threadIdx.x / WAVE;
    EdRow r = {nullptr, false, nullptr, nullptr, list.nb};
    const bool shared = SHARE && list.nb > WAVE && list.nb <= SK_LT;           // uniform
    int64_t i = 0;
    if (shared) {
        share[threadIdx.x] = (uint32_t)list.id;
        share[SK_LT + threadIdx.x] = __float_as_uint(list.val);
        __syncthreads();
    } else if (list.nb > WAVE) {
        ed_bias(r, ed, rec);
        if (r.nb > 4 * WAVE) i = ed_lower(r, seg_lo);
    }
#pragma unroll 1
    for (; i < r.nb; i += WAVE) {
        int id = list.id;
        float val = list.val;
        if (shared) {
            id = (int)share[i + lane];
            val = __uint_as_float(share[SK_LT + i + lane]);
        } else if (SHARE ? list.nb > WAVE : i > 0) {
            id = 0x7fffffff;
            if (i + lane < r.nb) {
                id = r.ids[i + lane];
                val = r.val[i + lane];
            }
        }
        const uint32_t rel = (uint32_t)id - (uint32_t)seg_lo;
        const bool here = rel < (uint32_t)n_in && ((rel >> 2) & (SK_LT - 1)) / WAVE == (uint32_t)w;
        if (__ballot(here) != 0ull) {                          // (most waves hold none of the 64)
#pragma unroll
            for (int q = 0; q < NL; ++q) {
                for (uint64_t m = __ballot(here && (int)(rel >> 2) / SK_LT == q); m; m &= m - 1) {
                    const int from = __ffsll((unsigned long long)m) - 1;
                    const uint32_t at = (uint32_t)read_lane((int)rel, from);
                    const float d = read_lane(val, from);
                    const bool mine = (int)((at >> 2) & (WAVE - 1)) == lane;
#pragma unroll
                    for (int c = 0; c < 4; ++c)                // (-0 leaves every number as it is)
                        x(q, c) = __fadd_rn(x(q, c), mine && (int)(at & 3u) == c ? d : -0.0f);
                }
            }
        }
        if (r.nb > 4 * WAVE && __ballot(id < seg_lo + n_in) != ~0ull) break;   // ascending: the rest lies behind
    }
}

// Token id's logit l with its mask and biases, on every lane (whole wave): NaN where it is not allowed.
__device__ __forceinline__ float ed_one(const EdRow& r, const EdList& list, float l, int id) {
    for (int64_t i = r.nb <= WAVE ? 0 : ed_lower(r, id); i < r.nb; i += WAVE) {
        const bool held = i == 0, in = i + lane_id() < r.nb;
        const int at = held ? list.id : in ? r.ids[i + lane_id()] : 0x7fffffff;
        const float val = held ? list.val : in ? r.val[i + lane_id()] : 0.0f;
        uint64_t m = __ballot(at == id);
        const bool more = m == ~0ull;
        for (; m; m &= m - 1) l = __fadd_rn(l, read_lane(val, __ffsll((unsigned long long)m) - 1));
        if (!more) break;
    }
    if (r.closed || (r.words && ((ld_const(r.words + (id >> 5)) >> (id & 31)) & 1u) == 0u)) l = __builtin_nanf("");
    return l;
}

// Four logits of type FS_F32, FS_BF16 or FS_F16 as floats; a resource over the segment's n_in logits (reads past them, in
// whole groups, are inside ld; past that, zeros).
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ i32x2 raw_buffer_load_i32x2(__amdgpu_buffer_rsrc_t rs, int voffset, int soffset, int aux)
    __asm("llvm.amdgcn.raw.ptr.buffer.load.v2i32");
template <int TYPE>
struct Logits4 {
    using raw = std::conditional_t<TYPE == FS_F32, f32x4, i32x2>;
    static constexpr int BYTES = TYPE == FS_F32 ? 4 : 2;
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* logits, int64_t at, int n_in) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>((const char*)logits + at * BYTES), (short)0,
                                                 ((n_in + 3) & ~3) * BYTES, 0x00020000);
    }
    // group: the place of the four in the segment
    static __device__ __forceinline__ raw load(__amdgpu_buffer_rsrc_t rs, int group) {
        if constexpr (TYPE == FS_F32) return raw_buffer_load_f32x4(rs, group * 16, 0, 2);    // nontemporal: read once
        else return raw_buffer_load_i32x2(rs, group * 8, 0, 2);
    }
    static __device__ __forceinline__ float half(uint32_t u) {
        if constexpr (TYPE == FS_BF16) return __uint_as_float(u << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)u);
    }
    static __device__ __forceinline__ void floats(const raw& t, float (&x)[4]) {
        if constexpr (TYPE == FS_F32) {
            x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
        } else {
            const uint32_t a = (uint32_t)t.x, b = (uint32_t)t.y;
            x[0] = half(a & 0xFFFFu); x[1] = half(a >> 16); x[2] = half(b & 0xFFFFu); x[3] = half(b >> 16);
        }
    }
    static __device__ __forceinline__ float one(const void* logits, int64_t at) {
        if constexpr (TYPE == FS_F32) return ((const float*)logits)[at];
        else return half(((const uint16_t*)logits)[at]);
    }
};

}  // namespace fs

#endif  // FERRO_EDIT_DEVICE_HPP
