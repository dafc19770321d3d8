// beam_device.hpp - the end of a beam search's selection: the best candidates of a stream's rows, the hypotheses that end and
// the places of the new beams.
// This code runs once per stream, behind everything else, from a cold instruction cache (about 40 ns per 64 bytes): loops stay
// rolled, and few candidates are put in order by counting those before each (a sort of 64 takes 1.7 us the first time).
#ifndef FERRO_BEAM_DEVICE_HPP
#define FERRO_BEAM_DEVICE_HPP

#include "sampler_device.hpp"
#include "sampler_launch.hpp"

namespace fs {

constexpr int BM_T = SK_LT;                // threads
constexpr int BM_ROWS = SK_NW;             // rows that a stream's last part ends by itself, a wave each

// The candidate of a row's edited logit x, in fp64 (-inf: none).
__device__ __forceinline__ double bm_score(const BeamRow& r, float x) {
    if (!(x > -__builtin_huge_valf()) || (x < r.M && !(r.M < __builtin_huge_valf()))) return -__builtin_huge_val();
    return r.a + ((x == r.M ? 0.0 : ((double)x - (double)r.M) / (double)r.T) - r.z);
}
// Scores as ordered integers (0: no candidate): the upper 51 bits, 39 of them the mantissa's, are compared; the lower 13 order
// equal ones where they are sorted, and lead back to the candidate.
constexpr int BM_LOW = 13;
constexpr uint32_t BM_OLD = 1u << 12;      // before others: of an earlier batch of rows (and 63 - its place), or the text's end
__device__ __forceinline__ uint64_t bm_key(double c, uint32_t low) {
    if (!((float)c > -__builtin_huge_valf())) return 0ull;
    const uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);
    return ((u >> 63 ? ~u : u | 0x8000000000000000ull) & ~(uint64_t)((1u << BM_LOW) - 1u)) | low;
}

constexpr int BM_HELD = 1024;              // entries of the lists kept in LDS
struct BeamJoin {                          // many rows or candidates
    BeamRow row[WAVE];
    uint64_t entry[BM_HELD];
    int from[2][BM_TOP], token[BM_TOP];    // of earlier batches: the beams (0), the ended (1)
    float value[2][BM_TOP];
};
struct BeamBest {                          // a stream's end
    union {
        BeamJoin join;
        uint64_t key[BM_T + 16];           // few: candidates, then what ends the text, one per thread; 0 past each
    };
    int from[BM_TOP], token[BM_TOP], efrom[BM_TOP], first[BM_TOP], place[BM_TOP];
    float value[BM_TOP], evalue[BM_TOP];
    int n_ends;
};
// (no larger than the parts' lists, whose place it takes)
struct BeamShared {
    union {
        uint64_t gather[SK_NW][512];       // a row's tokens, by the wave that ends it
        BeamBest best;
    };
    uint16_t at[SK_NW][LP_PARTS * SK_NW];
    BeamRow row[WAVE];                     // the stream's rows,
    uint64_t list[BM_T];                   // their candidates
    uint32_t turn;
};
__device__ __forceinline__ void bm_sync() {    // LDS stores and loads of one wave in order
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A row's results in memory, written and read on different XCDs: agent scope. A dead row wrote nothing.
constexpr int BM_WORDS = sizeof(BeamRow) / 8;
static_assert(sizeof(BeamRow) % 8 == 0, "a row's results are words");
__device__ __forceinline__ void bm_store_row(const BeamArgs& a, int64_t row, const BeamRow& br) {
    uint64_t w[BM_WORDS];
    __builtin_memcpy(w, &br, sizeof(br));
#pragma unroll
    for (int i = 0; i < BM_WORDS; ++i) st_agent(reinterpret_cast<uint64_t*>(a.rows + row) + i, w[i]);
}
__device__ __forceinline__ BeamRow bm_dead_row() { return {-__builtin_huge_val(), 0.0, 0.0f, 1.0f, -__builtin_huge_valf(), 0}; }
__device__ __forceinline__ BeamRow bm_load_row(const BeamArgs& a, int64_t row) {
    BeamRow br;
    uint64_t w[BM_WORDS];
    const float score = a.score ? a.score[row] : 0.0f;
#pragma unroll
    for (int i = 0; i < BM_WORDS; ++i) w[i] = ld_agent(reinterpret_cast<const uint64_t*>(a.rows + row) + i);
    __builtin_memcpy(&br, w, sizeof(br));
    return score > -__builtin_huge_valf() ? br : bm_dead_row();
}

// Of keys[0, n) those above key. The keys are 16-byte aligned, 0 up to a multiple of eight: eight at a time.
__device__ __forceinline__ int bm_above(const uint64_t* keys, int n, uint64_t key) {
    const ulonglong2* k = reinterpret_cast<const ulonglong2*>(keys);
    int r = 0;
#pragma unroll 1
    for (int i = 0; i < n; i += 8, k += 4) {
        const ulonglong2 a = k[0], b = k[1], c = k[2], d = k[3];
        r += (a.x > key ? 1 : 0) + (a.y > key ? 1 : 0) + (b.x > key ? 1 : 0) + (b.y > key ? 1 : 0) + (c.x > key ? 1 : 0) +
             (c.y > key ? 1 : 0) + (d.x > key ? 1 : 0) + (d.y > key ? 1 : 0);
    }
    return r;
}

// Few candidates: a thread each, its place the number of those before it. From sh.row and sh.list. Whole workgroup.
__device__ __forceinline__ bool bm_is_few(int m, int n) { return m <= WAVE && m * (n + 1) <= BM_T; }
__device__ __forceinline__ void bm_few(const BeamArgs& a, BeamShared& sh, int m, bool ends) {
    BeamBest& s = sh.best;
    const int t = threadIdx.x, n = a.n, E = m * n, E8 = (E + 7) & ~7, at = t < E ? t : t - E + E8;
    float v = -__builtin_huge_valf();
    uint64_t key = 0ull, e = 0ull;
    int r = 0;
    const bool beam = t < E, end = !beam && ends && t < E + m;
    if (beam || end) {
        r = beam ? t / n : t - E;
        const BeamRow br = sh.row[r];
        if (beam) e = sh.list[t];
        const double c = bm_score(br, end ? br.eos : e != 0ull ? val_of(comp_key(e)) : v);
        key = bm_key(c, beam ? (uint32_t)(BM_T - 1 - t) : BM_OLD + (uint32_t)(BM_T - 1 - t));
        v = (float)c;
    }
    if (t < 16) {                                              // (the places between and past them)
        if (t < E8 - E) s.key[E + t] = 0ull;
        if (t < 8) s.key[E8 + (ends ? m : 0) + t] = 0ull;
    }
    if (beam || end) s.key[at] = key;
    if (t < BM_TOP) {
        s.from[t] = -1;
        s.token[t] = -1;
        s.value[t] = -__builtin_huge_valf();
        s.efrom[t] = -1;
        s.evalue[t] = -__builtin_huge_valf();
    }
    if (t == 0) s.n_ends = 0;
    __syncthreads();
    if (key == 0ull) return;
    const int before = bm_above(s.key, E, key);
    if (beam) {
        if (before < n) {
            s.from[before] = r;
            s.token[before] = (int)comp_id(e);
            s.value[before] = v;
        }
    } else {
        const int ahead = bm_above(s.key + E8, m, key);
        if (before + ahead < n) {
            s.efrom[ahead] = r;
            s.evalue[ahead] = v;
            atomicAdd(&s.n_ends, 1);
        }
    }
}

// Any number of rows, by one wave: their lists, place by place (the rows' best first), 64 candidates at a time, sorted and
// merged into the best so far where one of them reaches the n-th. The first 64 of which none does end the walk: what follows
// is no better. Rows past the 64th are a batch of their own, whose candidates lose to equal ones of earlier batches.
__device__ __forceinline__ void bm_join(const BeamArgs& a, BeamShared& sh, int64_t r0, int m, bool ends) {
    BeamJoin& s = sh.best.join;
    const int lane = lane_id(), n = a.n;
    uint64_t acc = 0ull, end = 0ull;                           // sorted, one per lane
    int from = -1, token = -1, efrom = -1;
    float value = -__builtin_huge_valf(), evalue = value;
#pragma unroll 1
    for (int b = 0; b < m; b += WAVE) {
        const int k = m - b < WAVE ? m - b : WAVE;             // rows of this batch
        const uint64_t* lists = a.row_lists + (r0 + b) * BM_TOP;
        const int all = k * n;
        constexpr int U = 4;
        uint64_t e[U];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * WAVE + lane, p = i / k, r = i - p * k;
                e[u] = i < all ? ld_agent(lists + r * BM_TOP + p) : 0ull;
            }
        };
        BeamRow br = {0.0, 0.0, 0.0f, 1.0f, -__builtin_huge_valf(), 0};
        if (lane < k) br = bm_load_row(a, r0 + b + lane);
        fetch(0);
        s.row[lane] = br;
        if (b > 0) {
            s.from[0][lane] = from; s.token[lane] = token; s.value[0][lane] = value;
            s.from[1][lane] = efrom; s.value[1][lane] = evalue;
            acc = acc ? (acc & ~(uint64_t)((1u << BM_LOW) - 1u)) | BM_OLD | (uint32_t)(63 - lane) : 0ull;
            end = end ? (end & ~(uint64_t)((1u << BM_LOW) - 1u)) | BM_OLD | (uint32_t)(63 - lane) : 0ull;
        }
        bm_sync();
        bool more = true;
#pragma unroll 1
        for (int i0 = 0; more && i0 < all; i0 += U * WAVE) {
            if (i0 > 0) fetch(i0);
#pragma unroll 1
            for (int u = 0; u < U; ++u) {
                const uint64_t eu = u == 0 ? e[0] : u == 1 ? e[1] : u == 2 ? e[2] : e[3];
                const int i = i0 + u * WAVE + lane, p = i / k, r = i - p * k;
                if (i < BM_HELD) s.entry[i] = eu;
                uint64_t key = 0ull;
                if (eu != 0ull && i < all) key = bm_key(bm_score(s.row[r], val_of(comp_key(eu))), 4095u - (uint32_t)(r * 64 + p));
                const uint64_t nth = read_lane(acc, n - 1);
                if (more && i0 + u * WAVE < all) {             // uniform
                    if (__ballot(key > nth) != 0ull) acc = merge_top64(acc, sort64<false>(key));
                    else more = false;
                }
            }
        }
        bm_sync();
        // back from the keys to the candidates
        if (acc != 0ull) {
            const uint32_t low = (uint32_t)acc & ((1u << BM_LOW) - 1u);
            if (low & BM_OLD) {
                const int j = 63 - (int)(low & 63u);
                from = s.from[0][j]; token = s.token[j]; value = s.value[0][j];
            } else {
                const int at = (int)(4095u - low), r = at >> 6, p = at & 63, i = p * k + r;
                const uint64_t c = i < BM_HELD ? s.entry[i] : ld_agent(lists + r * BM_TOP + p);
                from = b + r;
                token = (int)comp_id(c);
                value = (float)bm_score(s.row[r], val_of(comp_key(c)));
            }
        }
        if (ends) {
            const uint64_t key = lane < k ? bm_key(bm_score(br, br.eos), 4095u - (uint32_t)(lane * 64)) : 0ull;
            if (__ballot(key != 0ull) != 0ull) {
                end = merge_top64(end, sort64<false>(key));
                if (end != 0ull) {
                    const uint32_t low = (uint32_t)end & ((1u << BM_LOW) - 1u);
                    if (low & BM_OLD) {
                        const int j = 63 - (int)(low & 63u);
                        efrom = s.from[1][j]; evalue = s.value[1][j];
                    } else {
                        const int r = (int)(4095u - low) >> 6;
                        efrom = b + r;
                        evalue = (float)bm_score(s.row[r], s.row[r].eos);
                    }
                }
            }
        }
        bm_sync();
    }
    // ended hypotheses: fewer than n candidates before them, ended ones among these (a prefix of the ended ones' order)
    int before = 0;
    if (__ballot(end != 0ull) != 0ull) {
#pragma unroll 1
        for (int j = 0; j < n; ++j) before += read_lane(acc, j) >> BM_LOW > end >> BM_LOW ? 1 : 0;
    }
    const bool ended = end != 0ull && before + lane < n;
    const bool live = lane < n && acc != 0ull;
    BeamBest& o = sh.best;
    o.from[lane] = live ? from : -1;
    o.token[lane] = live ? token : -1;
    o.value[lane] = live ? value : -__builtin_huge_valf();
    o.efrom[lane] = ended ? efrom : -1;
    o.evalue[lane] = ended ? evalue : -__builtin_huge_valf();
    const int d = __popcll(__ballot(ended));
    if (lane == 0) o.n_ends = d;
    bm_sync();
}

// Stream st without a candidate (one wave).
__device__ __forceinline__ void bm_nothing(const BeamArgs& a, int st) {
    const int lane = lane_id(), n = a.n;
    const int64_t o = (int64_t)st * n + lane;
    if (lane < n) {
        a.parent[o] = -1;
        a.tok[o] = -1;
        a.out_score[o] = -__builtin_huge_valf();
        if (a.done_parent) a.done_parent[o] = -1;
        if (a.done_score) a.done_score[o] = -__builtin_huge_valf();
    }
    if (a.done && lane == 0) a.done[st] = 0;
}

// The stream's outputs from what bm_few or bm_join found (one wave).
__device__ __forceinline__ void bm_finish(const BeamArgs& a, BeamBest& s, int st) {
    const int lane = lane_id(), n = a.n;
    const int64_t o = (int64_t)st * n;
    if (a.done && lane == 0) a.done[st] = s.n_ends;
    // the new beams' places: a parent's best child stays, the others take the free places in their order
    const int from = s.from[lane];
    int slot = lane;
    if (a.keep_slots) {
        s.first[lane] = WAVE;
        bm_sync();
        if (lane < n && from >= 0 && from < n) atomicMin(&s.first[from], lane);
        bm_sync();
        const bool stays = lane < n && from >= 0 && from < n && s.first[from] == lane;
        const bool open = lane < n && s.first[lane] == WAVE;   // (of place `lane`)
        const uint64_t om = __ballot(open), lm = __ballot(lane < n && !stays);
        if (open) s.place[mbcnt(om)] = lane;
        bm_sync();
        if (lane < n) slot = stays ? from : s.place[mbcnt(lm)];
    }
    if (lane < n) {
        a.parent[o + slot] = from;
        a.tok[o + slot] = s.token[lane];
        a.out_score[o + slot] = s.value[lane];
        if (a.done_parent) a.done_parent[o + lane] = s.efrom[lane];
        if (a.done_score) a.done_score[o + lane] = s.evalue[lane];
    }
}

// Whether this workgroup's share is the last of `of` (the ticket is left at 0). Whole workgroup, after its stores.
__device__ __forceinline__ bool bm_last(BeamShared& s, uint32_t* ticket, uint32_t share, uint32_t of) {
    vm_drain();
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t turn = __hip_atomic_fetch_add(ticket, share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + share;
        if (turn == of) st_agent(ticket, 0u);
        s.turn = turn;
    }
    __syncthreads();
    return s.turn == of;
}

// The stream of a beam's row: the largest s with row_off[s] <= row; its first row, its rows. Rows are most often dealt evenly.
struct BeamStream {
    int s, m;
    int64_t r0;
};
__device__ __forceinline__ BeamStream bm_stream(const BeamArgs& b, int row, int R) {
    if (!b.row_off) return {row / b.W, b.W, (int64_t)(row / b.W) * b.W};
    int s = (int)((int64_t)row * b.S / R);
    int64_t r0 = ld_const(b.row_off + s), r1 = ld_const(b.row_off + s + 1);
    if (row < r0 || row >= r1) {
        int s0 = 0, s1 = b.S;
        while (s1 - s0 > 1) {
            const int m = (s0 + s1) >> 1;
            if (ld_const(b.row_off + m) <= row) s0 = m; else s1 = m;
        }
        s = s0;
        r0 = ld_const(b.row_off + s);
        r1 = ld_const(b.row_off + s + 1);
    }
    return {s, (int)(r1 - r0), r0};
}

}  // namespace fs

#endif  // FERRO_BEAM_DEVICE_HPP
