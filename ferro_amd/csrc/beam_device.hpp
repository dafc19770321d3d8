// beam_device.hpp - the end of a beam search's selection: the best candidates of a stream's rows, the hypotheses that end and
// the places of the new beams.
// This code runs once per stream, behind everything else, from a cold instruction cache (about 40 ns per 64 bytes): loops stay
// rolled, and few candidates are put in order by counting those before each (a sort of 64 takes 1.7 us the first time): 16 of
// four rows 1.1 us, 64 and their ends of eight rows 1.8; 64 of 64 rows' 4096 (bm_many) about 7, by sorts and merges 13.7.
#ifndef FERRO_BEAM_DEVICE_HPP
#define FERRO_BEAM_DEVICE_HPP

#include "row_device.hpp"

namespace fs {

constexpr int BM_T = SK_LT;                // threads
constexpr int BM_ROWS = SK_NW;             // rows that a stream's last part ends by itself, a wave each

// The candidate of a row's edited logit x, in fp64 (-inf: none).
__device__ __forceinline__ double bm_score(const BeamRow& r, float x) {
    if (!(x > -__builtin_huge_valf()) || (x < r.M && !(r.M < __builtin_huge_valf()))) return -__builtin_huge_val();
    return r.a + ((x == r.M ? 0.0 : ((double)x - (double)r.M) / (double)r.T) - r.z);
}
// Scores as ordered integers (0: no candidate): the upper 51 bits, 39 of them the mantissa's, are compared; the lower 13 order
// equal ones by row and place, and make the integers distinct.
constexpr int BM_LOW = 13;
constexpr uint32_t BM_OLD = 1u << 12;      // before others: of earlier rows, or the text's end
__device__ __forceinline__ uint64_t bm_key(double c, uint32_t low) {
    if (!((float)c > -__builtin_huge_valf())) return 0ull;
    const uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);
    return ((u >> 63 ? ~u : u | 0x8000000000000000ull) & ~(uint64_t)((1u << BM_LOW) - 1u)) | low;
}

struct BeamBest {                          // a stream's end
    uint64_t key[BM_T + 16];               // candidates; 0 up to a multiple of eight (few: then what ends the text)
    uint64_t ekey[2 * BM_TOP + 8], ebest[BM_TOP];
    uint64_t entry[BM_T];
    int crow[BM_T];
    uint32_t hi[SK_NW][WAVE];
    float cvalue[BM_TOP];
    int cnt, room, again;
    int from[BM_TOP], token[BM_TOP], efrom[BM_TOP], first[BM_TOP], place[BM_TOP];
    float value[BM_TOP], evalue[BM_TOP];
    int n_ends;
};
// (it takes the place of the parts' lists; four workgroups of 40 KB fit a CU)
struct BeamShared {
    union {
        uint64_t gather[SK_NW][1024];      // a row's tokens, by the wave that ends it
        BeamBest best;
    };
    uint16_t at[SK_NW][BM_PARTS * SK_NW];
    BeamRow row[WAVE];                     // the stream's rows,
    uint64_t list[BM_T];                   // their candidates
    int cnt[SK_NW];
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

// Any number of rows, 64 at a time (a batch), a row per lane; wave w takes places w, w + 4, .. of their lists, which are in order.
// Of the first four places n reach a bound (as lp_nth); a wave goes on down the lists as long as one of them reaches it. The
// candidates so found (about 1.5 n) are put in order, a thread each, with the best of earlier batches; where there is no room for
// more, they are before the walk goes on.
constexpr uint64_t BM_MASK = ~(uint64_t)((1u << BM_LOW) - 1u);
__device__ __forceinline__ void bm_many(const BeamArgs& a, BeamShared& sh, int64_t r0, int m, bool ends) {
    BeamBest& s = sh.best;
    const int t = threadIdx.x, lane = lane_id(), w = t / WAVE, n = a.n;
    constexpr float NONE = -__builtin_huge_valf();
    uint32_t least = 1u;                                       // (of the keys' upper halves)
    int held = 0;                                              // of s.key: the best so far, in order
    if (t < BM_TOP) {
        s.ebest[t] = 0ull;
        s.efrom[t] = -1;
        s.evalue[t] = NONE;
    }
    __syncthreads();
#pragma unroll 1
    for (int b = 0; b < m; b += WAVE) {
        const int k = m - b < WAVE ? m - b : WAVE;             // rows of this batch
        const uint64_t* list = a.row_lists + (r0 + b + lane) * BM_TOP;
        auto fetch = [&](int p) { return lane < k && p < n ? ld_agent(list + p) : (uint64_t)0; };
        int p = w;
        uint64_t e = fetch(p), next = fetch(p + SK_NW);
        BeamRow br = bm_dead_row();
        if (lane < k) br = bm_load_row(a, r0 + b + lane);
        if (w == 0) {
            sh.row[lane] = br;
            if (lane < held) s.key[lane] = (s.key[lane] & BM_MASK) | BM_OLD | (uint32_t)(63 - lane);   // before equal ones
        }
        // what ends the text: the batch's rows (wave 2) and the best of earlier ones (wave 3), which come before equal ones
        uint64_t ek = 0ull;
        int efrom = -1;
        float evalue = NONE;
        if (ends && w == 3) {
            ek = s.ebest[lane];
            efrom = s.efrom[lane];
            evalue = s.evalue[lane];
        }
        uint64_t key = 0ull;
#pragma unroll 1
        for (int round = 0;; ++round) {
            bool go = true;
            auto key_now = [&](bool end) {
                const double c = bm_score(br, end ? br.eos : e ? val_of(comp_key(e)) : NONE);
                if (end) evalue = (float)c;
                return bm_key(c, 4095u - (uint32_t)(lane * 64 + (end ? 0 : p)));
            };
            if (round == 0) {
#pragma unroll 1
                for (int end = ends && w == 2 ? 1 : 0; end >= 0; --end) {
                    const uint64_t kk = key_now(end != 0);
                    if (end) {
                        ek = kk;
                        efrom = b + lane;
                    } else {
                        key = kk;
                    }
                }
                s.hi[w][lane] = (uint32_t)(key >> 32);
                if (w >= 2) s.ekey[t - 2 * WAVE] = ek;
                if (t < 8) s.ekey[2 * BM_TOP + t] = 0ull;
            }
            if (t == 0) {
                s.cnt = held;
                s.room = BM_T;
                s.again = 0;
            }
            __syncthreads();
            if (round == 0) {
                const uint32_t hi[4] = {s.hi[0][lane], s.hi[1][lane], s.hi[2][lane], s.hi[3][lane]};
                // (the lists are in order: all of these reach the least of the fourth places)
                const uint32_t reach = wave_min(lane >= k ? ~0u : hi[3] > 1u ? hi[3] : 1u);
                least = lp_nth(hi, 4 * k >= n && reach > least ? reach : least, n);
            }
#pragma unroll 1
            while (go) {
                const bool in = (uint32_t)(key >> 32) >= least;
                const uint64_t mm = __ballot(in);
                go = mm != 0ull;                               // (in order: no more below places that none reaches)
                if (!go) break;
                int at = 0;
                if (lane == 0) at = atomicAdd(&s.cnt, __popcll(mm));
                at = read_lane(at, 0);
                if (at + __popcll(mm) > BM_T) {                // no room: in the next round (what follows has none either)
                    if (lane == 0) {
                        atomicMin(&s.room, at);
                        s.again = 1;
                    }
                    break;
                }
                if (in) {
                    const int i = at + (int)mbcnt(mm);
                    s.key[i] = key;
                    s.entry[i] = e;
                    s.crow[i] = b + lane;
                }
                p += SK_NW;
                e = next;
                next = fetch(p + SK_NW);
                key = key_now(false);
            }
            __syncthreads();
            const int all = s.cnt < s.room ? s.cnt : s.room;
            const bool again = s.again != 0;
            if (t < 8) s.key[all + t] = 0ull;
            const uint64_t ck = t < all ? s.key[t] : 0ull, c = t < all ? s.entry[t] : 0ull;
            const int row = t < all ? s.crow[t] : -1;
            float value = t < BM_TOP ? s.cvalue[t] : NONE;     // (of the best of earlier rounds)
            if (t < all && t >= held) value = (float)bm_score(sh.row[row - b], val_of(comp_key(c)));
            __syncthreads();
            const int at = ck ? bm_above(s.key, all, ck) : BM_T;
            const int eat = round == 0 && ek ? bm_above(s.ekey, 2 * BM_TOP, ek) : BM_T;
            __syncthreads();
            if (at < n) {
                s.key[at] = ck;
                s.entry[at] = c;
                s.crow[at] = row;
                s.cvalue[at] = value;
            }
            if (round == 0 && t < BM_TOP) s.ebest[t] = 0ull;
            held = all < n ? all : n;
            if (t < 8) s.key[held + t] = 0ull;
            __syncthreads();
            if (eat < n) {
                s.ebest[eat] = (ek & BM_MASK) | BM_OLD | (uint32_t)(63 - eat);
                s.efrom[eat] = efrom;
                s.evalue[eat] = evalue;
            }
            if (held == n) least = (uint32_t)(s.key[n - 1] >> 32);
            if (!again) break;                                 // (uniform: a wave that has come to its end goes along)
        }
        __syncthreads();
    }
    if (t < BM_TOP) {
        const bool live = t < held;
        const uint64_t key = s.ebest[t];
        s.from[t] = live ? s.crow[t] : -1;
        s.token[t] = live ? (int)comp_id(s.entry[t]) : -1;
        s.value[t] = live ? s.cvalue[t] : NONE;
        // the ended: fewer than n candidates before them, the ended among these (so the first few in their order)
        bool ended = false;
        if (__ballot(key != 0ull) != 0ull) ended = key != 0ull && bm_above(s.key, held, key | ~BM_MASK) + t < n;
        const int d = __popcll(__ballot(ended));
        if (!ended) {
            s.efrom[t] = -1;
            s.evalue[t] = NONE;
        }
        if (t == 0) s.n_ends = d;
    }
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

// The stream's outputs from what bm_few or bm_many found (one wave).
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

// The stream of a beam's row: the largest s with row_off[s] <= row; its first row, its rows (of the R there are; 0: the row lies
// behind the last stream's, and would be counted as one of them). Rows are most often dealt evenly.
struct BeamStream {
    int s, m;
    int64_t r0;
};
__device__ __forceinline__ BeamStream bm_stream(const BeamArgs& b, int row, int R) {
    if (!b.row_off) return {row / b.W, b.W, (int64_t)(row / b.W) * b.W};
    int s = (int)((int64_t)row * b.S / R);
    int64_t r0 = ld_const(b.row_off + s), r1 = ld_const(b.row_off + s + 1);
    if (__builtin_expect((uint64_t)r0 > (uint64_t)row || row >= r1 || r1 > R, 0)) {
        int s0 = 0, s1 = b.S;
        while (s1 - s0 > 1) {
            const int m = (s0 + s1) >> 1;
            if (ld_const(b.row_off + m) <= row) s0 = m; else s1 = m;
        }
        s = s0;
        r0 = ld_const(b.row_off + s);
        r1 = ld_const(b.row_off + s + 1);
        r0 = r0 < 0 ? 0 : r0;
        r1 = row < r0 || row >= r1 ? r0 : r1 < R ? r1 : R;
    }
    return {s, (int)(r1 - r0), r0};
}

}  // namespace fs

#endif  // FERRO_BEAM_DEVICE_HPP
