// sampler_launch.hpp - the launchers that the host side (sampler_kernels.hip) calls in the other kernel files.
#ifndef FERRO_SAMPLER_LAUNCH_HPP
#define FERRO_SAMPLER_LAUNCH_HPP

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ferro_sampler.h"

namespace fs {

struct Args;
// The fused kernel's grid (segments, then merges), and its merge alone (alone != 0: each row from its logits).
hipError_t launch_segments(const Args& a, unsigned grid, hipStream_t st);
hipError_t launch_merges(const Args& a, unsigned rows, int nseg, int alone, hipStream_t st);

// The edits of a call's logits (fs_edits) beside the penalties: masks of allowed tokens and biases.
struct EdArgs {
    const uint32_t* mask;                  // [n_masks][mask_ld] words (NULL: no masks)
    int64_t mask_ld;
    int n_masks;
    const int32_t* mask_of;                // [rows] (NULL: row r takes mask r)
    const int32_t* bias_ids;               // CSR, ids ascending (bias_off NULL: no biases)
    const float* bias;
    const int64_t* bias_off;
};

constexpr int SK_LT = 256;                 // threads per segment workgroup
constexpr int SK_NW = SK_LT / 64;
constexpr int SK_K = 64;                   // largest k (one candidate per lane of the finishing wave)
constexpr int SK_GCAP = 128;               // groups of four a wave can hand to the expansion
constexpr int SK_CAP = 512;                // candidates a segment ranks in LDS
constexpr int SK_MAX_SEGS = 64;            // segments per row

struct SkArgs {
    const float* logits;
    int64_t ld;
    int B, V, nseg;
    const int32_t* hist;
    const int64_t* hist_off;
    const fs_row_params* params;
    const double* u;
    int32_t* tok;
    int kcap;
    int32_t* cand_ids;
    double* cand_probs;
    int32_t* keep;
    uint64_t* lists;                       // [B * nseg][SK_K]: each segment's top k, sorted, 0-padded
    uint32_t* ticket;                      // [B]: segments finished (left at 0)
    int32_t* err;
    uint64_t* trace;                       // FS_TRACE builds: per-workgroup phase timestamps (NULL: none)
    // verification windows (mode MODE_VERIFY; the host sends only windows without an active penalty here)
    int mode;
    const int32_t* rows;                   // token fed at each row
    const int64_t* row_off;                // stream -> rows
    int n_streams, eos;
    int32_t* accepted;
    uint32_t* stream_cnt;                  // [3 n_streams]: 64-bit counts + stop bits, 32-bit counts (left at 0)
    // a decode step (fs_decode_step_hp; NULL otherwise): draw streams and the histories with the tokens appended
    uint64_t* dmt;
    int32_t* didx;
    int32_t* out_hist;
    int64_t* out_hist_off;
    int64_t out_cap;
    EdArgs ed;                             // the edited instantiations: masks and biases
};

// flags of a launch: some row has an active penalty window; a decode step (the histories are copied); a verification
// window (mid-k kernel); a call with masks, with biases
constexpr int SK_MAY_PEN = 1, SK_COPY = 2, MK_VERIFY = 4, ED_MASKS = 8, ED_BIASES = 16;
// Float4 loads per thread that do not wait for the row's mask. 4, 8, 12, 16 of the 16: verification rows inside a string
// (almost all allowed) 17.5, 16.4, 16.4, 15.8 us, at a structural position (few allowed) 13.9, 14.8, 15.4, 16.0; 64 rows of
// 262144, a third of each kind and a sixth unmasked, 20.4, 21.2, 21.8, 21.6.
constexpr int ED_FIRST = 4;
// nl: float4 loads per thread (4, 8 or 16); the grid and k's layout come from the small-k plan. edited: under k.ed.
hipError_t launch_small_k(int nl, bool capped, bool all_greedy, bool edited, unsigned grid, int flags, const SkArgs& k,
                          hipStream_t st);

// The mid-k kernel: the small-k kernel's arguments (lists and ticket unused) and its own workspace.
constexpr int MK_LIST = 4096;              // entries of a row's candidate list
constexpr int MK_SPILL = 16384;            // entries of a row's list of penalised logits past those its segments keep in LDS
constexpr int MK_CTR = 128;                // words of a row's counters; from 64 on two per segment
// Segments per row, which wait for each other. A process has four hardware queues unless it asks for more, and each can
// hold one row whose segments are not all dispatched: 4 * 31 workgroups waiting leave room on an XCD (32 CUs of four
// workgroups), so calls of several contexts on several streams always go on. With 64 segments three calls could fill an
// XCD and wait out their limit. It is faster, too: 16 rows of 262144 logits, k 100: 18.1 us with 64 segments, 14.3 with 32.
constexpr int MK_MAX_SEGS = 32;
static_assert(64 + 2 * MK_MAX_SEGS <= MK_CTR, "");
struct MkArgs {
    SkArgs a;
    uint32_t* ctr;                         // [B][MK_CTR], left at 0
    uint32_t* qk;                          // [B][nseg][SK_NW][16] published lane maxima
    uint64_t* list;                        // [B][MK_LIST]
    uint64_t* spill;                       // [B][MK_SPILL]
    uint64_t* mass;                        // [B][2048] mass bins of rows with every token a candidate, left at 0
    uint32_t spins;                        // bounded wait for a row's segments (polls)
};
// all: some row samples with every token a candidate; edited: under m.a.ed
hipError_t launch_mid_k(int nl, bool capped, bool all, bool edited, unsigned grid, int flags, const MkArgs& m,
                        hipStream_t st);

// Edited logits written out (edit_kernels.hip). nl: groups of four logits per thread (2, 4 or 8).
struct EditArgs {
    const void* logits;
    int type;                              // FS_F32, FS_BF16, FS_F16
    int64_t ld;
    int B, V, nseg;
    const int32_t* hist;
    const int64_t* hist_off;
    const fs_row_params* params;           // NULL: no softcap, no penalties
    EdArgs ed;
    const int32_t* rows;                   // verification windows (n_streams > 0): params, histories and biases by stream
    const int64_t* row_off;
    int n_streams;
    float* out;
    int64_t out_ld;
    int32_t* err;
    uint32_t* any;                         // rows for the sampling kernels: [B], nonzero where a row has a candidate (else NULL)
    fs_row_params* rparams;                //   and their parameters, the penalties and the softcap off
};
hipError_t launch_edit(int nl, const EditArgs& e, hipStream_t st);

// The end of a sampling call on such rows: rows without a candidate get token -1, then a window's accepted prefixes.
struct EditEnd {
    int B;
    uint32_t* any;                         // left at 0
    const fs_row_params* rparams;
    int32_t* tok;
    int32_t* keep;
    int kcap;
    int32_t* cand_ids;
    double* cand_probs;
    const int32_t* rows;
    const int64_t* row_off;
    int n_streams, eos;
    int32_t* accepted;
};
hipError_t launch_edit_end(const EditEnd& e, hipStream_t st);

// Log-probabilities (logprob_kernel.hip).
constexpr int LP_TOP = 64;                 // largest n: one entry per lane of the finishing wave
constexpr int LP_LINE = 32;                // words of a 128-byte line
constexpr int LP_PARTS = 64;               // parts per row: the join holds one per lane
constexpr int LP_NL(int type) { return type == FS_F32 ? 4 : 8; }   // groups of four per thread in a chunk of 16 KB
constexpr int lp_group(int nseg) {         // logarithm of the lanes whose largest logit a wave publishes: 256 groups in a
    return nseg <= 4 ? 2 : nseg <= 8 ? 3 : nseg <= 16 ? 4 : nseg <= 32 ? 5 : 6;   // row of up to 64 parts
}
// What a row's waves publish: by part and wave [lists] the sums, their references, the logits above the chosen token's,
// bounds and list lengths, then the groups' largest logits.
constexpr size_t lp_row_bytes(int nseg) {
    const size_t lists = (size_t)nseg * SK_NW, keys = (lists * 64) >> lp_group(nseg);
    return (lists * (8 + 4 * 4) + keys * 4 + 127) / 128 * 128;
}
struct LpArgs {
    const void* logits;
    int64_t ld;
    int B, V, nseg, n;                     // nseg: parts per row
    const fs_row_params* params;           // NULL: no softcap, temperature 1
    EdArgs ed;
    const int32_t* tok;
    float* lp;
    int32_t* rank;
    int32_t* ids;                          // [B][n]
    float* top;
    char* rows;                            // [B][lp_row_bytes(nseg)]
    uint64_t* lists;                       // [B][nseg][SK_NW][LP_TOP]
    uint32_t* ticket;                      // [B][LP_LINE]: parts that have published (left at 0), in lines of their own
    int32_t* err;
};
hipError_t launch_logprobs(int type, const LpArgs& a, hipStream_t st);

// Beam search (beam_kernels.hip).
constexpr int BM_TOP = FS_MAX_TOP;         // new beams per stream, at most
struct BeamRow {                           // a row: what its candidates' scores follow from
    double a, z;                           // its score; the logarithm of its sum
    float M, T, eos;                       // its largest logit, its temperature, the logit that ends the text (-inf: none)
    int unused;
};
constexpr int BM_LIST = 2 * BM_TOP;        // entries of a wave's list
// Parts per row: more lists cost a row's end more than more workgroups save. 16 rows of 262144, 8 beams, with 64, 32, 16 parts
// 16.3, 14.8, 15.9 us; 4 rows of 151936, 64 beams, with 38, 32, 16 31.0, 22.8, 24.1.
constexpr int BM_PARTS = 32;
struct BeamArgs {
    int S, W, n, eos;                      // streams; rows of each where row_off is NULL
    int keep_slots;
    const int64_t* row_off;
    const float* score;                    // NULL: zeros
    int32_t* parent;                       // [S][n]
    int32_t* tok;
    float* out_score;
    int32_t* done;                         // [S]
    int32_t* done_parent;                  // [S][n]
    float* done_score;
    BeamRow* rows;                         // [rows]
    uint64_t* row_lists;                   // [rows][BM_TOP]
    uint32_t* ticket;                      // [S][LP_LINE]: what has ended of a stream (left at 0)
};
struct LpBeamArgs {                        // lp: params and biases by stream; lists of BM_LIST; tok and its outputs unused
    LpArgs lp;
    BeamArgs b;
};
hipError_t launch_beam_select(int type, const LpBeamArgs& a, hipStream_t st);

struct ForkArgs {
    const int32_t* hist;
    const int64_t* hist_off;
    const int64_t* row_off;                // NULL: n rows each
    int S, n;
    const int32_t* parent;
    const int32_t* tok;                    // NULL: nothing behind the histories
    int32_t* out;
    int64_t out_cap;
    int64_t* out_off;
    int32_t* err;
};
hipError_t launch_hist_fork(const ForkArgs& a, int cus, hipStream_t st);

constexpr int ST_MAX = 32;                 // states per launch (their records travel in the argument segment)
struct StateArgs {
    int n_states, alike, S, n_src, n;      // alike: all states have as many columns
    const int32_t* parent;
    const int32_t* from;
    const int32_t* len;
    int32_t* err;
    fs_state z[ST_MAX];
};
// vb: bytes per column (1 to 16); cols: columns of all states' and streams' blocks
hipError_t launch_reorder_states(int vb, StateArgs a, int64_t cols, int cus, hipStream_t st);

hipError_t launch_lookup_draft(int n_streams, const int32_t* hist, const int64_t* hist_off, const int32_t* kmax,
                               const int32_t* min_n, int eos, int32_t* draft, int draft_ld, int32_t* ndraft,
                               hipStream_t st);
hipError_t launch_hist_append(int S, const int32_t* hist, const int64_t* hist_off, const int32_t* tok,
                              const int64_t* row_off, const int32_t* count, int32_t* out, int64_t* out_off,
                              int64_t out_cap, int32_t* err, hipStream_t st);

}  // namespace fs

#endif  // FERRO_SAMPLER_LAUNCH_HPP
