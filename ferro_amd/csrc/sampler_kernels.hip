// sampler_kernels.hip - the C ABI of include/ferro_sampler.h: contexts, plans, the kernel choice and the launches; and the
// small kernels around sampling (softcap, penalties in place, draw streams).
#include "sampler_device.hpp"
#include "sampler_launch.hpp"

#include <utility>

namespace fs {

__global__ __launch_bounds__(256) void softcap_kernel(const float* in, float* out, int64_t n, float cap) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        out[i] = softcap_one(in[i], cap);
}

// In-place penalty pass (fs_penalize_batch): ferro's sample() leaves its host row penalised (sampler.cpp:11-18),
// and a caller that reads the row back afterwards (lm_cli.cpp:353) sees those values. One workgroup per
// (row, 8192-id chunk): the window's ids that fall in the chunk are counted in a 16-bit LDS table, then every
// counted logit is rewritten once with the same arithmetic as the sampling kernels.
constexpr int PEN_BLOCK = 256;
constexpr int PEN_CHUNK = 8192;

__global__ __launch_bounds__(PEN_BLOCK) void penalize_kernel(float* logits, int64_t ld, int V, const int32_t* hist,
                                                            const int64_t* hist_off, const fs_row_params* params,
                                                            int nchunk, int32_t* err) {
    __shared__ uint32_t cnt[PEN_CHUNK / 2];
    const int tid = threadIdx.x;
    const int row = (int)blockIdx.x / nchunk;
    const int lo = ((int)blockIdx.x - row * nchunk) * PEN_CHUNK;
    const fs_row_params p = ld_const(params + row);
    const bool rep_on = p.repetition_penalty != 1.0f;
    const bool fp_on = p.frequency_penalty != 0.0f || p.presence_penalty != 0.0f;
    if (!(rep_on || fp_on) || p.repeat_last_n == 0 || !hist || !hist_off) return;
    const int64_t h0 = ld_const(hist_off + row);
    const int64_t len = ld_const(hist_off + row + 1) - h0;
    const int64_t b = window_begin(len, p);
    if (b >= len) return;
    for (int i = tid; i < PEN_CHUNK / 2; i += PEN_BLOCK) cnt[i] = 0u;
    __syncthreads();
    bool ovf = false;
    for (int64_t i = b + tid; i < len; i += PEN_BLOCK) {
        const int id = hist[h0 + i];
        const uint32_t rel = (uint32_t)(id - lo);
        if (id >= 0 && id < V && rel < (uint32_t)PEN_CHUNK) {
            const uint32_t sh = (rel & 1u) * 16u;
            const uint32_t old = atomicAdd(&cnt[rel >> 1], 1u << sh);
            ovf |= ((old >> sh) & 0xFFFFu) == 0xFFFFu;
        }
    }
    if (ovf) atomicOr(err, FS_DEVERR_COUNT_OVERFLOW);
    __syncthreads();
    float* rowp = logits + (int64_t)row * ld + lo;
    for (int i = tid; i < PEN_CHUNK / 2; i += PEN_BLOCK) {
        const uint32_t c2 = cnt[i];
        if (c2 == 0u) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t c = (c2 >> (16 * q)) & 0xFFFFu;
            if (c != 0u) {                                  // a counted id is < V
                float l = rowp[2 * i + q];
                if (rep_on) l = l > 0.0f ? __fdiv_rn(l, p.repetition_penalty) : __fmul_rn(l, p.repetition_penalty);
                if (fp_on) l = __fsub_rn(l, __fadd_rn(__fmul_rn((float)c, p.frequency_penalty), p.presence_penalty));
                rowp[2 * i + q] = l;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ draw streams
// std::mt19937_64 (the standard's parameters: n = 312, m = 156, r = 31, a = 0xB5026F5AA96619E9, tempering
// u = 29 / d = 0x5555555555555555, s = 17 / b = 0x71D67FFFEDA60000, t = 37 / c = 0xFFF7EEE000000000, l = 43) per
// stream, and libstdc++'s generate_canonical<double, 53> of one 64-bit output: (double)x / 2^64, kept below 1.
// This is ferro::Sampler's draw (sampler.h:25,32; sampler.cpp:45-46) moved next to the sampler.

// One thread per stream. Stream s owns rows row_off[s] .. row_off[s+1]-1 (row_off NULL: row s alone); each row
// whose stream samples takes one draw, in row order; greedy streams take none and get u = 0. peek != 0 leaves the
// state unchanged (the draws are computed from it: at most MT_M draws past a twist).
__global__ __launch_bounds__(64) void drng_draw_kernel(uint64_t* mts, int32_t* idxs, int n_streams,
                                                       const int64_t* row_off, const fs_row_params* params,
                                                       double* u, int peek, int32_t* err) {
    const int sidx = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (sidx >= n_streams) return;
    uint64_t* mt = mts + (int64_t)sidx * MT_N;
    int idx = idxs[sidx];
    const int64_t r0 = row_off ? row_off[sidx] : sidx;
    const int64_t r1 = row_off ? row_off[sidx + 1] : sidx + 1;
    const bool smp = samples(params[sidx]);
    for (int64_t r = r0; r < r1; ++r) {
        if (!smp) { u[r] = 0.0; continue; }
        uint64_t y;
        if (!peek) {
            if (idx >= MT_N) { mt_twist(mt); idx = 0; }
            y = mt[idx++];
        } else {
            if (idx < MT_N) {
                y = mt[idx++];
            } else {
                const int k = idx - MT_N;                    // the k-th value of the next twist, from the old state
                if (k >= MT_M) { atomicOr(err, FS_DEVERR_INTERNAL); u[r] = 0.0; continue; }
                y = mt_twist_one(mt[k], mt[k + 1], mt[k + MT_M]);
                ++idx;
            }
        }
        u[r] = mt_canonical(mt_temper(y));
    }
    if (!peek) idxs[sidx] = idx;
}

// Advance stream s by counts[s] draws, or, for a stream that does not sample, by none.
__global__ __launch_bounds__(64) void drng_skip_kernel(uint64_t* mts, int32_t* idxs, int n_streams,
                                                       const int32_t* counts, const fs_row_params* params) {
    const int sidx = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (sidx >= n_streams || !samples(params[sidx])) return;
    uint64_t* mt = mts + (int64_t)sidx * MT_N;
    int idx = idxs[sidx];
    for (int32_t c = counts[sidx]; c > 0;) {
        if (idx >= MT_N) { mt_twist(mt); idx = 0; }
        const int take = MT_N - idx < c ? MT_N - idx : c;
        idx += take;
        c -= take;
    }
    idxs[sidx] = idx;
}

}  // namespace fs

// ================================================================================================ host side
struct fs_context {
    std::recursive_mutex mu;   // (an edited call holds it while the launches it is made of take it)
    int device = -1;
    int cus = 0;               // compute units of the device
    int xccs = 0;              // XCDs of the device (hipDeviceAttributeNumberOfXccs)
    bool seg_layout = true;    // the segment grid's hand-off holds on this device (XCDS % xccs == 0)
    int32_t* hflag = nullptr;  // host-mapped: a merge of an earlier call gave up (set by the kernel, read here)
    int32_t* hflag_dev = nullptr;
    bool frozen = false;       // a call under edits is being recorded into a graph: nothing may be allocated
    bool captured = false;     // a call was recorded into a graph: workspaces are retired, never freed, on growth
    std::vector<void*> retired;
    uint64_t* sk_lists = nullptr;   // small-k kernel: [slots][SK_K] sorted segment lists
    size_t sk_slots = 0;
    uint32_t* sk_ticket = nullptr;  // small-k kernel: [rows] segment tickets, left at 0
    size_t sk_rows = 0;
    uint32_t* mk_ctr = nullptr;     // mid-k kernel: [mk_ctr_rows][MK_CTR] counters, left at 0
    uint64_t* mk_list = nullptr;    //   [mk_list_rows][MK_LIST] candidate lists
    uint64_t* mk_spill = nullptr;   //   [mk_spill_rows][MK_SPILL] penalised logits (batches with penalties)
    uint64_t* mk_mass = nullptr;    //   [mk_mass_rows][2048] mass bins, left at 0 (batches with every token a candidate)
    uint32_t* mk_qk = nullptr;      //   [mk_segs][SK_NW][16] published lane maxima
    size_t mk_ctr_rows = 0, mk_list_rows = 0, mk_spill_rows = 0, mk_mass_rows = 0, mk_segs = 0;
    int mk_wait = 0;                //   calls that still go without trying again after an allocation failed
    uint64_t* cand = nullptr;
    size_t cand_slots = 0;     // chunk slots of CAP entries
    uint32_t* meta = nullptr;
    uint32_t* rhist = nullptr;  // [row_cap][RBINS]
    uint64_t* rmass = nullptr;  // [row_cap][LB]
    size_t row_cap = 0;
    uint32_t* stream_cnt = nullptr;
    size_t stream_cap = 0;
    int32_t* err = nullptr;        // [0]: error bits; [1]: dirty (a merge gave up; see fs_device_error); [2..3]: hflag_dev
    uint32_t merge_spins = fs::MERGE_SPINS;
    float* ed_rows = nullptr;          // calls under edits: [ed_logits] edited logits,
    fs_row_params* ed_params = nullptr;//   [ed_param_rows] their parameters,
    uint32_t* ed_any = nullptr;        //   [ed_any_rows] whether a row has a candidate (left at 0),
    double* ed_u = nullptr;            //   [ed_u_rows] a decode step's draws,
    int64_t* ed_off = nullptr;         //   [ed_off_rows] zeros: the offsets of empty histories
    size_t ed_logits = 0, ed_param_rows = 0, ed_any_rows = 0, ed_u_rows = 0, ed_off_rows = 0;
    char* lp_row = nullptr;            // fs_logprobs: [lp_row_bytes] what the rows' waves publish,
    uint32_t* lp_ticket = nullptr;     //   [lp_rows][LP_LINE] their tickets, left at 0,
    uint64_t* lp_lists = nullptr;      //   [lp_list_cap] entries of their lists
    size_t lp_row_bytes = 0, lp_rows = 0, lp_list_cap = 0;
    fs::BeamRow* bm_rows = nullptr;    // fs_beam_select: [bm_row_cap] the rows' results
    uint64_t* bm_lists = nullptr;      //   [bm_list_cap][BM_TOP] and lists,
    uint32_t* bm_ticket = nullptr;     //   [bm_streams][LP_LINE] the streams' tickets, left at 0
    size_t bm_row_cap = 0, bm_list_cap = 0, bm_streams = 0;
    int static_dev = -1;       // device whose static workspace fs_sample_batch_static used with this context
    uint64_t* trace = nullptr; // FS_TRACE builds: phase timestamps, trace_cap entries (fs_trace_set)
    int64_t trace_cap = 0;
    fs_row_params* greedy = nullptr;      // fs_argmax_batch without parameters: [greedy_cap] greedy records
    size_t greedy_cap = 0;
    std::vector<fs_row_params> h_greedy;  //   and their host copy (the small-k kernel's greedy path)
};

namespace fs {
__global__ __launch_bounds__(256) void zero_words_kernel(uint32_t* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0u;
}
// n parameter records of a greedy row without penalties (fs_argmax_batch without parameters)
__global__ __launch_bounds__(256) void greedy_params_kernel(fs_row_params* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        fs_row_params r;
        r.temperature = 0.0f; r.top_k = 1; r.top_p = 1.0f; r.min_p = 0.0f; r.repetition_penalty = 1.0f;
        r.frequency_penalty = 0.0f; r.presence_penalty = 0.0f; r.repeat_last_n = 0; r.penalty_from = 0;
        r.softcap = 0.0f;
        p[i] = r;
    }
}
}  // namespace fs

namespace {

// Zero n words on st with a fill kernel (no hipMemsetAsync: the call may be recorded into a graph).
void clear_words(hipStream_t st, void* p, int64_t n) {
    if (!p || n <= 0) return;
    const int64_t blocks = std::min<int64_t>(1024, (n + 255) / 256);
    hipLaunchKernelGGL(fs::zero_words_kernel, dim3((unsigned)blocks), dim3(256), 0, st, (uint32_t*)p, n);
}

// A workspace buffer that is replaced: freed, or, once a call of the context has been recorded into a HIP graph
// (whose replays keep using the old addresses), kept until fs_destroy.
void release(fs_context* c, void* p) {
    if (!p) return;
    if (c->captured) c->retired.push_back(p);
    else (void)hipFree(p);
}

// A failed allocation is this call's answer, not the next launch's (whose error check would still find it).
int no_memory() {
    (void)hipGetLastError();
    return FS_E_NOMEM;
}

int grow(fs_context* c, size_t slots, size_t rows, size_t streams) {
    if (c->frozen && (slots > c->cand_slots || rows > c->row_cap || streams > c->stream_cap || !c->hflag || !c->err))
        return FS_E_NOMEM;
    if (slots > c->cand_slots) {
        release(c, c->cand);
        release(c, c->meta);
        c->cand = nullptr; c->meta = nullptr; c->cand_slots = 0;
        if (hipMalloc(&c->cand, slots * fs::CAP * sizeof(uint64_t)) != hipSuccess) return no_memory();
        if (hipMalloc(&c->meta, slots * 2 * sizeof(uint32_t)) != hipSuccess) return no_memory();
        c->cand_slots = slots;
    }
    if (rows > c->row_cap) {
        release(c, c->rhist);
        release(c, c->rmass);
        c->rhist = nullptr; c->rmass = nullptr; c->row_cap = 0;
        if (hipMalloc(&c->rhist, rows * fs::RBINS * sizeof(uint32_t)) != hipSuccess) return no_memory();
        if (hipMemset(c->rhist, 0, rows * fs::RBINS * sizeof(uint32_t)) != hipSuccess) return FS_E_HIP;
        if (hipMalloc(&c->rmass, rows * fs::LB * sizeof(uint64_t)) != hipSuccess) return no_memory();
        if (hipMemset(c->rmass, 0, rows * fs::LB * sizeof(uint64_t)) != hipSuccess) return FS_E_HIP;
        c->row_cap = rows;
    }
    if (streams > c->stream_cap) {
        release(c, c->stream_cnt);
        c->stream_cnt = nullptr; c->stream_cap = 0;
        if (hipMalloc(&c->stream_cnt, streams * sizeof(uint32_t)) != hipSuccess) return no_memory();
        if (hipMemset(c->stream_cnt, 0, streams * sizeof(uint32_t)) != hipSuccess) return FS_E_HIP;
        c->stream_cap = streams;
    }
    if (!c->hflag) {
        if (hipHostMalloc((void**)&c->hflag, sizeof(int32_t), hipHostMallocMapped) != hipSuccess) return no_memory();
        *(volatile int32_t*)c->hflag = 0;
        if (hipHostGetDevicePointer((void**)&c->hflag_dev, c->hflag, 0) != hipSuccess) return FS_E_HIP;
    }
    if (!c->err) {
        // error bits, dirty flag, then the device address of the host-mapped give-up flag (read by a give-up only)
        int32_t h[4] = {0, 0, 0, 0};
        const uint64_t fa = (uint64_t)(uintptr_t)c->hflag_dev;
        memcpy(h + 2, &fa, sizeof(fa));
        if (hipMalloc(&c->err, sizeof(h)) != hipSuccess) return no_memory();
        if (hipMemcpy(c->err, h, sizeof(h), hipMemcpyHostToDevice) != hipSuccess) return FS_E_HIP;
    }
    return FS_OK;
}

// Segments: at most two per CU over the whole batch (all resident at once: a second round of a few workgroups
// would double the time), at least one per row; a segment streams >= 1 full tile of 4096 logits. The merge
// handles each row's partial last tile (all of a row shorter than one tile). Sets a.nseg / a.seg_tiles and the
// workspace the call needs (items = (row, segment) slots).
// max_slots > 0 caps the workspace slots (XCDS * nseg * ceil(rows / XCDS)) by taking fewer segments per row; one
// segment per row always fits rows <= max_slots.
int plan(int cus, fs::Args& a, int64_t rows, int64_t& items, int64_t& seg_grid, int64_t max_slots = 0,
         int per_cu = 2) {
    const int64_t tiles_row = a.V / fs::TILE;
    const int64_t per_slot = (rows + fs::XCDS - 1) / fs::XCDS;
    a.nseg = 0;
    a.seg_tiles = 1;
    if (tiles_row > 0) {
        int64_t want = ((int64_t)per_cu * (int64_t)cus) / rows;
        if (want < 1) want = 1;
        if (want > tiles_row) want = tiles_row;
        if (want > fs::BLOCK - 1) want = fs::BLOCK - 1;   // the merge gives each list (segments + tail) a thread
        for (;;) {
            a.seg_tiles = (int)((tiles_row + want - 1) / want);
            a.nseg = (int)((tiles_row + a.seg_tiles - 1) / a.seg_tiles);
            if (max_slots <= 0 || want <= 1 || (int64_t)fs::XCDS * a.nseg * per_slot <= max_slots) break;
            --want;
        }
    }
    if (a.nseg > fs::MAX_SEGS) return FS_E_INVALID;
    items = rows * a.nseg;
    if (items > 0x7fffffff) return FS_E_INVALID;
    // one workgroup per (row, segment), the rows dealt to XCDS slots (segment_kernel); each segment workgroup's
    // list slot is its index, so the workspace holds seg_grid slots
    seg_grid = items > 0 ? (int64_t)fs::XCDS * a.nseg * ((rows + fs::XCDS - 1) / fs::XCDS) : 0;
    if (seg_grid > 0x7fffffff) return FS_E_INVALID;
    items = seg_grid;
    // balanced layouts (sampling, >= 2 segments per row, >= 2 rows on some XCD, <= WAVE rows per XCD)
    // Balanced layouts: sampling, >= 2 segments per row, 16 to WAVE rows per XCD. Computing the layout delays every
    // workgroup by about 2 us, which pays on large mixed batches (B=256 x V=262144 with k from 1 to 2048: -20 us)
    // but not on small ones.
    a.balance = (a.mode == fs::MODE_SAMPLE && a.nseg >= 2 && (rows + fs::XCDS - 1) / fs::XCDS >= 16 &&
                 (rows + fs::XCDS - 1) / fs::XCDS <= fs::WAVE) ? 1 : 0;
    return FS_OK;
}

// Launches the sampling grid on a bound workspace (a.cand / meta / rhist / stream_cnt / err / dirty).
int launch_planned(const fs::Args& a, int64_t rows, int64_t seg_grid, hipStream_t st) {
    if (seg_grid > 0) {                            // the segments, then one merging workgroup per row (same grid)
        const int64_t grid = seg_grid + (int64_t)fs::XCDS * ((rows + fs::XCDS - 1) / fs::XCDS);
        if (grid > 0x7fffffff) return FS_E_INVALID;
        return fs::launch_segments(a, (unsigned)grid, st) == hipSuccess ? FS_OK : FS_E_HIP;
    }
    return fs::launch_merges(a, (unsigned)rows, a.nseg, 0, st) == hipSuccess ? FS_OK : FS_E_HIP;
}

// Every row sampled alone by one workgroup from its logits (a device whose XCD layout the segment grid's hand-off
// does not fit).
int launch_alone(fs::Args a, int64_t rows, hipStream_t st) {
    a.nseg = 0;
    a.balance = 0;
    return fs::launch_merges(a, (unsigned)rows, 0, 1, st) == hipSuccess ? FS_OK : FS_E_HIP;
}

// The segment grid places a row's segments and its merging workgroup on workgroups of one index class mod XCDS, so
// that they share an XCD (and its L2) under round-robin dispatch over the device's XCDs: that holds when the XCD
// count divides XCDS (8, 4, 2 or 1: every MI355X partition mode). On other devices every row is sampled alone.
bool layout_fits(int xccs) { return xccs >= 1 && fs::XCDS % xccs == 0; }

int device_of(fs_context* ctx) {
    if (ctx->device < 0) {
        int dev = -1;
        if (hipGetDevice(&dev) != hipSuccess) return FS_E_HIP;
        if (hipDeviceGetAttribute(&ctx->cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
            return FS_E_HIP;
        int x = 0;
        if (hipDeviceGetAttribute(&x, hipDeviceAttributeNumberOfXccs, dev) != hipSuccess) return FS_E_HIP;
        ctx->xccs = x;
        ctx->seg_layout = layout_fits(x);
        ctx->device = dev;
    }
    return FS_OK;
}

// Whether an earlier call's merge gave up waiting for its segments (the kernel sets the host-mapped flag). The
// caller then enqueues, ahead of its own launch, fill kernels that clear what the late segments may have left (they
// have finished once the stream reaches the fills), so the call runs normally instead of computing every row alone;
// it returns FS_W_RECOVERED. The error bits stay for fs_device_error.
bool gave_up(int32_t* flag) {
    if (!flag || *(volatile int32_t*)flag == 0) return false;
    *(volatile int32_t*)flag = 0;
    return true;
}

bool capturing(hipStream_t st) {
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(st, &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}

// ---- small-k kernel (fs_sample_batch_hp)
// Whether every row of the batch fits the small-k kernel: greedy, or k = min(top_k or V, V) <= SK_K, with no
// frequency / presence penalty (h: the host copy of the parameters).
// A batch whose rows cost very differently: rows sampled with 64 < k <= KMAX beside greedy or k <= 64 rows, none on
// the whole-row path (k > KMAX), 16 to 64 rows per XCD (the balanced layout). The host copy of the parameters shows
// the mix, and such batches take about four segments per CU instead of two, which gives the balanced layout finer
// shares to apportion. It is reached by batches the mid-k kernel does not take (more than 262144 logits, or too few for
// their largest k). k spread evenly over 1 to 2048 by its logarithm, with two segments per CU and with four: 384 rows of
// 262208 logits 224 us and 167, of 50000 106 and 88; but 256 rows of 262208 116 and 131, of 32000 89 and 96 (the rule dates
// from 256 rows of 262144, which the mid-k kernel now has). Uniform batches lose with more segments (more lists to merge, a
// second round of workgroups).
bool mixed_merges(const fs_row_params* h, int64_t B, int32_t V) {
    const int64_t per_x = (B + fs::XCDS - 1) / fs::XCDS;
    if (per_x < 16 || per_x > fs::WAVE) return false;
    bool heavy = false, light = false;
    for (int64_t b = 0; b < B; ++b) {
        const fs_row_params& p = h[b];
        const bool greedy = !(p.temperature > 0.0f && p.top_k != 1);
        const int64_t k = greedy ? 1 : ((p.top_k > 0 && p.top_k < V) ? p.top_k : V);
        if (k > fs::KMAX) return false;
        if (k > 64) heavy = true;
        else light = true;
    }
    return heavy && light;
}

bool small_k_batch(const fs_row_params* h, int64_t B, int32_t V) {
    for (int64_t b = 0; b < B; ++b) {
        const fs_row_params& p = h[b];
        const bool greedy = p.temperature <= 0.0f || p.top_k == 1;
        if (!greedy && (p.frequency_penalty != 0.0f || p.presence_penalty != 0.0f)) return false;
        const int64_t k = (p.top_k > 0 && p.top_k < V) ? p.top_k : V;
        if (!greedy && k > fs::SK_K) return false;
    }
    return true;
}

// Logits per thread (NL float4 loads) and segments per row: the largest segments that still give every CU four
// workgroups, else the smallest (most workgroups) whose row fits SK_MAX_SEGS lists; 0 when none does.
int small_k_plan(int cus, int64_t B, int32_t V, int& nl, int& nseg) {
    nl = 0;
    nseg = 0;
    const int nls[3] = {16, 8, 4};
    for (int i = 0; i < 3; ++i) {
        const int64_t seg = (int64_t)fs::SK_LT * nls[i] * 4;
        const int64_t n = ((int64_t)V + seg - 1) / seg;
        if (n > fs::SK_MAX_SEGS) break;
        nl = nls[i];
        nseg = (int)n;
        if (B * n >= 4 * (int64_t)cus) break;
    }
    return nl > 0 ? FS_OK : FS_E_INVALID;
}

// The same for calls under edits: the smallest segments that leave few lists to a row's end and do not crowd the tickets, two
// workgroups per CU of 4096 logits or three of 8192 (greedy rows, whose lists are one entry: four), else 16384. Measured with
// 4, 8 and 16 loads, k 64: 1 row of 65536 logits 9.9, 10.1, 11.2 us; 32 rows 12.6, 12.6, 13.5; 64 rows 15.5, 13.5, 14.4; 200
// rows 31.8, 23.7, 19.3; 1 row of 151936 18.9, 11.3, 11.3; 30 rows of 262144 33.4, 19.6, 16.2; 48 rows 42.6, 26.4, 18.6; 40 of
// 131072 22.9, 14.7, 15.4. Greedy: 1 row of 262144 6.5, 7.1, 8.5; 12 rows 14.6, 10.6, 11.1; 128 of 65536 16.9, 12.7, 13.7.
int small_k_edited_plan(int cus, int64_t B, int32_t V, bool greedy, int& nl, int& nseg) {
    for (const int l : {4, 8, 16}) {
        const int64_t seg = (int64_t)fs::SK_LT * l * 4, n = ((int64_t)V + seg - 1) / seg;
        if (n > fs::SK_MAX_SEGS) continue;
        const int per_cu = l == 4 ? 2 : greedy ? 4 : 3;
        nl = l;
        nseg = (int)n;
        if ((greedy || n <= 16) && B * n <= per_cu * (int64_t)cus) break;
    }
    return nl > 0 ? FS_OK : FS_E_INVALID;
}

int grow_small(fs_context* c, size_t slots, size_t rows) {
    if (c->frozen && (slots > c->sk_slots || rows > c->sk_rows)) return FS_E_NOMEM;
    if (slots > c->sk_slots) {
        release(c, c->sk_lists);
        c->sk_lists = nullptr; c->sk_slots = 0;
        if (hipMalloc(&c->sk_lists, slots * fs::SK_K * sizeof(uint64_t)) != hipSuccess) return no_memory();
        c->sk_slots = slots;
    }
    if (rows > c->sk_rows) {
        release(c, c->sk_ticket);
        c->sk_ticket = nullptr; c->sk_rows = 0;
        if (hipMalloc(&c->sk_ticket, rows * sizeof(uint32_t)) != hipSuccess) return no_memory();
        if (hipMemset(c->sk_ticket, 0, rows * sizeof(uint32_t)) != hipSuccess) return FS_E_HIP;
        c->sk_rows = rows;
    }
    return FS_OK;
}

// Verification windows fit the small-k kernel when every stream does and none has an active penalty (a row's
// history would then include the drafts fed before it).
bool small_k_windows(const fs_row_params* h, int64_t S, int32_t V) {
    if (!small_k_batch(h, S, V)) return false;
    for (int64_t s = 0; s < S; ++s)
        if ((h[s].repetition_penalty != 1.0f || h[s].frequency_penalty != 0.0f || h[s].presence_penalty != 0.0f) &&
            h[s].repeat_last_n != 0)
            return false;
    return true;
}

// B greedy parameter records without penalties on the device (filled by a kernel on st, no memset: the call may be
// captured) and on the host. The caller holds ctx->mu.
int greedy_params(fs_context* ctx, int64_t B, hipStream_t st) {
    if ((size_t)B <= ctx->greedy_cap) return FS_OK;
    const size_t cap = std::max<size_t>((size_t)B, 2 * ctx->greedy_cap);
    release(ctx, ctx->greedy);
    ctx->greedy = nullptr;
    ctx->greedy_cap = 0;
    if (hipMalloc(&ctx->greedy, cap * sizeof(fs_row_params)) != hipSuccess) return no_memory();
    const int64_t blocks = std::min<int64_t>(1024, ((int64_t)cap + 255) / 256);
    hipLaunchKernelGGL(fs::greedy_params_kernel, dim3((unsigned)blocks), dim3(256), 0, st, ctx->greedy, (int64_t)cap);
    if (hipGetLastError() != hipSuccess) return FS_E_HIP;
    fs_row_params r = {};
    r.temperature = 0.0f; r.top_k = 1; r.top_p = 1.0f; r.repetition_penalty = 1.0f;
    ctx->h_greedy.assign(cap, r);
    ctx->greedy_cap = cap;
    return FS_OK;
}

// The small-k kernel's plan for n host parameter records (B rows, or n_streams windows with `verify`): false when
// the batch does not fit it (the fused kernel runs). nl / nseg: its segments; all_greedy: the greedy-only form;
// capped: some row has a softcap; may_pen: some row has an active penalty window.
struct SmallKChoice {
    int nl = 0, nseg = 0;
    bool all_greedy = true, capped = false, may_pen = false;
};
bool small_k_choice(int cus, const fs_row_params* h, int64_t n, int64_t B, int32_t V, bool verify, SmallKChoice& c,
                    bool edited = false) {
    if (verify ? !small_k_windows(h, n, V) : !small_k_batch(h, n, V)) return false;
    if (small_k_plan(cus, B, V, c.nl, c.nseg) != FS_OK) return false;
    bool counts = false;
    for (int64_t b = 0; b < n; ++b) {
        const fs_row_params& p = h[b];
        const bool fp = p.frequency_penalty != 0.0f || p.presence_penalty != 0.0f;
        c.all_greedy = c.all_greedy && !(p.temperature > 0.0f && p.top_k != 1);
        c.capped |= p.softcap > 0.0f;
        c.may_pen |= (p.repetition_penalty != 1.0f || fp) && p.repeat_last_n != 0;
        counts |= fp && p.repeat_last_n != 0;
    }
    if (edited && !counts) (void)small_k_edited_plan(cus, B, V, c.all_greedy, c.nl, c.nseg);
    if ((int64_t)fs::XCDS * c.nseg * ((B + fs::XCDS - 1) / fs::XCDS) > 0x7fffffff) return false;
    return !(counts && c.nl != 4);               // count tables fit segments of 4096 logits only: the fused kernel
}

fs::SkArgs row_args(const fs_context* ctx, const fs::Args& a, int nseg) {
    fs::SkArgs k = {};
    k.logits = a.logits; k.ld = a.ld; k.B = a.B; k.V = a.V; k.nseg = nseg;
    k.hist = a.hist; k.hist_off = a.hist_off; k.params = a.params; k.u = a.u; k.tok = a.tok; k.kcap = a.kcap;
    k.cand_ids = a.cand_ids; k.cand_probs = a.cand_probs; k.keep = a.keep;
    k.err = ctx->err;
    k.mode = a.mode; k.rows = a.rows; k.row_off = a.row_off; k.n_streams = a.n_streams; k.eos = a.eos;
    k.accepted = a.accepted; k.stream_cnt = ctx->stream_cnt;
    k.dmt = a.dmt; k.didx = a.didx; k.out_hist = a.out_hist; k.out_hist_off = a.out_hist_off; k.out_cap = a.out_cap;
    return k;
}

int edit_flags(const fs::EdArgs* ed) {
    return !ed ? 0 : (ed->mask ? fs::ED_MASKS : 0) | (ed->bias_off ? fs::ED_BIASES : 0);
}

// Whether the batch fits the small-k kernel (fits; else nothing grows), and the workspace it needs there. ed: the rows'
// masks and biases. The caller holds ctx->mu and has the context's device.
int reserve_small(fs_context* ctx, const fs::Args& a, const fs_row_params* h_params, const fs::EdArgs* ed, SmallKChoice& ch,
                  bool& fits) {
    fits = false;
    const bool verify = a.mode == fs::MODE_VERIFY;
    if (!ctx->seg_layout) return FS_OK;
    if (!small_k_choice(ctx->cus, h_params, verify ? (int64_t)a.n_streams : (int64_t)a.B, a.B, a.V, verify, ch,
                        ed != nullptr))
        return FS_OK;
    if (ed && ed->bias_off && ch.capped) return FS_OK;     // (the softcap, late in this kernel, comes before the biases)
    // the error word and the verify stream counters: a 64-bit word per stream, then the 32-bit counters of streams
    // longer than 32 rows
    int rc = grow(ctx, 0, 0, verify ? 3 * (size_t)a.n_streams : 0);
    if (rc != FS_OK) return rc;
    int most = ch.nseg;
    if (ed && !ctx->frozen) {                      // (a shape warmed up with any parameters records with others)
        int l = 0, n = 0;
        for (const bool greedy : {false, true})
            if (small_k_edited_plan(ctx->cus, a.B, a.V, greedy, l, n) == FS_OK) most = std::max(most, n);
        if (small_k_plan(ctx->cus, a.B, a.V, l, n) == FS_OK) most = std::max(most, n);
    }
    rc = grow_small(ctx, (size_t)a.B * most, (size_t)a.B);
    fits = rc == FS_OK;
    return rc;
}

// Launches the small-k kernel when the batch fits it; *used = false (nothing launched) otherwise. a.mode selects
// sampling (h_params: B records) or verification windows (h_params: n_streams records).
// h_params NULL: every row greedy without penalties (fs_argmax_batch without parameters): the context's greedy
// records stand for the parameters, on the device and the host. ed: the rows' masks and biases.
int launch_small(fs_context* ctx, const fs::Args& a_in, const fs_row_params* h_params, hipStream_t st, bool& used,
                 const fs::EdArgs* ed = nullptr) {
    used = false;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    int rc = device_of(ctx);
    if (rc != FS_OK) return rc;
    fs::Args a = a_in;
    if (!h_params) {
        rc = greedy_params(ctx, a.B, st);
        if (rc != FS_OK) return rc;
        h_params = ctx->h_greedy.data();
        a.params = ctx->greedy;
    }
    const bool verify = a.mode == fs::MODE_VERIFY;
    SmallKChoice ch;
    bool fits = false;
    rc = reserve_small(ctx, a, h_params, ed, ch, fits);
    if (rc != FS_OK || !fits) return rc;
    const int nl = ch.nl, nseg = ch.nseg;
    const int64_t per_x = ((int64_t)a.B + fs::XCDS - 1) / fs::XCDS;
    const int64_t grid = (int64_t)fs::XCDS * nseg * per_x;
    if (capturing(st)) ctx->captured = true;
    fs::SkArgs k = row_args(ctx, a, nseg);
    k.lists = ctx->sk_lists; k.ticket = ctx->sk_ticket;
    if (ed) k.ed = *ed;
    k.trace = nullptr;
#ifdef FS_TRACE
    if (ctx->trace && grid * fs::TRACE_W <= ctx->trace_cap) k.trace = ctx->trace;
#endif
    const bool capped = ch.capped, all_greedy = ch.all_greedy;
    bool may_pen = ch.may_pen;
    // a verification window reaches this kernel only without an active penalty (small_k_windows)
    may_pen = may_pen && !verify && a.hist && a.hist_off;
    const int flags = (may_pen ? fs::SK_MAY_PEN : 0) | (a.out_hist_off ? fs::SK_COPY : 0) | edit_flags(ed);
    if (fs::launch_small_k(nl, capped, all_greedy, ed != nullptr, (unsigned)grid, flags, k, st) != hipSuccess) return FS_E_HIP;
    used = true;
    return FS_OK;
}

// ---- mid-k kernel (fs_sample_batch_hp, fs_verify_hp, fs_decode_step_hp)
// Every row greedy or sampling from k <= 2048 candidates or from every token, with any penalty. The row's bound comes from its lanes'
// maxima (one per 4 * nl logits): twice as many as the largest k keep the candidates at about 1.4 k, and a row's
// segments publish at most 64 lists of 16 per 4 * nl loads, which the bound's search reads in one round.
struct MidKChoice {
    int nl = 0, nseg = 0;
    bool capped = false, may_pen = false, all = false;
};
bool mid_k_choice(int cus, const fs_row_params* h, int64_t n, int64_t rows, int32_t V, bool outputs, bool edited,
                  MidKChoice& c) {
    int64_t kmax = 1;
    for (int64_t b = 0; b < n; ++b) {
        const fs_row_params& p = h[b];
        const bool greedy = !(p.temperature > 0.0f && p.top_k != 1);
        const int64_t k = greedy ? 1 : ((p.top_k > 0 && p.top_k < V) ? p.top_k : V);
        if (k == V && k > fs::KMAX) {
            // every token a candidate: no candidate outputs and no min-p (its count and sum over the kept logits)
            // (taken whatever the rows hold, which the host cannot see. Rows whose mass is a few logits take about as long as
            // on the fused kernel with its short list: heavy-tailed logits at temperature 0.3, 1 row of 65536 19.1 us here
            // and 18.4 there, 16 rows 19.2 and 19.1, 64 of 262144 33.5 and 36.4. Rows with a body gain: 16 rows of 65536
            // N(0, 2) logits 24.0 and 28.3 at temperature 0.2, 27.5 and 62.4 at 1)
            if (outputs || p.min_p > 0.0f) return false;
            c.all = true;
        } else {
            kmax = std::max(kmax, k);
        }
        c.capped |= p.softcap > 0.0f;
        c.may_pen |= (p.repetition_penalty != 1.0f || p.frequency_penalty != 0.0f || p.presence_penalty != 0.0f) &&
                     p.repeat_last_n != 0;
    }
    if (kmax > fs::KMAX) return false;
    // the smallest segments whose workgroups are all resident at once (four per CU), else the largest: a second round of
    // a few workgroups delays its rows by a whole one (40 rows of 262144 logits, 1280 workgroups of 8192 logits: 30.8 us
    // against 24 with 640 of 16384)
    c.nl = 0;
    for (const int nl : {4, 8, 16}) {
        const int64_t seg = (int64_t)fs::SK_LT * nl * 4, n = ((int64_t)V + seg - 1) / seg;
        if (n * nl > 256 || n > fs::MK_MAX_SEGS) continue;
        // under edits the other way to sample the batch writes the rows out first, so smaller segments that hold enough lanes
        // for the largest k are taken in more rounds instead (mixed rows, k <= 2048: 143 of 103794 logits 108 -> 49.4 us, 102
        // of 138266 107 -> 43.0, 52 of 166347 92 -> 31.4)
        if (edited && c.nl != 0 && (int64_t)V < 8 * nl * kmax) break;
        c.nl = nl;
        c.nseg = (int)n;
        if (rows * n <= 4 * (int64_t)cus) break;
    }
    if (c.nl == 0 || (int64_t)V < 8 * c.nl * kmax) return false;
    return (int64_t)fs::XCDS * c.nseg * ((rows + fs::XCDS - 1) / fs::XCDS) <= 0x7fffffff;
}

// One buffer of the mid-k kernel's workspace: at least n elements of `per` words each, half as many again when it grows.
// FS_E_NOMEM leaves the old one as it was.
template <class T>
int grow_buffer(fs_context* c, T*& p, size_t& cap, size_t n, size_t per, bool zero) {
    if (n <= cap) return FS_OK;
    if (c->frozen) return FS_E_NOMEM;
    T* q = nullptr;
    size_t m = std::max(n, cap + cap / 2);
    if (hipMalloc(&q, m * per * sizeof(T)) != hipSuccess) {
        m = n;
        if (hipMalloc(&q, m * per * sizeof(T)) != hipSuccess) return no_memory();
    }
    if (zero && hipMemset(q, 0, m * per * sizeof(T)) != hipSuccess) {
        (void)hipFree(q);
        return FS_E_HIP;
    }
    release(c, p);
    p = q;
    cap = m;
    return FS_OK;
}

// Whether a call needs more than the context holds.
bool mid_grows(const fs_context* c, const MidKChoice& ch, size_t rows) {
    return rows * ch.nseg > c->mk_segs || rows > c->mk_ctr_rows || rows > c->mk_list_rows ||
           (ch.may_pen && rows > c->mk_spill_rows) || (ch.all && rows > c->mk_mass_rows);
}

// About 33 KB per row, 128 KB more with penalties and 16 KB with every token a candidate. After a failed allocation the
// next 64 calls that would have to grow don't try.
int grow_mid(fs_context* c, const MidKChoice& ch, size_t rows) {
    if (!mid_grows(c, ch, rows)) return FS_OK;
    if (c->mk_wait > 0) {
        --c->mk_wait;
        return FS_E_NOMEM;
    }
    int rc = grow_buffer(c, c->mk_qk, c->mk_segs, rows * ch.nseg, fs::SK_NW * 16, false);
    if (rc == FS_OK) rc = grow_buffer(c, c->mk_ctr, c->mk_ctr_rows, rows, fs::MK_CTR, true);
    if (rc == FS_OK) rc = grow_buffer(c, c->mk_list, c->mk_list_rows, rows, fs::MK_LIST, false);
    if (rc == FS_OK && ch.may_pen) rc = grow_buffer(c, c->mk_spill, c->mk_spill_rows, rows, fs::MK_SPILL, false);
    if (rc == FS_OK && ch.all) rc = grow_buffer(c, c->mk_mass, c->mk_mass_rows, rows, 2048, true);
    if (rc == FS_E_NOMEM) c->mk_wait = 64;
    return rc;
}

// The fused kernel's layout for a call (a.nseg, a.seg_tiles, a.balance, its grid) and the workspace it needs.
int grow_fused(fs_context* ctx, fs::Args& a, int64_t rows, int64_t streams, int per_cu, int64_t* grid) {
    int64_t items = 0;
    const int rc = plan(ctx->cus, a, rows, items, *grid, 0, per_cu);
    if (rc != FS_OK) return rc;
    // verify: a 64-bit word per stream, then the 32-bit counters of streams longer than 32 rows
    return grow(ctx, (size_t)(items > 0 ? items : 1), (size_t)rows, (size_t)(streams > 0 ? 3 * streams : 1));
}

// Whether the batch fits the mid-k kernel (fits), and the workspace it needs there. Under capture a workspace that would
// have to grow leaves the batch to the fused kernel (no allocation in a capture that worked without one), and so does one
// that the device has no room for: fits is false.
// per_cu: as launch's; the fused kernel's workspace grows as launch would grow it, so that a context warmed up with any
// parameters of a shape allocates nothing when a call of that shape with others is recorded. The caller holds ctx->mu and
// has the context's device.
int reserve_mid(fs_context* ctx, const fs::Args& a, const fs_row_params* h_params, hipStream_t st, int per_cu,
                const fs::EdArgs* ed, MidKChoice& ch, bool& fits) {
    fits = false;
    if (!ctx->seg_layout) return FS_OK;
    const bool verify = a.mode == fs::MODE_VERIFY;
    if (!mid_k_choice(ctx->cus, h_params, verify ? (int64_t)a.n_streams : (int64_t)a.B, a.B, a.V,
                      a.cand_ids || a.cand_probs, ed != nullptr, ch))
        return FS_OK;
    if (ed && ed->bias_off && ch.capped) return FS_OK;     // (the softcap, late in this kernel, comes before the biases)
    const size_t streams = verify ? 3 * (size_t)a.n_streams : 0;
    const bool cap = capturing(st);
    if (cap && (mid_grows(ctx, ch, (size_t)a.B) || streams > ctx->stream_cap || !ctx->err)) return FS_OK;
    int rc = FS_OK;
    if (!cap) {
        fs::Args fused = a;
        int64_t fused_grid = 0;
        rc = grow_fused(ctx, fused, a.B, verify ? a.n_streams : 0, per_cu, &fused_grid);
    }
    if (rc == FS_E_NOMEM || rc == FS_E_INVALID) {   // (this kernel does not need it)
        (void)hipGetLastError();
        rc = grow(ctx, 0, 0, streams);
    }
    if (rc != FS_OK) return rc;
    rc = grow_mid(ctx, ch, (size_t)a.B);
    fits = rc == FS_OK;
    return rc == FS_E_NOMEM ? FS_OK : rc;
}

// Launches the mid-k kernel when the batch fits it; *used = false (nothing launched) otherwise.
int launch_mid(fs_context* ctx, const fs::Args& a, const fs_row_params* h_params, hipStream_t st, bool& used, int per_cu = 2,
               const fs::EdArgs* ed = nullptr) {
    used = false;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    int rc = device_of(ctx);
    if (rc != FS_OK) return rc;
    const bool verify = a.mode == fs::MODE_VERIFY;
    MidKChoice ch;
    bool fits = false;
    rc = reserve_mid(ctx, a, h_params, st, per_cu, ed, ch, fits);
    if (rc != FS_OK || !fits) return rc;
    if (capturing(st)) ctx->captured = true;
    fs::MkArgs m = {};
    m.a = row_args(ctx, a, ch.nseg);
    m.ctr = ctx->mk_ctr; m.qk = ctx->mk_qk; m.list = ctx->mk_list; m.spill = ctx->mk_spill;
    m.mass = ctx->mk_mass; m.spins = ctx->merge_spins;
    if (ed) m.a.ed = *ed;
    const int64_t grid = (int64_t)fs::XCDS * ch.nseg * (((int64_t)a.B + fs::XCDS - 1) / fs::XCDS);
#ifdef FS_TRACE
    if (ctx->trace && grid * fs::TRACE_W <= ctx->trace_cap) m.a.trace = ctx->trace;
#endif
    const int flags = (ch.may_pen ? fs::SK_MAY_PEN : 0) | (a.out_hist_off ? fs::SK_COPY : 0) |
                      (verify ? fs::MK_VERIFY : 0) | edit_flags(ed);
    if (fs::launch_mid_k(ch.nl, ch.capped, ch.all, ed != nullptr, (unsigned)grid, flags, m, st) != hipSuccess) return FS_E_HIP;
    used = true;
    return FS_OK;
}

int launch(fs_context* ctx, fs::Args a, int64_t rows, int64_t streams, hipStream_t st, int per_cu = 2) {
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    int rc = device_of(ctx);
    if (rc != FS_OK) return rc;
    int64_t seg_grid = 0;
    rc = grow_fused(ctx, a, rows, streams, per_cu, &seg_grid);
    if (rc != FS_OK) return rc;
    if (capturing(st)) ctx->captured = true;
    a.cand = ctx->cand; a.meta = ctx->meta; a.rhist = ctx->rhist; a.rmass = ctx->rmass;
    a.stream_cnt = ctx->stream_cnt; a.err = ctx->err; a.dirty = ctx->err + 1; a.merge_spins = ctx->merge_spins;
    a.trace = nullptr;
    int done = FS_OK;
    if (gave_up(ctx->hflag)) {
        clear_words(st, ctx->rhist, (int64_t)(ctx->row_cap * fs::RBINS));
        clear_words(st, ctx->rmass, (int64_t)(ctx->row_cap * fs::LB * 2));
        clear_words(st, ctx->stream_cnt, (int64_t)ctx->stream_cap);
        clear_words(st, ctx->err + 1, 1);
        if (hipGetLastError() != hipSuccess) return FS_E_HIP;
        done = FS_W_RECOVERED;
    }
    if (!ctx->seg_layout) {
        rc = launch_alone(a, rows, st);
        return rc != FS_OK ? rc : done;
    }
#ifdef FS_TRACE
    {
        const int64_t grid = seg_grid > 0 ? seg_grid + (int64_t)fs::XCDS * ((rows + fs::XCDS - 1) / fs::XCDS) : rows;
        if (ctx->trace && grid * fs::TRACE_W <= ctx->trace_cap) a.trace = ctx->trace;   // else: untraced
    }
#endif
    rc = launch_planned(a, rows, seg_grid, st);
    return rc != FS_OK ? rc : done;
}

// ---- calls under edits (fs_sample_edited, fs_verify_edited, fs_decode_step_edited)
// For such a call's time: the context's lock is held (a composed call's launches follow one another and bind one set of
// workspace pointers, whatever other host threads enqueue on the context), the context is on the current device, and no
// workspace grows where the call is being recorded (an allocation would end the capture).
struct Edited {
    std::lock_guard<std::recursive_mutex> lock;
    fs_context* c;
    int rc = FS_OK;
    Edited(fs_context* ctx, hipStream_t st) : lock(ctx->mu), c(ctx) {
        rc = device_of(c);
        int dev = -1;
        if (rc == FS_OK && hipGetDevice(&dev) != hipSuccess) rc = FS_E_HIP;
        if (rc == FS_OK && dev != c->device) rc = FS_E_INVALID;
        if (rc == FS_OK && capturing(st)) c->frozen = c->captured = true;
    }
    ~Edited() { c->frozen = false; }               // (before the lock goes)
};

// Groups of four logits per thread and segments per row of the edit kernel: the largest segments that still give every CU
// four workgroups. Measured with 2, 4 and 8 groups, bf16 with masks, 30 biases and a window: 1 row of 262144 4.4, 5.2, 6.7 us;
// 32 rows 14.3, 12.5, 12.2; 64 rows 23.4, 22.6, 18.5; 256 rows 83.9, 72.0, 75.4; 64 rows of 32000 6.6, 6.8, 8.6. fp16 rows of
// 100003 with a softcap, windows of 4096 ids and 300 biases, which every segment reads again: 1 row 10.0, 15.0, 24.3; 24 rows
// 16.9, 20.1, 28.9; 64 rows 30.6, 31.7, 39.9; 64 of 262144 61.9, 59.3, 63.3.
int edit_plan(int cus, int64_t B, int32_t V, int& nseg) {
    int nl = 2;
    for (const int l : {8, 4, 2}) {
        nl = l;
        nseg = (int)(((int64_t)V + fs::SK_LT * l * 4 - 1) / (fs::SK_LT * l * 4));
        if (B * nseg >= 4 * (int64_t)cus) break;
    }
    return nl;
}

// The rows edited into the workspace, sampled there without penalties by whichever kernel takes them, and the call's end:
// rows without a candidate, a window's accepted prefix. Right for every batch. Every buffer of the call, the sampling
// kernel's among them, is there before the first launch: a call that is refused leaves nothing on its stream (or in the
// graph that records it), and no draw is taken. Inside an Edited.
int launch_composed(fs_context* ctx, const fs::Args& a, const fs_row_params* h_params, const fs::EdArgs& ed, hipStream_t st) {
    const bool verify = a.mode == fs::MODE_VERIFY, decode = a.dmt != nullptr;
    const size_t B = (size_t)a.B, ld = ((size_t)a.V + 3) & ~(size_t)3;
    std::unique_ptr<fs_row_params[]> h;
    if (h_params && !verify) {                     // (a window's rows have their streams' parameters, known on the device)
        h.reset(new (std::nothrow) fs_row_params[B]);
        if (!h) return FS_E_NOMEM;
        for (size_t b = 0; b < B; ++b) {
            h[b] = h_params[b];
            h[b].repetition_penalty = 1.0f; h[b].frequency_penalty = 0.0f; h[b].presence_penalty = 0.0f;
            h[b].repeat_last_n = 0; h[b].penalty_from = 0; h[b].softcap = 0.0f;
        }
    }
    const int per_cu = h && mixed_merges(h.get(), a.B, a.V) ? 4 : 2;
    fs::Args s = {};
    s.ld = (int64_t)ld; s.B = a.B; s.V = a.V; s.u = a.u; s.tok = a.tok;
    s.kcap = a.kcap; s.cand_ids = a.cand_ids; s.cand_probs = a.cand_probs; s.keep = a.keep;
    s.mode = fs::MODE_SAMPLE; s.eos = -1;
    bool small = false, mid = false;               // the kernel that samples the rows (neither: the fused one)
    int nseg = 0;
    const int nl = edit_plan(ctx->cus, a.B, a.V, nseg);
    if ((int64_t)a.B * nseg > 0x7fffffff) return FS_E_INVALID;
    int rc = grow(ctx, 0, 0, 0);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->ed_rows, ctx->ed_logits, B * ld, 1, false);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->ed_params, ctx->ed_param_rows, B, 1, false);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->ed_any, ctx->ed_any_rows, B, 1, true);
    if (rc == FS_OK && decode) rc = grow_buffer(ctx, ctx->ed_u, ctx->ed_u_rows, B, 1, false);
    if (rc == FS_OK && decode && !a.hist_off) rc = grow_buffer(ctx, ctx->ed_off, ctx->ed_off_rows, B + 1, 1, true);
    if (rc == FS_OK && h) {
        SmallKChoice sc;
        MidKChoice mc;
        rc = reserve_small(ctx, s, h.get(), nullptr, sc, small);
        if (rc == FS_E_NOMEM && ctx->frozen) rc = FS_OK;       // (another kernel's workspace may be there)
        if (rc == FS_OK && !small) rc = reserve_mid(ctx, s, h.get(), st, per_cu, nullptr, mc, mid);
    }
    if (rc == FS_OK && (!(small || mid) || !ctx->frozen)) {    // (a shape warmed up so records with other parameters)
        fs::Args f = s;
        int64_t grid = 0;
        rc = grow_fused(ctx, f, a.B, 0, per_cu, &grid);
        if ((small || mid) && (rc == FS_E_NOMEM || rc == FS_E_INVALID)) rc = FS_OK;
    }
    if (rc != FS_OK) return rc;
    fs::EditArgs e = {};
    e.logits = a.logits; e.type = FS_F32; e.ld = a.ld; e.B = a.B; e.V = a.V; e.nseg = nseg;
    e.hist = a.hist; e.hist_off = a.hist_off; e.params = a.params; e.ed = ed;
    if (verify) { e.rows = a.rows; e.row_off = a.row_off; e.n_streams = a.n_streams; }
    e.out = ctx->ed_rows; e.out_ld = (int64_t)ld; e.err = ctx->err; e.any = ctx->ed_any; e.rparams = ctx->ed_params;
    if (fs::launch_edit(nl, e, st) != hipSuccess) return FS_E_HIP;
    auto failed = [&](int rc) {                    // (the rows' marks are left at 0)
        clear_words(st, ctx->ed_any, (int64_t)B);
        return rc;
    };

    s.logits = ctx->ed_rows; s.params = ctx->ed_params;
    if (decode) {
        hipLaunchKernelGGL(fs::drng_draw_kernel, dim3((unsigned)((B + 63) / 64)), dim3(64), 0, st, a.dmt, a.didx, a.B,
                           (const int64_t*)nullptr, a.params, ctx->ed_u, 0, ctx->err);
        if (hipGetLastError() != hipSuccess) return failed(FS_E_HIP);
        s.u = ctx->ed_u;
    }
    bool used = false;
    if (small) rc = launch_small(ctx, s, h.get(), st, used);
    else if (mid) rc = launch_mid(ctx, s, h.get(), st, used, per_cu);
    if (rc == FS_OK && !used) rc = launch(ctx, s, a.B, 0, st, per_cu);
    if (rc < 0) return failed(rc);

    fs::EditEnd f = {};
    f.B = a.B; f.any = ctx->ed_any; f.rparams = ctx->ed_params; f.tok = a.tok; f.keep = a.keep;
    f.kcap = a.kcap; f.cand_ids = a.cand_ids; f.cand_probs = a.cand_probs;
    if (verify) {
        f.rows = a.rows; f.row_off = a.row_off; f.n_streams = a.n_streams; f.eos = a.eos; f.accepted = a.accepted;
    }
    if (fs::launch_edit_end(f, st) != hipSuccess) return FS_E_HIP;
    if (decode) {
        const int32_t* hist = a.hist ? a.hist : a.tok;         // (empty histories: never read)
        const int64_t* off = a.hist_off ? a.hist_off : ctx->ed_off;
        if (fs::launch_hist_append(a.B, hist, off, a.tok, nullptr, nullptr, a.out_hist, a.out_hist_off, a.out_cap, ctx->err,
                                   st) != hipSuccess)
            return FS_E_HIP;
    }
    return rc;
}

// The kernels that read masks and biases themselves where one takes the batch, else the edited rows.
int launch_edited(fs_context* ctx, const fs::Args& a, const fs_row_params* h_params, const fs::EdArgs& ed, hipStream_t st) {
    const Edited call(ctx, st);
    if (call.rc != FS_OK) return call.rc;
    if (h_params) {
        bool used = false;
        int rc = launch_small(ctx, a, h_params, st, used, &ed);
        if (rc != FS_OK || used) return rc;
        rc = launch_mid(ctx, a, h_params, st, used, 2, &ed);
        if (rc != FS_OK || used) return rc;
    }
    return launch_composed(ctx, a, h_params, ed, st);
}

// The host's checks of a call's edits; `edits` NULL: none.
int edit_args(const fs_edits* edits, int32_t rows, int32_t V, fs::EdArgs& ed) {
    ed = {};
    if (!edits) return FS_OK;
    if (edits->d_mask) {
        if (edits->mask_ld < ((int64_t)V + 31) / 32 || edits->n_masks < 0) return FS_E_INVALID;
        if (!edits->d_mask_of && edits->n_masks < rows) return FS_E_INVALID;
        if (((uintptr_t)edits->d_mask & 3u) != 0) return FS_E_INVALID;
    } else if (edits->d_mask_of || edits->n_masks != 0) {
        return FS_E_INVALID;
    }
    if (edits->d_bias_off ? (!edits->d_bias_ids || !edits->d_bias) : (edits->d_bias_ids || edits->d_bias)) return FS_E_INVALID;
    ed.mask = edits->d_mask; ed.mask_ld = edits->mask_ld; ed.n_masks = edits->n_masks; ed.mask_of = edits->d_mask_of;
    ed.bias_ids = edits->d_bias_ids; ed.bias = edits->d_bias; ed.bias_off = edits->d_bias_off;
    return FS_OK;
}

// Parts per row of fs_logprobs and fs_beam_select, at most `parts`. Four workgroups fit a CU; p parts take ceil(B p / 4 CUs)
// rounds of ceil(n / p) chunks of a row's n and of about 4 chunks' time to begin and join, and the p with the shortest of these
// is taken. For few rows that fills the device once (64 rows of 262144, n 20: 16 parts 25.6 us, 8 30.7, 32 31.2; 256 rows: 4 parts 57.6, 2 78.7, 8 66.3);
// past half of the slots more parts fill a last round (600 rows of 151936: 3 parts 84.1 us, 1 94.0; 1100 rows of bf16, n 1:
// 2 parts 79.1, 1 86.1; 700 rows: 1 part 52.5, 2 56.3).
int logprob_parts(const fs_context* c, int64_t B, int32_t V, int32_t type, int parts) {
    if (!c->seg_layout) return 1;                  // (a row's parts would not share an L2)
    const int64_t chunk = (int64_t)fs::SK_LT * 4 * fs::LP_NL(type), n = ((int64_t)V + chunk - 1) / chunk;
    const int64_t slots = 4 * (int64_t)c->cus, most = std::min<int64_t>(n, parts);
    if (B * most <= slots) return (int)most;
    int64_t best = 1, least = INT64_MAX;
    for (int64_t p = 1; p <= most; ++p) {
        const int64_t cost = (B * p + slots - 1) / slots * ((n + p - 1) / p + 4);
        if (cost < least) { least = cost; best = p; }
    }
    return (int)best;
}

// ---- fs_reorder_states
// Bytes per column: what the pointers, the strides and a position's bytes are all multiples of, 16 at most (streams of more
// than 32 rows, whose columns are all in registers: 8; launch_reorder_states has the times of both).
int state_bytes(const fs_state& z, int rows) {
    const uint64_t all = (uint64_t)(uintptr_t)z.d_src | (uint64_t)(uintptr_t)z.d_dst | (uint64_t)z.src_row |
                         (uint64_t)z.src_block | (uint64_t)z.src_pos | (uint64_t)z.dst_row | (uint64_t)z.dst_block |
                         (uint64_t)z.dst_pos | (uint64_t)z.pos_bytes;
    int vb = rows > 32 ? 8 : 16;
    while (vb > 1 && (all & (uint64_t)(vb - 1)) != 0) vb >>= 1;
    return vb;
}
int64_t state_cols(const fs_state& z, int vb) {
    return (int64_t)z.blocks * std::max(1, z.positions) * (z.pos_bytes / vb);
}
int check_state(const fs_state& z, int64_t S, int32_t n_src, int32_t n) {
    const bool empty = z.blocks == 0 || z.pos_bytes == 0 || S == 0;
    if ((!empty && (!z.d_src || !z.d_dst)) || z.pos_bytes < 0 || z.blocks < 0 || z.positions < 0 || z.src_row < 0 || z.src_block < 0 ||
        z.src_pos < 0 || z.dst_row < 0 || z.dst_block < 0 || z.dst_pos < 0)
        return FS_E_INVALID;
    // columns are counted in 32 bits; nor do spans come near 64
    const int64_t most = int64_t(1) << 46;
    const int64_t pos = std::max(1, z.positions);
    if (z.pos_bytes > 0x7fffffff || (int64_t)z.blocks * pos > 0x7fffffff) return FS_E_INVALID;
    for (const int64_t stride : {z.src_row, z.src_block, z.src_pos, z.dst_row, z.dst_block, z.dst_pos})
        if (stride > most) return FS_E_INVALID;
    if ((double)z.blocks * (double)pos * (double)z.pos_bytes > 2e9 * state_bytes(z, n > n_src ? n : n_src)) return FS_E_INVALID;
    if (empty) return FS_OK;
    // places of d_dst that lie over the next ones: what is stored there last would count
    if ((S * n > 1 && z.dst_row < z.pos_bytes) || (z.blocks > 1 && z.dst_block < z.pos_bytes) ||
        (pos > 1 && z.dst_pos < z.pos_bytes))
        return FS_E_INVALID;
    if (z.d_src == z.d_dst && n == n_src && z.src_row == z.dst_row && z.src_block == z.dst_block && z.src_pos == z.dst_pos)
        return FS_OK;
    auto span = [&](int64_t rows, int64_t row, int64_t block, int64_t p) {
        return (double)(rows - 1) * (double)row + (double)(z.blocks - 1) * (double)block + (double)(pos - 1) * (double)p +
               (double)z.pos_bytes;
    };
    const double s0 = (double)(uintptr_t)z.d_src, s1 = s0 + span(S * n_src, z.src_row, z.src_block, z.src_pos);
    const double d0 = (double)(uintptr_t)z.d_dst, d1 = d0 + span(S * n, z.dst_row, z.dst_block, z.dst_pos);
    return s0 < d1 && d0 < s1 ? FS_E_INVALID : FS_OK;
}

// The parts, the rows and the workspace of a log-probability kernel's launch (top: the largest it lists; parts, list: the most
// parts of a row, entries of a wave's list).
int reserve_logprobs(fs_context* ctx, const void* d_logits, int32_t type, int64_t ld, int32_t B, int32_t V, int32_t top,
                     int parts, int list, fs::LpArgs& a) {
    a.nseg = logprob_parts(ctx, B, V, type, parts);
    if (((int64_t)B + fs::XCDS) * a.nseg > 0x7fffffff) return FS_E_INVALID;
    const size_t entries = (size_t)B * a.nseg * fs::SK_NW * list;
    int rc = grow(ctx, 0, 0, 0);
    if (rc == FS_OK)
        rc = grow_buffer(ctx, ctx->lp_row, ctx->lp_row_bytes, (size_t)B * fs::lp_row_bytes(a.nseg), 1, false);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->lp_ticket, ctx->lp_rows, (size_t)B, fs::LP_LINE, true);
    if (rc == FS_OK && top > 0) rc = grow_buffer(ctx, ctx->lp_lists, ctx->lp_list_cap, entries, 1, false);
    if (rc != FS_OK) return rc;
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.n = top;
    a.rows = ctx->lp_row; a.ticket = ctx->lp_ticket; a.lists = ctx->lp_lists; a.err = ctx->err;
    return FS_OK;
}

size_t type_size(int32_t type) { return type == FS_F32 ? 4 : type == FS_BF16 || type == FS_F16 ? 2 : 0; }

// Rows of logits of any type: check_rows for FS_F32, four logits' alignment for the others.
int check_typed(const void* d_logits, int32_t type, int64_t ld, int32_t B, int32_t V) {
    const size_t size = type_size(type);
    if (size == 0 || !d_logits || B < 0 || V < 1 || V > FS_MAX_VOCAB || ld < V || (ld & 3) != 0 ||
        ((uintptr_t)d_logits & (4 * size - 1)) != 0)
        return FS_E_INVALID;
    return FS_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------------ static workspace
// fs_sample_batch_static's workspace: one file-scope device array per GPU, held until the process ends, so the
// call allocates nothing. Layout (bytes): error word and dirty flag | meta [ST_SLOTS][2] | row histograms
// [ST_ROWS][RBINS] | large rows' mass histograms [ST_ROWS][LB] | candidate lists [ST_SLOTS][CAP]. The row and mass
// histograms (counters included) must be zero when a call starts; the kernels leave them so, and the first call on a
// device clears them with a fill kernel (no hipMemsetAsync: the call may be recorded into a graph).
constexpr int64_t ST_ROWS = 512;                                  // rows per call
constexpr int64_t ST_SLOTS = 512;                                 // (row, segment) slots per call
constexpr size_t ST_ERR_OFF = 0;                                  // int32 [2]: error bits, dirty
constexpr size_t ST_META_OFF = 256;
constexpr size_t ST_RHIST_OFF = ST_META_OFF + ((ST_SLOTS * 2 * sizeof(uint32_t) + 255) / 256) * 256;
constexpr size_t ST_RMASS_OFF = ST_RHIST_OFF + (size_t)ST_ROWS * fs::RBINS * sizeof(uint32_t);
constexpr size_t ST_CAND_OFF = ST_RMASS_OFF + (size_t)ST_ROWS * fs::LB * sizeof(uint64_t);
constexpr size_t ST_BYTES = ST_CAND_OFF + (size_t)ST_SLOTS * fs::CAP * sizeof(uint64_t);   // 50,336,000 B

static __device__ __align__(256) unsigned char scratch[ST_BYTES];


namespace {

constexpr int ST_MAX_DEVICES = 64;
std::mutex g_static_mu;
unsigned char* g_static_ptr[ST_MAX_DEVICES] = {};   // the device address of `scratch` on each device
int32_t* g_static_flag[ST_MAX_DEVICES] = {};        // host-mapped give-up flag of each device's static workspace

__global__ void store_u64_kernel(uint64_t* p, uint64_t v) { *p = v; }

// The static workspace of the current device: its address from hipGetSymbolAddress (the array's name is not a
// device address in host code), once per device; the first call also zeroes the error words and row histograms
// on `st`, ahead of its own launch.
int static_workspace(int dev, hipStream_t st, unsigned char** out) {
    if (dev < 0 || dev >= ST_MAX_DEVICES) return FS_E_INVALID;
    std::lock_guard<std::mutex> g(g_static_mu);
    if (!g_static_ptr[dev]) {
        void* ptr = nullptr;
        if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess || !ptr) return FS_E_HIP;
        unsigned char* base = (unsigned char*)ptr;
        int32_t* flag = nullptr;
        int32_t* flag_dev = nullptr;
        if (hipHostMalloc((void**)&flag, sizeof(int32_t), hipHostMallocMapped) != hipSuccess) return FS_E_NOMEM;
        *(volatile int32_t*)flag = 0;
        if (hipHostGetDevicePointer((void**)&flag_dev, flag, 0) != hipSuccess) return FS_E_HIP;
        hipLaunchKernelGGL(fs::zero_words_kernel, dim3(1), dim3(256), 0, st, (uint32_t*)(base + ST_ERR_OFF),
                           (int64_t)(ST_META_OFF / 4));
        // error word 2..3: the give-up flag's device address (a kernel store: the call may be under graph capture)
        hipLaunchKernelGGL(store_u64_kernel, dim3(1), dim3(1), 0, st, (uint64_t*)(base + ST_ERR_OFF + 8),
                           (uint64_t)(uintptr_t)flag_dev);
        g_static_flag[dev] = flag;
        hipLaunchKernelGGL(fs::zero_words_kernel, dim3(1024), dim3(256), 0, st, (uint32_t*)(base + ST_RHIST_OFF),
                           (int64_t)((ST_CAND_OFF - ST_RHIST_OFF) / 4));   // row and mass histograms
        if (hipGetLastError() != hipSuccess) return FS_E_HIP;
        g_static_ptr[dev] = base;
    }
    *out = g_static_ptr[dev];
    return FS_OK;
}

}  // namespace

namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

int check_rows(const float* d_logits, int64_t ld, int32_t B, int32_t V) {
    if (!d_logits || B < 0 || V < 1 || V > FS_MAX_VOCAB || ld < V || (ld & 3) != 0 || !aligned16(d_logits))
        return FS_E_INVALID;
    return FS_OK;
}

}  // namespace

extern "C" {

int fs_create(fs_context** out) {
    if (!out) return FS_E_INVALID;
    *out = new (std::nothrow) fs_context();
    return *out ? FS_OK : FS_E_NOMEM;
}

int fs_destroy(fs_context* c) {
    if (!c) return FS_E_INVALID;
    (void)hipFree(c->sk_lists);
    (void)hipFree(c->sk_ticket);
    (void)hipFree(c->mk_ctr);
    (void)hipFree(c->mk_list);
    (void)hipFree(c->mk_spill);
    (void)hipFree(c->mk_mass);
    (void)hipFree(c->mk_qk);
    (void)hipFree(c->cand);
    (void)hipFree(c->meta);
    (void)hipFree(c->rhist);
    (void)hipFree(c->rmass);
    (void)hipFree(c->stream_cnt);
    (void)hipFree(c->err);
    (void)hipFree(c->greedy);
    (void)hipFree(c->ed_rows);
    (void)hipFree(c->ed_params);
    (void)hipFree(c->ed_any);
    (void)hipFree(c->ed_u);
    (void)hipFree(c->ed_off);
    (void)hipFree(c->lp_row);
    (void)hipFree(c->lp_ticket);
    (void)hipFree(c->lp_lists);
    (void)hipFree(c->bm_rows);
    (void)hipFree(c->bm_lists);
    (void)hipFree(c->bm_ticket);
    for (void* p : c->retired) (void)hipFree(p);
    if (c->hflag) (void)hipHostFree(c->hflag);
    delete c;
    return FS_OK;
}

int fs_sample_batch(fs_context* ctx, const float* d_logits, int64_t ld, int32_t B, int32_t V, const int32_t* d_hist,
                    const int64_t* d_hist_off, const fs_row_params* d_params, const double* d_u, int32_t* d_tok,
                    int32_t kcap, int32_t* d_cand_ids, double* d_cand_probs, int32_t* d_keep, void* stream) {
    if (!ctx || !d_params || !d_tok || kcap < 0 || ((d_cand_ids || d_cand_probs) && kcap == 0)) return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = d_u; a.tok = d_tok; a.kcap = kcap; a.cand_ids = d_cand_ids; a.cand_probs = d_cand_probs; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    return launch(ctx, a, B, 0, (hipStream_t)stream);
}

int fs_sample_batch_hp(fs_context* ctx, const float* d_logits, int64_t ld, int32_t B, int32_t V,
                       const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params,
                       const fs_row_params* h_params, const double* d_u, int32_t* d_tok, int32_t kcap,
                       int32_t* d_cand_ids, double* d_cand_probs, int32_t* d_keep, void* stream) {
    if (!ctx || !d_params || !d_tok || kcap < 0 || ((d_cand_ids || d_cand_probs) && kcap == 0)) return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = d_u; a.tok = d_tok; a.kcap = kcap; a.cand_ids = d_cand_ids; a.cand_probs = d_cand_probs; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    if (h_params) {
        bool used = false;
        rc = launch_small(ctx, a, h_params, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
        const int per_cu = mixed_merges(h_params, B, V) ? 4 : 2;
        rc = launch_mid(ctx, a, h_params, (hipStream_t)stream, used, per_cu);
        if (rc != FS_OK || used) return rc;
        return launch(ctx, a, B, 0, (hipStream_t)stream, per_cu);
    }
    return launch(ctx, a, B, 0, (hipStream_t)stream);
}

int fs_verify_hp(fs_context* ctx, const float* d_logits, int64_t ld, int32_t n_streams, int32_t total_rows, int32_t V,
                 const int32_t* d_rows, const int64_t* d_row_off, const int32_t* d_hist, const int64_t* d_hist_off,
                 const fs_row_params* d_params, const fs_row_params* h_params, const double* d_u, int32_t eos_id,
                 int32_t* d_tok, int32_t* d_accepted, void* stream) {
    if (!ctx || !d_rows || !d_row_off || !d_params || !d_tok || !d_accepted || n_streams < 0 || total_rows < 0)
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, total_rows, V);
    if (rc != FS_OK) return rc;
    if (total_rows == 0 || n_streams == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = total_rows; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off;
    a.params = d_params; a.u = d_u; a.tok = d_tok; a.rows = d_rows; a.row_off = d_row_off; a.n_streams = n_streams;
    a.eos = eos_id; a.accepted = d_accepted; a.mode = fs::MODE_VERIFY;
    if (h_params) {
        bool used = false;
        rc = launch_small(ctx, a, h_params, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
        rc = launch_mid(ctx, a, h_params, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
    }
    return launch(ctx, a, total_rows, n_streams, (hipStream_t)stream);
}

int fs_small_k_plan(int32_t cus, int32_t B, int32_t V, int32_t* nl, int32_t* nseg) {
    if (cus < 1 || B < 1 || V < 1 || V > FS_MAX_VOCAB || !nl || !nseg) return FS_E_INVALID;
    int l = 0, n = 0;
    const int rc = small_k_plan(cus, B, V, l, n);
    *nl = l;
    *nseg = n;
    return rc == FS_OK ? FS_OK : FS_E_LIMIT;
}

int fs_route_plan(int32_t cus, const fs_row_params* h_params, int32_t n, int32_t total_rows, int32_t V,
                  int32_t verify, int32_t* kernel, int32_t* nl, int32_t* nseg, int32_t* per_cu) {
    if (cus < 1 || !h_params || n < 1 || total_rows < 1 || V < 1 || V > FS_MAX_VOCAB || !kernel || !nl || !nseg ||
        !per_cu)
        return FS_E_INVALID;
    if (!verify && total_rows != n) return FS_E_INVALID;
    SmallKChoice ch;
    *nl = 0;
    if (small_k_choice(cus, h_params, n, total_rows, V, verify != 0, ch)) {
        *kernel = ch.all_greedy ? 2 : 1;
        *nl = ch.nl;
        *nseg = ch.nseg;
        *per_cu = 0;
        return FS_OK;
    }
    fs::Args a = {};
    a.V = V;
    a.mode = verify ? fs::MODE_VERIFY : fs::MODE_SAMPLE;
    *per_cu = (!verify && mixed_merges(h_params, n, V)) ? 4 : 2;
    int64_t items = 0, seg_grid = 0;
    const int rc = plan(cus, a, total_rows, items, seg_grid, 0, *per_cu);
    if (rc != FS_OK) return rc;
    *kernel = 0;
    *nseg = a.nseg;
    return FS_OK;
}

int fs_mid_k_plan(int32_t cus, const fs_row_params* h_params, int32_t n, int32_t total_rows, int32_t V, int32_t* nl,
                  int32_t* nseg) {
    if (cus < 1 || !h_params || n < 1 || total_rows < 1 || V < 1 || V > FS_MAX_VOCAB || !nl || !nseg) return FS_E_INVALID;
    MidKChoice c;
    const bool fits = mid_k_choice(cus, h_params, n, total_rows, V, false, false, c);
    *nl = fits ? c.nl : 0;
    *nseg = fits ? c.nseg : 0;
    return fits ? FS_OK : FS_E_LIMIT;
}

int fs_sample_batch_static(fs_context* ctx, const float* d_logits, int64_t ld, int32_t B, int32_t V,
                           const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params,
                           const double* d_u, int32_t* d_tok, int32_t kcap, int32_t* d_cand_ids, double* d_cand_probs,
                           int32_t* d_keep, void* stream) {
    if (!ctx || !d_params || !d_tok || kcap < 0 || ((d_cand_ids || d_cand_probs) && kcap == 0)) return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    if (B > ST_ROWS) return FS_E_LIMIT;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = d_u; a.tok = d_tok; a.kcap = kcap; a.cand_ids = d_cand_ids; a.cand_probs = d_cand_probs; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    const hipStream_t st = (hipStream_t)stream;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    rc = device_of(ctx);
    if (rc != FS_OK) return rc;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return FS_E_HIP;
    if (ctx->static_dev >= 0 && ctx->static_dev != dev) return FS_E_INVALID;   // a context stays on one device
    int64_t items = 0, seg_grid = 0;
    rc = plan(ctx->cus, a, B, items, seg_grid, ST_SLOTS);        // fewer segments per row where the slots run out
    if (rc != FS_OK) return rc;
    if (items > ST_SLOTS) return FS_E_LIMIT;
    unsigned char* base = nullptr;
    rc = static_workspace(dev, st, &base);
    if (rc != FS_OK) return rc;
    ctx->static_dev = dev;
    a.err = (int32_t*)(base + ST_ERR_OFF); a.dirty = a.err + 1;
    a.meta = (uint32_t*)(base + ST_META_OFF);
    a.rhist = (uint32_t*)(base + ST_RHIST_OFF);
    a.rmass = (uint64_t*)(base + ST_RMASS_OFF);
    a.cand = (uint64_t*)(base + ST_CAND_OFF);
    a.stream_cnt = nullptr;                          // sampling mode has no verify streams
    a.merge_spins = ctx->merge_spins;
    int done = FS_OK;
    int32_t* sflag = nullptr;
    {
        std::lock_guard<std::mutex> gs(g_static_mu);
        sflag = g_static_flag[dev];
    }
    if (gave_up(sflag)) {                            // an earlier call on the device gave up: clear what it left
        clear_words(st, base + ST_RHIST_OFF, (int64_t)((ST_CAND_OFF - ST_RHIST_OFF) / 4));
        clear_words(st, a.dirty, 1);
        if (hipGetLastError() != hipSuccess) return FS_E_HIP;
        done = FS_W_RECOVERED;
    }
    rc = ctx->seg_layout ? launch_planned(a, B, seg_grid, st) : launch_alone(a, B, st);
    return rc != FS_OK ? rc : done;
}

int fs_argmax_batch(fs_context* ctx, const float* d_logits, int64_t ld, int32_t B, int32_t V, const int32_t* d_hist,
                    const int64_t* d_hist_off, const fs_row_params* d_params, int32_t* d_tok, void* stream) {
    if (!ctx || !d_tok) return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_params ? d_hist_off : nullptr;
    a.params = d_params; a.tok = d_tok; a.mode = fs::MODE_ARGMAX; a.eos = -1;
    if (!d_params) {
        // no penalties: every row greedy, so the small-k kernel's greedy path takes the batch (its parameters are
        // greedy records the context keeps on the device and the host)
        fs::Args g = a;
        g.mode = fs::MODE_SAMPLE;
        g.hist = nullptr;
        bool used = false;
        rc = launch_small(ctx, g, nullptr, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
    }
    return launch(ctx, a, B, 0, (hipStream_t)stream);
}

int fs_verify(fs_context* ctx, const float* d_logits, int64_t ld, int32_t n_streams, int32_t total_rows, int32_t V,
              const int32_t* d_rows, const int64_t* d_row_off, const int32_t* d_hist, const int64_t* d_hist_off,
              const fs_row_params* d_params, const double* d_u, int32_t eos_id, int32_t* d_tok, int32_t* d_accepted,
              void* stream) {
    if (!ctx || !d_rows || !d_row_off || !d_params || !d_tok || !d_accepted || n_streams < 0 || total_rows < 0)
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, total_rows, V);
    if (rc != FS_OK) return rc;
    if (total_rows == 0 || n_streams == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = total_rows; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off;
    a.params = d_params; a.u = d_u; a.tok = d_tok; a.rows = d_rows; a.row_off = d_row_off; a.n_streams = n_streams;
    a.eos = eos_id; a.accepted = d_accepted; a.mode = fs::MODE_VERIFY;
    return launch(ctx, a, total_rows, n_streams, (hipStream_t)stream);
}

int fs_sample_edited(fs_context* ctx, const float* d_logits, int64_t ld, int32_t B, int32_t V, const int32_t* d_hist,
                     const int64_t* d_hist_off, const fs_row_params* d_params, const fs_row_params* h_params,
                     const fs_edits* edits, const double* d_u, int32_t* d_tok, int32_t kcap, int32_t* d_cand_ids,
                     double* d_cand_probs, int32_t* d_keep, void* stream) {
    if (!ctx || !edits || !d_params || !d_tok || kcap < 0 || ((d_cand_ids || d_cand_probs) && kcap == 0))
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    fs::EdArgs ed;
    rc = edit_args(edits, B, V, ed);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = d_u; a.tok = d_tok; a.kcap = kcap; a.cand_ids = d_cand_ids; a.cand_probs = d_cand_probs; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    return launch_edited(ctx, a, h_params, ed, (hipStream_t)stream);
}

int fs_verify_edited(fs_context* ctx, const float* d_logits, int64_t ld, int32_t n_streams, int32_t total_rows, int32_t V,
                     const int32_t* d_rows, const int64_t* d_row_off, const int32_t* d_hist, const int64_t* d_hist_off,
                     const fs_row_params* d_params, const fs_row_params* h_params, const fs_edits* edits,
                     const double* d_u, int32_t eos_id, int32_t* d_tok, int32_t* d_accepted, void* stream) {
    if (!ctx || !edits || !d_rows || !d_row_off || !d_params || !d_tok || !d_accepted || n_streams < 0 || total_rows < 0)
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, total_rows, V);
    if (rc != FS_OK) return rc;
    fs::EdArgs ed;
    rc = edit_args(edits, total_rows, V, ed);
    if (rc != FS_OK) return rc;
    if (total_rows == 0 || n_streams == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = total_rows; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off;
    a.params = d_params; a.u = d_u; a.tok = d_tok; a.rows = d_rows; a.row_off = d_row_off; a.n_streams = n_streams;
    a.eos = eos_id; a.accepted = d_accepted; a.mode = fs::MODE_VERIFY;
    return launch_edited(ctx, a, h_params, ed, (hipStream_t)stream);
}

int fs_edit_batch(fs_context* ctx, const void* d_logits, int32_t type, int64_t ld, int32_t B, int32_t V,
                  const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params, const fs_edits* edits,
                  float* d_out, int64_t out_ld, void* stream) {
    if (!ctx || !d_out || out_ld < V || (out_ld & 3) != 0 || !aligned16(d_out)) return FS_E_INVALID;
    int rc = check_typed(d_logits, type, ld, B, V);
    if (rc != FS_OK) return rc;
    fs::EditArgs e = {};
    rc = edit_args(edits, B, V, e.ed);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    if (!(type == FS_F32 && d_out == d_logits && out_ld == ld)) {
        const uintptr_t i0 = (uintptr_t)d_logits, i1 = i0 + ((size_t)(B - 1) * (size_t)ld + (size_t)V) * type_size(type);
        const uintptr_t o0 = (uintptr_t)d_out, o1 = o0 + ((size_t)(B - 1) * (size_t)out_ld + (size_t)V) * sizeof(float);
        if (i0 < o1 && o0 < i1) return FS_E_INVALID;
    }
    const Edited call(ctx, (hipStream_t)stream);
    if (call.rc != FS_OK) return call.rc;
    rc = grow(ctx, 0, 0, 0);                                   // the error word
    if (rc != FS_OK) return rc;
    const int nl = edit_plan(ctx->cus, B, V, e.nseg);
    if ((int64_t)B * e.nseg > 0x7fffffff) return FS_E_INVALID;
    e.logits = d_logits; e.type = type; e.ld = ld; e.B = B; e.V = V;
    e.hist = d_hist; e.hist_off = d_hist_off; e.params = d_params;
    e.out = d_out; e.out_ld = out_ld; e.err = ctx->err;
    return fs::launch_edit(nl, e, (hipStream_t)stream) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_logprobs(fs_context* ctx, const void* d_logits, int32_t type, int64_t ld, int32_t B, int32_t V,
                const fs_row_params* d_params, const fs_edits* edits, const int32_t* d_tok, int32_t n, float* d_lp,
                int32_t* d_rank, int32_t* d_top_ids, float* d_top_lp, void* stream) {
    if (!ctx || n < 0 || n > FS_MAX_TOP || ((d_lp || d_rank) && !d_tok) || ((d_top_ids || d_top_lp) && n == 0))
        return FS_E_INVALID;
    int rc = check_typed(d_logits, type, ld, B, V);
    if (rc != FS_OK) return rc;
    fs::LpArgs a = {};
    rc = edit_args(edits, B, V, a.ed);
    if (rc != FS_OK) return rc;
    if (B == 0) return FS_OK;
    const hipStream_t st = (hipStream_t)stream;
    const int top = d_top_ids || d_top_lp ? n : 0;
    const Edited call(ctx, st);
    if (call.rc != FS_OK) return call.rc;
    rc = reserve_logprobs(ctx, d_logits, type, ld, B, V, top, fs::LP_PARTS, fs::LP_TOP, a);
    if (rc != FS_OK) return rc;
    a.params = d_params; a.tok = d_tok; a.lp = d_lp; a.rank = d_rank; a.ids = d_top_ids; a.top = d_top_lp;
    return fs::launch_logprobs(type, a, st) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_beam_select(fs_context* ctx, const void* d_logits, int32_t type, int64_t ld, int32_t n_streams, int32_t total_rows,
                   int32_t V, const int64_t* d_row_off, const float* d_score, const fs_row_params* d_params,
                   const fs_edits* edits, int32_t eos_id, int32_t n, int32_t flags, int32_t* d_parent, int32_t* d_tok,
                   float* d_out_score, int32_t* d_done, int32_t* d_done_parent, float* d_done_score, void* stream) {
    if (!ctx || n_streams < 0 || n < 1 || n > FS_MAX_TOP || (flags & ~FS_BEAM_KEEP_SLOTS) != 0 || !d_parent || !d_tok ||
        !d_out_score)
        return FS_E_INVALID;
    if (!d_row_off && n_streams > 0 && total_rows % n_streams != 0) return FS_E_INVALID;
    int rc = check_typed(d_logits, type, ld, total_rows, V);
    if (rc != FS_OK) return rc;
    fs::LpBeamArgs a = {};
    rc = edit_args(edits, total_rows, V, a.lp.ed);
    if (rc != FS_OK) return rc;
    if (n_streams == 0) return FS_OK;
    // a stream's outputs are written while parts of others' rows, and of its own dead ones, may still read theirs
    const size_t beams = (size_t)n_streams * n * 4;
    const std::pair<const void*, size_t> in[] = {{d_score, (size_t)total_rows * 4}, {d_row_off, ((size_t)n_streams + 1) * 8},
                                                 {d_params, (size_t)n_streams * sizeof(fs_row_params)}};
    const std::pair<const void*, size_t> out[] = {{d_parent, beams}, {d_tok, beams}, {d_out_score, beams},
                                                  {d_done, (size_t)n_streams * 4}, {d_done_parent, beams}, {d_done_score, beams}};
    for (const auto& i : in)
        for (const auto& o : out)
            if (i.first && o.first && (uintptr_t)i.first < (uintptr_t)o.first + o.second &&
                (uintptr_t)o.first < (uintptr_t)i.first + i.second)
                return FS_E_INVALID;
    const hipStream_t st = (hipStream_t)stream;
    const Edited call(ctx, st);
    if (call.rc != FS_OK) return call.rc;
    rc = reserve_logprobs(ctx, d_logits, type, ld, total_rows, V, n, fs::BM_PARTS, fs::BM_LIST, a.lp);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->bm_rows, ctx->bm_row_cap, (size_t)total_rows, 1, false);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->bm_lists, ctx->bm_list_cap, (size_t)total_rows, fs::BM_TOP, false);
    if (rc == FS_OK) rc = grow_buffer(ctx, ctx->bm_ticket, ctx->bm_streams, (size_t)n_streams, fs::LP_LINE, true);
    if (rc != FS_OK) return rc;
    a.lp.params = d_params;
    fs::BeamArgs& b = a.b;
    b.S = n_streams; b.W = total_rows / n_streams; b.n = n; b.eos = eos_id; b.keep_slots = flags & FS_BEAM_KEEP_SLOTS;
    b.row_off = d_row_off; b.score = d_score; b.parent = d_parent; b.tok = d_tok; b.out_score = d_out_score;
    b.done = d_done; b.done_parent = d_done_parent; b.done_score = d_done_score;
    b.rows = ctx->bm_rows; b.row_lists = ctx->bm_lists; b.ticket = ctx->bm_ticket;
    return fs::launch_beam_select(type, a, st) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_hist_fork(fs_context* ctx, int32_t n_streams, const int32_t* d_hist, const int64_t* d_hist_off,
                 const int64_t* d_row_off, int32_t n, const int32_t* d_parent, const int32_t* d_tok, int32_t* d_out_hist,
                 int64_t out_cap, int64_t* d_out_hist_off, void* stream) {
    if (!ctx || n_streams < 0 || n < 1 || out_cap < 0 || (int64_t)n_streams * n > 0x3fffffff || !d_out_hist_off ||
        (out_cap > 0 && !d_out_hist))
        return FS_E_INVALID;
    if (n_streams > 0 && (!d_hist_off || !d_parent)) return FS_E_INVALID;
    if (d_out_hist_off == d_hist_off || (d_out_hist && (d_out_hist == d_hist || d_out_hist == d_tok || d_out_hist == d_parent)))
        return FS_E_INVALID;                                   // out of place
    const hipStream_t st = (hipStream_t)stream;
    const Edited call(ctx, st);
    if (call.rc != FS_OK) return call.rc;
    const int rc = grow(ctx, 0, 0, 0);
    if (rc != FS_OK) return rc;
    fs::ForkArgs a = {};
    a.hist = d_hist; a.hist_off = d_hist_off; a.row_off = d_row_off; a.S = n_streams; a.n = n; a.parent = d_parent;
    a.tok = d_tok; a.out = d_out_hist; a.out_cap = out_cap; a.out_off = d_out_hist_off; a.err = ctx->err;
    return fs::launch_hist_fork(a, ctx->cus, st) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_reorder_states(fs_context* ctx, int32_t n_states, const fs_state* states, int32_t n_streams, int32_t n_src, int32_t n,
                      const int32_t* d_parent, const int32_t* d_from, const int32_t* d_len, void* stream) {
    if (!ctx || n_states < 0 || (n_states > 0 && !states) || n_streams < 0 || n_src < 1 || n_src > FS_MAX_TOP || n < 1 ||
        n > FS_MAX_TOP || (n_streams > 0 && !d_parent))
        return FS_E_INVALID;
    for (int32_t i = 0; i < n_states; ++i) {
        const int rc = check_state(states[i], n_streams, n_src, n);
        if (rc != FS_OK) return rc;
        for (int32_t j = 0; j < i; ++j)            // (interleaved states are fine; one given twice would move twice)
            if (states[i].d_dst && (states[i].d_dst == states[j].d_dst || states[i].d_dst == states[j].d_src ||
                                    states[i].d_src == states[j].d_dst))
                return FS_E_INVALID;
    }
    if (n_streams == 0 || n_states == 0) return FS_OK;
    const hipStream_t st = (hipStream_t)stream;
    const Edited call(ctx, st);
    if (call.rc != FS_OK) return call.rc;
    const int rc = grow(ctx, 0, 0, 0);
    if (rc != FS_OK) return rc;
    for (int32_t i = 0; i < n_states;) {           // runs of states whose columns are of one width
        fs::StateArgs a = {};
        a.S = n_streams; a.n_src = n_src; a.n = n; a.parent = d_parent; a.from = d_from; a.len = d_len; a.err = ctx->err;
        const int vb = state_bytes(states[i], n > n_src ? n : n_src);
        int64_t cols = 0;
        a.alike = 1;
        for (; i < n_states && a.n_states < fs::ST_MAX && state_bytes(states[i], n > n_src ? n : n_src) == vb; ++i) {
            const fs_state& z = states[i];
            a.alike &= z.blocks == a.z[0].blocks && z.positions == a.z[0].positions && z.pos_bytes == a.z[0].pos_bytes ||
                       a.n_states == 0;
            a.z[a.n_states++] = z;
            cols += state_cols(states[i], vb) * n_streams;
        }
        if (cols > 0 && fs::launch_reorder_states(vb, a, cols, ctx->cus, st) != hipSuccess) return FS_E_HIP;
    }
    return FS_OK;
}

int fs_penalize_batch(fs_context* ctx, float* d_logits, int64_t ld, int32_t B, int32_t V, const int32_t* d_hist,
                      const int64_t* d_hist_off, const fs_row_params* d_params, void* stream) {
    if (!ctx || !d_params) return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    if (B == 0 || !d_hist || !d_hist_off) return FS_OK;
    const int64_t nchunk = ((int64_t)V + fs::PEN_CHUNK - 1) / fs::PEN_CHUNK;
    if ((int64_t)B * nchunk > 0x7fffffff) return FS_E_INVALID;
    {
        std::lock_guard<std::recursive_mutex> g(ctx->mu);
        rc = grow(ctx, 0, 0, 0);
        if (rc != FS_OK) return rc;
    }
    hipLaunchKernelGGL(fs::penalize_kernel, dim3((unsigned)(B * nchunk)), dim3(fs::PEN_BLOCK), 0, (hipStream_t)stream,
                       d_logits, ld, V, d_hist, d_hist_off, d_params, (int)nchunk, ctx->err);
    return hipGetLastError() == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_softcap_batch(const float* d_in, float* d_out, int64_t n, float cap, void* stream) {
    if (n < 0 || (n > 0 && (!d_in || !d_out)) || !(cap > 0.0f)) return FS_E_INVALID;
    if (n == 0) return FS_OK;
    int64_t blocks = (n + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    hipLaunchKernelGGL(fs::softcap_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, d_in, d_out, n,
                       cap);
    return hipGetLastError() == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_lookup_draft(fs_context* ctx, int32_t n_streams, const int32_t* d_hist, const int64_t* d_hist_off,
                    const int32_t* d_kmax, const int32_t* d_min_n, int32_t eos_id, int32_t* d_draft, int32_t draft_ld,
                    int32_t* d_ndraft, void* stream) {
    if (!ctx || n_streams < 0 || !d_hist_off || !d_draft || !d_ndraft || draft_ld < 1) return FS_E_INVALID;
    if (n_streams == 0) return FS_OK;
    return fs::launch_lookup_draft(n_streams, d_hist, d_hist_off, d_kmax, d_min_n, eos_id, d_draft, draft_ld, d_ndraft,
                                   (hipStream_t)stream) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_hist_append(fs_context* ctx, int32_t n_streams, const int32_t* d_hist, const int64_t* d_hist_off,
                   const int32_t* d_tok, const int64_t* d_row_off, const int32_t* d_count, int32_t* d_out_hist,
                   int64_t out_cap, int64_t* d_out_hist_off, void* stream) {
    if (!ctx || n_streams < 0 || !d_hist_off || !d_out_hist_off || out_cap < 0) return FS_E_INVALID;
    if (n_streams > 0 && (!d_tok || !d_hist)) return FS_E_INVALID;
    if (out_cap > 0 && !d_out_hist) return FS_E_INVALID;
    if (d_out_hist_off == d_hist_off || (d_out_hist && d_out_hist == d_hist)) return FS_E_INVALID;   // out of place
    {
        std::lock_guard<std::recursive_mutex> g(ctx->mu);
        const int rc = grow(ctx, 1, 1, 1);               // the device error word
        if (rc != FS_OK) return rc;
    }
    return fs::launch_hist_append(n_streams, d_hist, d_hist_off, d_tok, d_row_off, d_count, d_out_hist, d_out_hist_off,
                                  out_cap, ctx->err, (hipStream_t)stream) == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_device_error(fs_context* ctx, void* stream, int32_t* bits) {
    if (!ctx || !bits) return FS_E_INVALID;
    *bits = 0;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    if (!ctx->err && ctx->static_dev < 0) return FS_OK;
    if (hipStreamSynchronize((hipStream_t)stream) != hipSuccess) return FS_E_HIP;
    if (ctx->err) {
        int32_t h[2] = {0, 0};
        if (hipMemcpy(h, ctx->err, sizeof(h), hipMemcpyDeviceToHost) != hipSuccess) return FS_E_HIP;
        *bits |= h[0];
        if (h[1] != 0) {
            // a merge gave up: the segments it did not wait for have finished by now (the stream is idle), so the
            // row histograms and counters are cleared and the context leaves its compute-alone mode
            if (ctx->rhist && hipMemset(ctx->rhist, 0, ctx->row_cap * fs::RBINS * sizeof(uint32_t)) != hipSuccess)
                return FS_E_HIP;
            if (ctx->rmass && hipMemset(ctx->rmass, 0, ctx->row_cap * fs::LB * sizeof(uint64_t)) != hipSuccess)
                return FS_E_HIP;
            if (ctx->stream_cnt && hipMemset(ctx->stream_cnt, 0, ctx->stream_cap * sizeof(uint32_t)) != hipSuccess)
                return FS_E_HIP;
        }
        if (hipMemset(ctx->err, 0, sizeof(h)) != hipSuccess) return FS_E_HIP;
    }
    if (ctx->static_dev >= 0) {
        // the device's static workspace (fs_sample_batch_static), shared by every context on the device
        unsigned char* base = nullptr;
        {
            std::lock_guard<std::mutex> gs(g_static_mu);
            base = g_static_ptr[ctx->static_dev];
        }
        if (base) {
            int32_t h[2] = {0, 0};
            if (hipMemcpy(h, base + ST_ERR_OFF, sizeof(h), hipMemcpyDeviceToHost) != hipSuccess) return FS_E_HIP;
            *bits |= h[0];
            if (h[1] != 0 && hipMemset(base + ST_RHIST_OFF, 0, ST_CAND_OFF - ST_RHIST_OFF) != hipSuccess)
                return FS_E_HIP;
            if (hipMemset(base + ST_ERR_OFF, 0, sizeof(h)) != hipSuccess) return FS_E_HIP;
        }
    }
    return FS_OK;
}

int fs_plan_layout(int32_t cus, int32_t xccs, int32_t B, int32_t V, int32_t static_ws, int32_t* nseg,
                   int32_t* seg_tiles, int64_t* slots) {
    if (cus < 1 || xccs < 0 || B < 1 || V < 1 || V > FS_MAX_VOCAB || !nseg || !seg_tiles || !slots) return FS_E_INVALID;
    if (static_ws && B > ST_ROWS) return FS_E_LIMIT;
    *nseg = 0; *seg_tiles = 0; *slots = 0;
    if (!layout_fits(xccs)) return FS_OK;                 // every row sampled alone by one workgroup
    fs::Args a = {};
    a.B = B; a.V = V; a.mode = fs::MODE_SAMPLE;
    int64_t items = 0, seg_grid = 0;
    const int rc = plan(cus, a, B, items, seg_grid, static_ws ? ST_SLOTS : 0);
    if (rc != FS_OK) return rc;
    if (static_ws && items > ST_SLOTS) return FS_E_LIMIT;
    *nseg = a.nseg; *seg_tiles = a.seg_tiles; *slots = items;
    return FS_OK;
}

int fs_error_word(fs_context* ctx, const int32_t** d_bits) {
    if (!ctx || !d_bits) return FS_E_INVALID;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    const int rc = grow(ctx, 0, 0, 0);
    if (rc != FS_OK) return rc;
    *d_bits = ctx->err;
    return FS_OK;
}

int fs_set_wait_limit(fs_context* ctx, uint32_t polls) {
    if (!ctx) return FS_E_INVALID;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    ctx->merge_spins = polls == FS_WAIT_GIVE_UP ? 0u : (polls ? polls : fs::MERGE_SPINS);
    return FS_OK;
}

// Per-stream draw source of ferro::Sampler (sampler.h:25,32 and the draw at sampler.cpp:45-46): the same libstdc++
// engine and canonical mapping, so u * tot equals uniform_real_distribution<double>(0, tot)(rng) bit for bit.
struct fs_rng {
    std::mt19937_64 eng;
};

int fs_rng_create(uint64_t seed, fs_rng** out) {
    if (!out) return FS_E_INVALID;
    *out = new (std::nothrow) fs_rng();
    if (!*out) return FS_E_NOMEM;
    (*out)->eng.seed(seed ? seed : (uint64_t)std::random_device{}());
    return FS_OK;
}

int fs_rng_destroy(fs_rng* r) {
    if (!r) return FS_E_INVALID;
    delete r;
    return FS_OK;
}

int fs_rng_next_u(fs_rng* r, double* u, int32_t n) {
    if (!r || !u || n < 0) return FS_E_INVALID;
    for (int32_t i = 0; i < n; ++i) u[i] = std::generate_canonical<double, 53>(r->eng);
    return FS_OK;
}

int fs_rng_copy(const fs_rng* src, fs_rng* dst) {
    if (!src || !dst) return FS_E_INVALID;
    dst->eng = src->eng;
    return FS_OK;
}

// Device draw streams (see fs::drng_draw_kernel): the engines' states live in device memory; seeding follows the
// standard's seed sequence for mt19937_64 (x0 = seed, x_i = 6364136223846793005 * (x_{i-1} ^ (x_{i-1} >> 62)) + i),
// so stream s reproduces std::mt19937_64(seed_s) and ferro::Sampler's draws.
struct fs_drng {
    int device = -1;
    int n = 0;
    uint64_t* mt = nullptr;     // [n][312]
    int32_t* idx = nullptr;     // [n]
    int32_t* err = nullptr;
};

// fs_decode_step: fs_sample_batch with the draws taken from the device streams r (row s = stream s) and each row's
// token appended to its stream's history out of place, in the sampling grid itself (one launch).
int fs_decode_step_hp(fs_context* ctx, fs_drng* r, const float* d_logits, int64_t ld, int32_t B, int32_t V,
                      const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params,
                      const fs_row_params* h_params, int32_t* d_tok, int32_t* d_keep, int32_t* d_out_hist,
                      int64_t* d_out_hist_off, int64_t out_cap, void* stream) {
    if (!ctx || !r || !d_params || !d_tok || !d_out_hist_off || out_cap < 0 || (out_cap > 0 && !d_out_hist) ||
        (d_hist == nullptr) != (d_hist_off == nullptr) || B > r->n)
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return FS_E_HIP;
    if (dev != r->device) return FS_E_INVALID;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = nullptr; a.tok = d_tok; a.kcap = 0; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    a.dmt = r->mt; a.didx = r->idx; a.out_hist = d_out_hist; a.out_hist_off = d_out_hist_off; a.out_cap = out_cap;
    if (h_params) {
        bool used = false;
        rc = launch_small(ctx, a, h_params, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
        rc = launch_mid(ctx, a, h_params, (hipStream_t)stream, used);
        if (rc != FS_OK || used) return rc;
    }
    return launch(ctx, a, B, 0, (hipStream_t)stream);
}

int fs_decode_step_edited(fs_context* ctx, fs_drng* r, const float* d_logits, int64_t ld, int32_t B, int32_t V,
                          const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params,
                          const fs_row_params* h_params, const fs_edits* edits, int32_t* d_tok, int32_t* d_keep,
                          int32_t* d_out_hist, int64_t* d_out_hist_off, int64_t out_cap, void* stream) {
    if (!ctx || !r || !edits || !d_params || !d_tok || !d_out_hist_off || out_cap < 0 || (out_cap > 0 && !d_out_hist) ||
        (d_hist == nullptr) != (d_hist_off == nullptr) || B > r->n)
        return FS_E_INVALID;
    int rc = check_rows(d_logits, ld, B, V);
    if (rc != FS_OK) return rc;
    fs::EdArgs ed;
    rc = edit_args(edits, B, V, ed);
    if (rc != FS_OK) return rc;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess) return FS_E_HIP;
    if (dev != r->device) return FS_E_INVALID;
    if (B == 0) return FS_OK;
    fs::Args a = {};
    a.logits = d_logits; a.ld = ld; a.B = B; a.V = V; a.hist = d_hist; a.hist_off = d_hist_off; a.params = d_params;
    a.u = nullptr; a.tok = d_tok; a.kcap = 0; a.keep = d_keep;
    a.mode = fs::MODE_SAMPLE; a.eos = -1;
    a.dmt = r->mt; a.didx = r->idx; a.out_hist = d_out_hist; a.out_hist_off = d_out_hist_off; a.out_cap = out_cap;
    return launch_edited(ctx, a, h_params, ed, (hipStream_t)stream);
}

int fs_decode_step(fs_context* ctx, fs_drng* r, const float* d_logits, int64_t ld, int32_t B, int32_t V,
                   const int32_t* d_hist, const int64_t* d_hist_off, const fs_row_params* d_params, int32_t* d_tok,
                   int32_t* d_keep, int32_t* d_out_hist, int64_t* d_out_hist_off, int64_t out_cap, void* stream) {
    return fs_decode_step_hp(ctx, r, d_logits, ld, B, V, d_hist, d_hist_off, d_params, nullptr, d_tok, d_keep,
                             d_out_hist, d_out_hist_off, out_cap, stream);
}

int fs_drng_create(int32_t n_streams, const uint64_t* seeds, void* stream, fs_drng** out) {
    if (!out || n_streams < 1 || !seeds) return FS_E_INVALID;
    *out = nullptr;
    fs_drng* r = new (std::nothrow) fs_drng();
    if (!r) return FS_E_NOMEM;
    std::vector<uint64_t> mt((size_t)n_streams * fs::MT_N);
    std::vector<int32_t> idx((size_t)n_streams, fs::MT_N);
    std::random_device rd;
    for (int32_t s = 0; s < n_streams; ++s) {
        uint64_t* x = mt.data() + (size_t)s * fs::MT_N;
        x[0] = seeds[s] ? seeds[s] : (uint64_t)rd();                     // seed 0 = random, as ferro
        for (int i = 1; i < fs::MT_N; ++i) x[i] = 6364136223846793005ull * (x[i - 1] ^ (x[i - 1] >> 62)) + (uint64_t)i;
    }
    r->n = n_streams;
    int rc = FS_OK;
    if (hipGetDevice(&r->device) != hipSuccess) rc = FS_E_HIP;
    if (rc == FS_OK && (hipMalloc(&r->mt, mt.size() * sizeof(uint64_t)) != hipSuccess ||
                        hipMalloc(&r->idx, idx.size() * sizeof(int32_t)) != hipSuccess ||
                        hipMalloc(&r->err, sizeof(int32_t)) != hipSuccess))
        rc = FS_E_NOMEM;
    hipStream_t st = (hipStream_t)stream;
    if (rc == FS_OK && (hipMemcpyAsync(r->mt, mt.data(), mt.size() * sizeof(uint64_t), hipMemcpyHostToDevice, st) != hipSuccess ||
                        hipMemcpyAsync(r->idx, idx.data(), idx.size() * sizeof(int32_t), hipMemcpyHostToDevice, st) != hipSuccess ||
                        hipMemsetAsync(r->err, 0, sizeof(int32_t), st) != hipSuccess ||
                        hipStreamSynchronize(st) != hipSuccess))
        rc = FS_E_HIP;
    if (rc != FS_OK) { fs_drng_destroy(r); return rc; }
    *out = r;
    return FS_OK;
}

int fs_drng_destroy(fs_drng* r) {
    if (!r) return FS_E_INVALID;
    (void)hipFree(r->mt);
    (void)hipFree(r->idx);
    (void)hipFree(r->err);
    delete r;
    return FS_OK;
}

int fs_drng_draw(fs_drng* r, const int64_t* d_row_off, const fs_row_params* d_params, double* d_u, int32_t peek,
                 void* stream) {
    if (!r || !d_params || !d_u) return FS_E_INVALID;
    hipLaunchKernelGGL(fs::drng_draw_kernel, dim3((unsigned)((r->n + 63) / 64)), dim3(64), 0, (hipStream_t)stream,
                       r->mt, r->idx, r->n, d_row_off, d_params, d_u, peek ? 1 : 0, r->err);
    return hipGetLastError() == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_drng_skip(fs_drng* r, const int32_t* d_counts, const fs_row_params* d_params, void* stream) {
    if (!r || !d_counts || !d_params) return FS_E_INVALID;
    hipLaunchKernelGGL(fs::drng_skip_kernel, dim3((unsigned)((r->n + 63) / 64)), dim3(64), 0, (hipStream_t)stream,
                       r->mt, r->idx, r->n, d_counts, d_params);
    return hipGetLastError() == hipSuccess ? FS_OK : FS_E_HIP;
}

int fs_drng_error(fs_drng* r, void* stream, int32_t* bits) {
    if (!r || !bits) return FS_E_INVALID;
    if (hipStreamSynchronize((hipStream_t)stream) != hipSuccess) return FS_E_HIP;
    if (hipMemcpy(bits, r->err, sizeof(int32_t), hipMemcpyDeviceToHost) != hipSuccess) return FS_E_HIP;
    if (hipMemset(r->err, 0, sizeof(int32_t)) != hipSuccess) return FS_E_HIP;
    return FS_OK;
}

#ifdef FS_TRACE
// Trace builds only (not in the product library): phase timestamps of the next sampling grids into d_buf (cap
// entries, TRACE_W per workgroup); a grid larger than the buffer runs untraced.
int fs_trace_set(fs_context* ctx, uint64_t* d_buf, int64_t cap) {
    if (!ctx || cap < 0) return FS_E_INVALID;
    std::lock_guard<std::recursive_mutex> g(ctx->mu);
    ctx->trace = d_buf;
    ctx->trace_cap = d_buf ? cap : 0;
    return FS_OK;
}
#endif

const char* fs_strerror(int code) {
    switch (code) {
        case FS_OK: return "ok";
        case FS_E_INVALID: return "invalid argument";
        case FS_E_HIP: return "HIP runtime error";
        case FS_E_NOMEM: return "device allocation failed";
        case FS_E_DEVICE: return "device-side error";
        case FS_E_LIMIT: return "batch exceeds the static workspace of fs_sample_batch_static";
        case FS_W_RECOVERED: return "ok; an earlier call's merge gave up waiting and this call cleared its workspace";
        default: return "unknown error";
    }
}

}  // extern "C"
