// What a step of drafted tokens needs beside its attention: rows of logits constrained (biases, penalties for repeated
// tokens, masks of allowed ones), the path through a tree of drafts that the chosen tokens confirm, and the accepted
// nodes' rows of the cache moved together.
#include "tcgen.cuh"

#define DR_NODES 64               // most drafted tokens of a request: a path is a 64-bit number

// Entries start[i] .. start[i + 1] - 1 of a list of n; none of what is outside it.
__device__ __forceinline__ void dr_span(const int* start, int i, int n, int& lo, int& hi) {
    lo = min(max(start[i], 0), n);
    hi = min(max(start[i + 1], lo), n);
}

// ---------------------------------------------------------------------- logits_constrain
// Row r of request q = owner[r], token i:
//   x = logits[r, i] + bias_q(i)
//   c = how often i stands in the last `window` tokens of (q's history, then the drafted tokens of r's own path)
//   c > 0:  x = x > 0 ? x / repetition : x * repetition;  x -= presence + frequency * c
//   not allowed: x = -inf
// the order and the arithmetic of adjust_kernel (sampling.cu), which edits one row from counts made on the host and which the tests
// hold this to: both give the same bits.
// (Counts are integers: the order of the additions changes nothing.)
#define LC_THREADS 256
#define LC_COLUMNS 8192
#define LC_AHEAD 8                // tokens of the history that a thread reads at once
#define LC_BIASED 0x80000000u
#define LC_NONE (int)0x80000000   // no token: far from every column
#define LI_THREADS 512
#define LI_COLUMNS 16384

struct Constrain {
    const float* logits; float* out;
    long long in_stride, out_stride;
    int rows, vocab, requests, n_bias, n_history, n_drafts;
    const int* owner;
    const int *bias_start, *bias_ids; const float* bias;
    const int *history_start, *history;
    const float* penalties;                  // [requests][repetition, presence, frequency]
    const int* windows;                      // null: every history whole
    const int *draft_start, *draft_tokens; const unsigned long long* seen;
    const uint32_t* allowed; long long allowed_stride; int allowed_rows_n;
    const int* allowed_rows;
    int row0;                                // of a launch whose blocks take a row each
};

__device__ __forceinline__ float lc_edit(float x, uint32_t count, float rep, float presence, float frequency) {
    const bool use_rep = rep != 0.f && rep != 1.f;
    const bool use_add = presence != 0.f || frequency != 0.f;
    if (count) {
        if (use_rep) x = x > 0.f ? x / rep : x * rep;
        if (use_add) x -= presence + frequency * (float)count;
    }
    return x;
}

// What is done to a row beside its mask.
struct ConstrainRow {
    int b_lo, b_hi, h_lo, h_hi, d_lo;         // its biases, the history's tokens and the drafted ones that are counted
    unsigned long long path;                  // (these by bits)
    float rep, presence, frequency;
    bool counts;
    __device__ __forceinline__ void find(const Constrain& a, int r, int q) {           // q: its request
        b_lo = b_hi = h_lo = h_hi = d_lo = 0;
        path = 0;
        counts = false;
        if (q < 0 || q >= a.requests) return;
        if (a.bias_start) dr_span(a.bias_start, q, a.n_bias, b_lo, b_hi);
        if (!a.penalties) return;
        int room = 0;
        rep = a.penalties[3 * q]; presence = a.penalties[3 * q + 1]; frequency = a.penalties[3 * q + 2];
        counts = (rep != 0.f && rep != 1.f) || presence != 0.f || frequency != 0.f;
        if (a.history_start) dr_span(a.history_start, q, a.n_history, h_lo, h_hi);
        if (a.windows) room = a.windows[q];
        if (room <= 0) room = 0x7fffffff;
        if (a.seen) {
            int d_hi;
            dr_span(a.draft_start, q, a.n_drafts, d_lo, d_hi);
            const int n = min(d_hi - d_lo, DR_NODES);
            path = a.seen[r] & (n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull);
            const int length = __popcll(path);
            while (__popcll(path) > room) path &= path - 1;         // the last ones
            room -= min(room, length);
        }
        if (h_hi - h_lo > room) h_lo = h_hi - room;
    }
    // Token `tid` of the path, or none.
    __device__ __forceinline__ int drafted(const Constrain& a, int tid) const {
        const int t = tid < DR_NODES && path >> tid & 1ull ? a.draft_tokens[d_lo + tid] : LC_NONE;
        return t < 0 ? LC_NONE : t;
    }
};

__device__ __forceinline__ const uint32_t* lc_mask(const Constrain& a, int r) {
    if (!a.allowed) return nullptr;
    const int w = a.allowed_rows ? a.allowed_rows[r] : r;
    return w >= 0 && w < a.allowed_rows_n ? a.allowed + (size_t)w * a.allowed_stride : nullptr;
}

// In place and without masks: only columns that change are touched. A block takes a slice of a row. It adds the biases, counts
// the tokens that fall into its slice in shared memory, and after a barrier a thread comes for each of the tokens it counted,
// takes the count out, and, if it was the first to come, edits the column.
//   MEASURED, in a graph of calls: 64 rows of 151936 with histories of 4001 tokens 13.5 us (18.7 by the copying kernel below, which
// takes the rows over in place where there are masks: 14.9 with masks alone), of 300 5.9; 128 rows, 600 tokens 10.7 (28.2);
// one row, 700 tokens 2.8. What changes, by 32 bytes, and the histories are 10 and 3 MB (1.4 and 0.5 us): bound by latency and by
// every slice's look at the row's whole history: slices of 8192 17.6 and 16.7 us for 13.5 and 10.7, of 32768 17.8 and 14.1.
__global__ void __launch_bounds__(LI_THREADS) constrain_in_place_kernel(const Constrain a) {
    extern __shared__ __align__(16) uint32_t li_count[];
    pdl_wait();
    const int tid = threadIdx.x, r = a.row0 + blockIdx.y, col0 = blockIdx.x * LI_COLUMNS;
    const uint32_t width = (uint32_t)min(LI_COLUMNS, a.vocab - col0);
    float* x = a.out + (long long)r * a.out_stride + col0;
    ConstrainRow row;
    row.find(a, r, a.owner ? a.owner[r] : r);
    for (int i = row.b_lo + tid; i < row.b_hi; i += LI_THREADS) {
        const int id = a.bias_ids[i];
        if (id >= 0 && (uint32_t)(id - col0) < width) x[id - col0] += a.bias[i];
    }
    if (!row.counts) return;
    int said[LC_AHEAD];                       // this thread's first tokens
    const int drafted = row.drafted(a, tid);
#pragma unroll
    for (int j = 0; j < LC_AHEAD; ++j) said[j] = row.h_lo + j * LI_THREADS + tid < row.h_hi ? a.history[row.h_lo + j * LI_THREADS + tid] : LC_NONE;
    for (int i = tid; i < LI_COLUMNS / 4; i += LI_THREADS) ((uint4*)li_count)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    auto all = [&](auto&& each) {             // the tokens of this thread that the slice has, each with its column
        auto one = [&](int token) {
            const uint32_t c = (uint32_t)(token - col0);
            if (token >= 0 && c < width) each(c);
        };
        one(drafted);
#pragma unroll
        for (int j = 0; j < LC_AHEAD; ++j) one(said[j]);
        for (int i = row.h_lo + LC_AHEAD * LI_THREADS + tid; i < row.h_hi; i += LI_THREADS) one(a.history[i]);
    };
    all([&](uint32_t c) { atomicAdd(&li_count[c], 1u); });
    __syncthreads();
    all([&](uint32_t c) {
        const uint32_t n = atomicExch(&li_count[c], 0u);
        if (n) x[c] = lc_edit(x[c], n, row.rep, row.presence, row.frequency);
    });
}

// Where the two matrices' rows lie differently to 16-byte boundaries: a block copies a slice of a row, a thread a column at a
// time, with its counts beside it. A biased token is left to a second look, when everything else of the slice is done.
__global__ void __launch_bounds__(LC_THREADS) constrain_kernel(const Constrain a) {
    __shared__ __align__(16) uint32_t count[LC_COLUMNS];
    pdl_wait();
    const int tid = threadIdx.x, r = a.row0 + blockIdx.y, col0 = blockIdx.x * LC_COLUMNS;
    const int n_cols = min(LC_COLUMNS, a.vocab - col0);
    const float* src = a.logits + (long long)r * a.in_stride + col0;
    float* dst = a.out + (long long)r * a.out_stride + col0;
    ConstrainRow row;
    row.find(a, r, a.owner ? a.owner[r] : r);
    const uint32_t* words = lc_mask(a, r);
    if (words) words += col0 >> 5;
    for (int i = tid; i < LC_COLUMNS / 4; i += LC_THREADS) ((uint4*)count)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    if (row.counts) {
        const int d = row.drafted(a, tid) - col0;
        if (d >= 0 && d < n_cols) atomicAdd(&count[d], 1u);
        for (int i = row.h_lo + tid; i < row.h_hi; i += LC_AHEAD * LC_THREADS) {
            int c[LC_AHEAD];
#pragma unroll
            for (int k = 0; k < LC_AHEAD; ++k) c[k] = i + k * LC_THREADS < row.h_hi ? a.history[i + k * LC_THREADS] : -1;
#pragma unroll
            for (int k = 0; k < LC_AHEAD; ++k)
                if (c[k] >= col0 && c[k] - col0 < n_cols) atomicAdd(&count[c[k] - col0], 1u);
        }
    }
    for (int i = row.b_lo + tid; i < row.b_hi; i += LC_THREADS) {
        const int id = a.bias_ids[i];
        if (id >= col0 && id - col0 < n_cols) atomicOr(&count[id - col0], LC_BIASED);
    }
    __syncthreads();
#pragma unroll 4
    for (int c = tid; c < n_cols; c += LC_THREADS) {
        const bool ok = !words || words[c >> 5] >> (c & 31) & 1u;
        const uint32_t n = count[c];
        if (!(n & LC_BIASED)) dst[c] = ok ? lc_edit(src[c], n, row.rep, row.presence, row.frequency) : -INFINITY;
    }
    for (int i = row.b_lo + tid; i < row.b_hi; i += LC_THREADS) {
        const int id = a.bias_ids[i], c = id - col0;
        if (id < col0 || c >= n_cols) continue;
        const bool ok = !words || words[c >> 5] >> (c & 31) & 1u;
        dst[c] = ok ? lc_edit(src[c] + a.bias[i], count[c] & ~LC_BIASED, row.rep, row.presence, row.frequency) : -INFINITY;
    }
}

// Out of place, and in place with masks: persistent blocks take slices one after the other, each a run of them, mostly of one row,
// whose numbers then stay in registers. A slice comes into shared memory by one bulk copy, asked for while the slice before it is edited, is
// edited there where there is something to edit, and leaves by another: the copies wait for nothing but each other. They go
// by 16 bytes: a slice begins at a boundary, and what of a first or last 16 bytes belongs to another row is read but not
// stored. (Both matrices' rows lie alike to the boundaries.)
//   Every thread keeps tokens of the history and looks which of them the slice has: those are counted, and after a barrier a
// thread comes for each of its own, takes the count out, and, if it was the first to come, edits the column. No thread
// looks at the columns that no token met, but for the mask's, whose words are read a slice ahead.
//   MEASURED, in a graph of calls: 64 rows of 151936 copied 13.9 us (by torch 13.4), with histories of 4001 tokens 18.3, with
// 300 biases each 20.5; 128 rows of trees' nodes with a mask a row 31.3 of 26.2 for the copy; one row 4.1. What is left
// over the copy is a row's beginning, which waits for three reads in a row (owner, its starts, its tokens), and the slices'
// barriers: slices of 4096 took 24 and 41 for 20.5 and 31.3, of 8192 with one block an SM 25 and 44, 256 threads 27 and 36.
#define LS_THREADS 512
#define LS_BLOCKS 2                  // of an SM
#define LS_RING 3
#define LS_COLUMNS 6144              // a slice: a whole number of four columns a thread
#define LS_AHEAD 8                   // tokens of the history that a thread keeps for all the slices of a row

__device__ int drafts_error_flag = 0;

__device__ __forceinline__ void ls_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(tg_smem(dst)), "l"(src), "r"(bytes), "r"(tg_smem(bar)) : "memory");
}
__device__ __forceinline__ void ls_store(void* dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(tg_smem(src)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

__global__ void __launch_bounds__(LS_THREADS, LS_BLOCKS) constrain_stream_kernel(const Constrain a, int slices) {
    constexpr int GROUPS = LS_COLUMNS / 4 / LS_THREADS;         // of four columns a thread
    extern __shared__ __align__(128) unsigned char ls_raw[];
    float* ring = (float*)ls_raw;                              // [LS_RING][LS_COLUMNS]
    uint32_t* count = (uint32_t*)(ring + LS_RING * LS_COLUMNS);
    uint64_t* full = (uint64_t*)(count + LS_COLUMNS);          // [LS_RING]
    const int tid = threadIdx.x;
    if (tid == 0) {
        for (int i = 0; i < LS_RING; ++i) tg_init(&full[i], 1);
        tg_init_done();
    }
    for (int i = tid; i < LS_COLUMNS / 4; i += LS_THREADS) ((uint4*)count)[i] = make_uint4(0u, 0u, 0u, 0u);
    pdl_wait();
    // A row's places are its columns and, before them, the `skip` numbers from the boundary on.
    // this block's slices: `todo` from slice `part` of row `r` on
    const int units = a.rows * slices, each = units / (int)gridDim.x, more = units - each * (int)gridDim.x;
    const int u0 = (int)blockIdx.x * each + min((int)blockIdx.x, more), todo = each + ((int)blockIdx.x < more ? 1 : 0);
    int r = u0 / slices, part = u0 - r * slices;
    int ask_r = r, ask_part = part, asked = 0;                 // the slice that is asked for next, by one thread
    auto ask = [&]() {
        const float* from = a.logits + ask_r * a.in_stride;
        const int b = asked % LS_RING, skip = (int)((uintptr_t)from >> 2 & 3);
        const int n = min(LS_COLUMNS, skip + a.vocab - ask_part * LS_COLUMNS);
        const uint32_t bytes = n > 0 ? (uint32_t)(n + 3 & ~3) * 4u : 0u;
        tg_expect(&full[b], bytes);
        if (bytes) ls_load(ring + b * LS_COLUMNS, from - skip + ask_part * LS_COLUMNS, bytes, &full[b]);
        ++asked;
        if (++ask_part == slices) { ask_part = 0; ++ask_r; }
    };
    if (tid == 0)
        while (asked < todo && asked < LS_RING - 2) ask();
    __syncthreads();
    ConstrainRow row;
    bool ok = true;
    const bool in_place = a.logits == a.out;
    const uint32_t* mask = nullptr;
    int said[LS_AHEAD], drafted = LC_NONE, bias_id = -1;            // this thread's first tokens of the history, its drafted one, its
    float bias_of = 0.f;                                       // first biased one
    uint32_t next_word[GROUPS] = {};                           // of the mask, for the next slice; where four columns lie in two
    uint32_t next_more[GROUPS] = {};                           // words, the second ones
    int skip = 0;
    const int last_word = a.vocab - 1 >> 5;
    auto read_mask = [&](int first) {                          // of the columns from there on, four a group; nothing here waits
        if (!mask) return;                                     // for what is read
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const int at = first + (i * LS_THREADS + tid) * 4 >> 5;                 // columns outside the row: any word
            next_word[i] = mask[max(0, min(at, last_word))];
            if (skip) next_more[i] = mask[max(0, min(at + 1, last_word))];
        }
    };
    for (int k = 0, b = 0, phase = 0; k < todo; ++k) {
        float* buf = ring + b * LS_COLUMNS;
        if (tid == 0 && asked < todo) {
            // the buffer of a slice to come: what lay there has been read out, but for the last slice's
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            ask();
        }
        if (k == 0 || part == 0) skip = (int)((uintptr_t)(a.logits + r * a.in_stride) >> 2 & 3);
        const int col0 = part * LS_COLUMNS - skip, n_cols = min(LS_COLUMNS, a.vocab - col0);       // to the slice's first place
        if (k == 0 || part == 0) {                             // another row
            const int q = a.owner ? a.owner[r] : r;
            mask = lc_mask(a, r);
            read_mask(col0);
            row.find(a, r, q);
#pragma unroll
            for (int j = 0; j < LS_AHEAD; ++j) said[j] = row.h_lo + j * LS_THREADS + tid < row.h_hi ? a.history[row.h_lo + j * LS_THREADS + tid] : LC_NONE;
            drafted = row.drafted(a, tid);
#pragma unroll
            for (int j = 0; j < LS_AHEAD; ++j) said[j] = said[j] < 0 ? LC_NONE : said[j];
            bias_id = row.b_lo + tid < row.b_hi ? a.bias_ids[row.b_lo + tid] : -1;
            bias_of = row.b_lo + tid < row.b_hi ? a.bias[row.b_lo + tid] : 0.f;
        }
        uint32_t word[GROUPS];
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) word[i] = __funnelshift_r(next_word[i], next_more[i], col0 + (i * LS_THREADS + tid) * 4 & 31) & 0xfu;
        if (part + 1 < slices) read_mask(col0 + LS_COLUMNS);
        const uint32_t width = (uint32_t)max(n_cols, 0);
        uint32_t here = 0;                                     // which of this thread's tokens the slice has
        if (row.counts) {
            auto count_in = [&](int token) {
                const uint32_t c = (uint32_t)(token - col0);
                if (c < width) atomicAdd(&count[c], 1u);
                return c < width;
            };
            here = count_in(drafted) ? 1u << LS_AHEAD : 0u;
#pragma unroll
            for (int j = 0; j < LS_AHEAD; ++j) {
                if (row.h_lo + j * LS_THREADS >= row.h_hi) break;
                if (count_in(said[j])) here |= 1u << j;
            }
            for (int i = row.h_lo + LS_AHEAD * LS_THREADS + tid; i < row.h_hi; i += LS_THREADS)
                if (a.history[i] >= 0) count_in(a.history[i]);
        }
        if (ok) ok = tg_wait(&full[b], phase, &drafts_error_flag, 1);
        ok = __syncthreads_and(ok);                            // each thread times its own wait: all leave, and know why
        if (!ok) break;
        if (row.b_hi > row.b_lo) {
            const uint32_t mine = (uint32_t)(bias_id - col0);
            if (bias_id >= 0 && mine < width) buf[mine] += bias_of;
            for (int i = row.b_lo + LS_THREADS + tid; i < row.b_hi; i += LS_THREADS) {
                const int id = a.bias_ids[i];
                const uint32_t c = (uint32_t)(id - col0);
                if (id >= 0 && c < width) buf[c] += a.bias[i];
            }
            __syncthreads();
        }
        if (row.counts) {
            auto edit = [&](int token) {                       // by the first thread that comes for the column
                const uint32_t c = (uint32_t)(token - col0), n = atomicExch(&count[c], 0u);
                if (n) buf[c] = lc_edit(buf[c], n, row.rep, row.presence, row.frequency);
            };
            for (; here; here &= here - 1) {
                const int which = __ffs(here) - 1;
                int token = drafted;
#pragma unroll
                for (int j = 0; j < LS_AHEAD; ++j)
                    if (j == which) token = said[j];
                edit(token);
            }
            for (int i = row.h_lo + LS_AHEAD * LS_THREADS + tid; i < row.h_hi; i += LS_THREADS) {
                const int token = a.history[i];
                if (token >= 0 && (uint32_t)(token - col0) < width) edit(token);
            }
            __syncthreads();                                   // the next slice's tokens are counted in the same places
        }
        if (mask) {
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                const int g = i * LS_THREADS + tid;
                const uint32_t bits = word[i];
                if (bits == 0xfu) continue;
                float4 v;
                if (bits) v = ((const float4*)buf)[g];
                if (!(bits & 1u)) v.x = -INFINITY;
                if (!(bits & 2u)) v.y = -INFINITY;
                if (!(bits & 4u)) v.z = -INFINITY;
                if (!(bits & 8u)) v.w = -INFINITY;
                ((float4*)buf)[g] = v;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        float* dst = a.out + (long long)r * a.out_stride + col0;
        // whole 16 bytes by a copy, what is before and behind them one by one
        const int lo = part == 0 ? skip : 0, lo4 = lo + 3 & ~3, hi4 = max(n_cols, 0) & ~3;
        const bool same = in_place && !mask && !row.counts && row.b_hi <= row.b_lo;                       // as it lies there
        if (tid == 0) {
            if (hi4 > lo4 && !same) ls_store(dst + lo4, buf + lo4, (uint32_t)(hi4 - lo4) * 4u);
            else asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        if (tid >= 32 && tid < 40 && !same) {
            const int c = tid < 36 ? lo + tid - 32 : max(hi4, lo4) + tid - 36;
            if (tid < 36 ? c < min(lo4, n_cols) : c < n_cols) dst[c] = buf[c];
        }
        if (++part == slices) { part = 0; ++r; }
        if (++b == LS_RING) { b = 0; phase ^= 1; }
    }
    if (tid == 0) {
        if (!ok) tg_settle_copies(full, LS_RING, asked, &drafts_error_flag, 1);        // not left with copies under way
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
}

TGO_API int tgo_logits_constrain_error(int* value) { return (int)cudaMemcpyFromSymbol(value, drafts_error_flag, sizeof(int)); }

// Launches of as many rows as a grid's second extent takes, mostly one.
#define LC_ROWS 65535
template <typename Launch> static int by_rows(Constrain& a, Launch&& launch) {
    for (long long r = 0; r < a.rows; r += LC_ROWS) {
        a.row0 = (int)r;
        const int rc = launch(a.rows - a.row0 < LC_ROWS ? a.rows - a.row0 : LC_ROWS);
        if (rc) return rc;
    }
    return 0;
}

// Addresses that are null leave their stage out. strides in elements (words for `allowed`).
TGO_API int tgo_logits_constrain(const float* logits, long long in_stride, float* out, long long out_stride, int rows, int vocab,
                                 int requests, const int* owner, const int* bias_start, const int* bias_ids, const float* bias,
                                 int n_bias, const int* history_start, const int* history, int n_history, const float* penalties,
                                 const int* windows, const int* draft_start, const int* draft_tokens, int n_drafts, const void* seen, const void* allowed,
                                 long long allowed_stride, int allowed_rows_n, const int* allowed_rows, cudaStream_t stream) {
    if (rows <= 0 || vocab <= 0) return 0;
    const int slices = (vocab + LC_COLUMNS - 1) / LC_COLUMNS;
    if ((rows > 1 && (in_stride < vocab || out_stride < vocab || (logits == out && in_stride != out_stride))) || requests < 0 ||
        (allowed && allowed_stride < (vocab + 31) / 32))
        return TGO_E_BAD_ARG;
    Constrain a = {logits, out, in_stride, out_stride, rows, vocab, requests, n_bias, n_history, n_drafts, owner, bias_start, bias_ids, bias, history_start, history,
                   penalties, windows, draft_start, draft_tokens, (const unsigned long long*)seen, (const uint32_t*)allowed,
                   allowed_stride, allowed_rows_n, allowed_rows, 0};
    if ((logits != out || allowed) && ((uintptr_t)logits - (uintptr_t)out) % 16 == 0 && (rows == 1 || (in_stride - out_stride) % 4 == 0) &&
        (long long)rows * ((vocab + 3) / LS_COLUMNS + 1) <= 0x7fffffffll) {
        constexpr size_t smem = (LS_RING + 1) * LS_COLUMNS * sizeof(float) + LS_RING * 8;
        static bool set[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return (int)e;
        if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
        if (!set[dev]) {
            e = cudaFuncSetAttribute(constrain_stream_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return (int)e;
            set[dev] = true;
        }
        // slices of the row that has most numbers before its first column
        const bool even = (uintptr_t)logits % 16 == 0 && (rows == 1 || in_stride % 4 == 0);
        const int cuts = (vocab + (even ? 0 : 3) + LS_COLUMNS - 1) / LS_COLUMNS;
        const int units = rows * cuts, blocks = LS_BLOCKS * tgo_multiprocessors();
        return tgo_launch_pdl(constrain_stream_kernel, dim3(units < blocks ? units : blocks), dim3(LS_THREADS), smem, stream, a, cuts);
    }
    if (logits == out && !allowed) {
        constexpr size_t smem = LI_COLUMNS * sizeof(uint32_t);
        static bool set[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return (int)e;
        if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
        if (!set[dev]) {
            e = cudaFuncSetAttribute(constrain_in_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return (int)e;
            set[dev] = true;
        }
        if (!bias_start && !penalties) return 0;
        return by_rows(a, [&](int n) {
            return tgo_launch_pdl(constrain_in_place_kernel, dim3((vocab + LI_COLUMNS - 1) / LI_COLUMNS, n), dim3(LI_THREADS), smem, stream, a);
        });
    }
    return by_rows(a, [&](int n) { return tgo_launch_pdl(constrain_kernel, dim3(slices, n), dim3(LC_THREADS), 0, stream, a); });
}

// --------------------------------------------------------------------------- tree_accept
// A warp a request; a lane holds nodes `lane` and `lane + 32`. Bound by latency, a read of the inputs and two ballots a step: 1.2 us for
// one request of 8 nodes, 1.6 for 64 of 64. From the node it stands on, the request goes on to the first
// later node that is its child and holds the token chosen at it.
__global__ void __launch_bounds__(32) accept_kernel(const int* __restrict__ tokens, const int* __restrict__ parents,
                                                    const int* __restrict__ chosen, const int* __restrict__ q_start,
                                                    int T,
                                                    int* __restrict__ path, int* __restrict__ counts, int* __restrict__ following) {
    pdl_wait();
    const int b = blockIdx.x, lane = threadIdx.x;
    int t0, end;
    dr_span(q_start, b, T, t0, end);
    const int all = end - t0, n = min(all, DR_NODES);
    int token[2] = {-1, -1}, parent[2] = {-1, -1}, pick[2] = {-1, -1}, mine[2] = {-1, -1};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        if (i < n) { token[h] = tokens[t0 + i]; parent[h] = parents[t0 + i]; pick[h] = chosen[t0 + i]; }
    }
    int at = 0, count = n > 0 ? 1 : 0, want = -1;
    if (lane == 0 && n > 0) mine[0] = 0;
    if (n > 0) {
        for (;;) {
            const int lo = __shfl_sync(0xffffffffu, pick[0], at & 31), hi = __shfl_sync(0xffffffffu, pick[1], at & 31);
            want = at < 32 ? lo : hi;
            const uint32_t m0 = __ballot_sync(0xffffffffu, lane < n && lane > at && parent[0] == at && token[0] == want);
            const uint32_t m1 = __ballot_sync(0xffffffffu, lane + 32 < n && lane + 32 > at && parent[1] == at && token[1] == want);
            if (!(m0 | m1)) break;
            at = m0 ? __ffs(m0) - 1 : __ffs(m1) + 31;
            if (lane == (count & 31)) { if (count < 32) mine[0] = at; else mine[1] = at; }
            ++count;
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
        if (lane + 32 * h < n) path[t0 + lane + 32 * h] = mine[h];
    for (int i = DR_NODES + lane; i < all; i += 32) path[t0 + i] = -1;
    if (lane == 0) { counts[b] = count; following[b] = want; }
}

TGO_API int tgo_tree_accept(const int* tokens, const int* parents, const int* chosen, const int* q_start, int requests,
                            int T, int* path, int* counts, int* following, cudaStream_t stream) {
    if (requests <= 0) return 0;
    return tgo_launch_pdl(accept_kernel, dim3(requests), dim3(32), 0, stream, tokens, parents, chosen, q_start, T, path, counts, following);
}

// ----------------------------------------------------------------------------- tree_keep
// Row slots[q_start + j] <- row slots[q_start + path[j]] for the accepted nodes j of a request, in place, in every tensor of
// pages [outer][pages][heads][page_size][row]. A path ascends, path[j] >= j: a row is only written when every
// earlier place has its own and no later one wants it, so a thread that goes along the path with one piece of
// all the rows, reading some before it writes them, needs no other thread. A block lists its request's moves first, without
// the rows that stay (node 0's always does).
//   MEASURED, in a graph of calls: 48 requests of up to 6 rows, 36 layers of K and V, 8 heads of 256 bytes: 10.2 us for 42.6
// MB (4.2 TB/s; four reads in a row before the first row is under way: start, path, slots, row). 8 rows ahead 11.4.
#define TK_THREADS 256
#define TK_MAX_TENSORS 64
#define TK_AHEAD 4                // rows read before they are written

struct KeepRows {
    char* base[TK_MAX_TENSORS];
    long long outer_stride[TK_MAX_TENSORS], page_stride[TK_MAX_TENSORS], head_stride[TK_MAX_TENSORS];
    int outer[TK_MAX_TENSORS], heads[TK_MAX_TENSORS], row_bytes[TK_MAX_TENSORS], pages[TK_MAX_TENSORS];
    int page_size;
};

template <typename V>
__global__ void __launch_bounds__(TK_THREADS) keep_kernel(const __grid_constant__ KeepRows a, const int* __restrict__ slots,
                                                          const int* __restrict__ q_start, int T,
                                                          const int* __restrict__ path, const int* __restrict__ counts) {
    __shared__ long long from[DR_NODES], to[DR_NODES];         // the rows that move, as offsets into a head's pages
    __shared__ int moves;
    pdl_wait();
    const int b = blockIdx.y, t = blockIdx.z, tid = threadIdx.x;
    int t0, end;
    dr_span(q_start, b, T, t0, end);
    const int n = min(end - t0, DR_NODES), count = min(counts[b], n);
    if (count <= 1) return;
    if (tid < 32) {
        const long long rows = (long long)a.pages[t] * a.page_size;
        auto offset = [&](int slot) {
            return slot / a.page_size * a.page_stride[t] + (long long)(slot % a.page_size) * a.row_bytes[t];
        };
        int kept = 0;
        for (int j0 = 0; j0 < count; j0 += 32) {
            const int j = j0 + tid, p = j < count ? path[t0 + j] : -1;
            const int d = j < count ? slots[t0 + j] : -1, s = p > j && p < n ? slots[t0 + p] : -1;
            const bool go = s >= 0 && d >= 0 && s < rows && d < rows;
            const uint32_t going = __ballot_sync(0xffffffffu, go);
            if (go) {
                const int at = kept + __popc(going & (1u << tid) - 1u);
                from[at] = offset(s);
                to[at] = offset(d);
            }
            kept += __popc(going);
        }
        if (tid == 0) moves = kept;
    }
    __syncthreads();
    const uint32_t pieces = (uint32_t)a.row_bytes[t] / (uint32_t)sizeof(V), heads = (uint32_t)a.heads[t];
    const uint32_t i = blockIdx.x * TK_THREADS + tid, oh = i / pieces, o = oh / heads;
    if (o >= (uint32_t)a.outer[t]) return;
    char* base = a.base[t] + o * a.outer_stride[t] + (oh - o * heads) * a.head_stride[t] + (size_t)(i - oh * pieces) * sizeof(V);
    const int all = moves;
    for (int j = 0; j < all; j += TK_AHEAD) {
        V v[TK_AHEAD];
#pragma unroll
        for (int k = 0; k < TK_AHEAD; ++k)
            if (j + k < all) v[k] = *(const V*)(base + from[j + k]);
#pragma unroll
        for (int k = 0; k < TK_AHEAD; ++k)
            if (j + k < all) *(V*)(base + to[j + k]) = v[k];
    }
}

template <typename V>
static int keep_launch(const KeepRows& a, int n, int requests, long long blocks, const int* slots, const int* q_start,
                       int T, const int* path, const int* counts, cudaStream_t stream) {
    return tgo_launch_pdl(keep_kernel<V>, dim3((unsigned)blocks, requests, n), dim3(TK_THREADS), 0, stream, a, slots, q_start, T, path, counts);
}

// desc: per tensor five numbers: address, outer count, pages, heads, bytes of a row; all contiguous
// [outer][pages][heads][page_size][row].
TGO_API int tgo_tree_keep(const long long* desc, int tensors, int page_size, const int* slots, const int* q_start, int requests,
                          int T, const int* path, const int* counts, cudaStream_t stream) {
    if (tensors <= 0 || requests <= 0) return 0;
    if (page_size <= 0 || requests > 65535) return TGO_E_BAD_ARG;
    for (int first = 0; first < tensors; first += TK_MAX_TENSORS) {
        KeepRows a;
        const int n = tensors - first < TK_MAX_TENSORS ? tensors - first : TK_MAX_TENSORS;
        long long all = 0, blocks = 0;
        for (int i = 0; i < n; ++i) {
            const long long* q = desc + 5 * (first + i);
            if (q[1] <= 0 || q[1] > 0x7fffffff || q[2] <= 0 || q[3] <= 0 || q[3] > 0x7fffffff || q[4] <= 0 || q[4] > 0x7fffffff ||
                q[2] > 0x7fffffffll / page_size)
                return TGO_E_BAD_ARG;
            a.base[i] = (char*)q[0];
            a.outer[i] = (int)q[1];
            a.pages[i] = (int)q[2];
            a.heads[i] = (int)q[3];
            a.row_bytes[i] = (int)q[4];
            a.head_stride[i] = (long long)page_size * q[4];
            a.page_stride[i] = a.head_stride[i] * q[3];
            a.outer_stride[i] = a.page_stride[i] * q[2];
            all |= q[0] | q[4];
        }
        a.page_size = page_size;
        const int width = all & 1 ? 1 : all & 2 ? 2 : all & 4 ? 4 : all & 8 ? 8 : 16;
        for (int i = 0; i < n; ++i) {
            const long long c = ((long long)a.outer[i] * a.heads[i] * (a.row_bytes[i] / width) + TK_THREADS - 1) / TK_THREADS;
            blocks = c > blocks ? c : blocks;
        }
        if (blocks > 0x7fffffff / TK_THREADS) return TGO_E_BAD_ARG;         // pieces are counted in 32 bits
        int rc;
        if (width == 16) rc = keep_launch<uint4>(a, n, requests, blocks, slots, q_start, T, path, counts, stream);
        else if (width == 8) rc = keep_launch<uint2>(a, n, requests, blocks, slots, q_start, T, path, counts, stream);
        else if (width == 4) rc = keep_launch<uint32_t>(a, n, requests, blocks, slots, q_start, T, path, counts, stream);
        else if (width == 2) rc = keep_launch<uint16_t>(a, n, requests, blocks, slots, q_start, T, path, counts, stream);
        else return TGO_E_BAD_ARG;
        if (rc) return rc;
    }
    return 0;
}
