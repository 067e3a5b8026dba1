// What a step of drafted tokens needs beside its attention: rows of logits constrained (biases, penalties for repeated
// tokens, masks of allowed ones), the path through a tree of drafts that the chosen tokens confirm, and the accepted
// nodes' rows of the cache moved together.
#include "common.cuh"

#define DR_NODES 64               // most drafted tokens of a request: a path is a 64-bit number

// ---------------------------------------------------------------------- logits_constrain
// Row r of request q = owner[r], token i:
//   x = logits[r, i] + bias_q(i)
//   c = how often i stands in the last `window` tokens of (q's history, then the drafted tokens of r's own path)
//   c > 0:  x = x > 0 ? x / repetition : x * repetition;  x -= presence + frequency * c
//   not allowed: x = -inf
// the order and the arithmetic of the sampler's single rows (adjust_kernel of sampling.cu), so that both give the same bits.
//
// A block takes a slice of 8192 columns of a row. It asks for the slice's logits first, counts the history's tokens that fall
// into its slice in shared memory while they come (integers: the order of the additions changes nothing), and then edits
// and stores. A biased token is left to a second look, when everything else of the slice is done. In place, a
// group of four columns without a counted or a forbidden token is neither read nor written.
#define LC_THREADS 256
#define LC_VPT 8                  // groups of four columns a thread
#define LC_COLUMNS (LC_THREADS * LC_VPT * 4)
#define LC_BIASED 0x80000000u

struct Constrain {
    const float* logits; float* out;
    long long in_stride, out_stride;
    int rows, vocab, requests;
    const int* owner;
    const int *bias_start, *bias_ids; const float* bias;
    const int *history_start, *history;
    const float* penalties;                  // [requests][repetition, presence, frequency]
    const int* windows;                      // null: every history whole
    const int *draft_start, *draft_tokens; const unsigned long long* seen;
    const uint32_t* allowed; long long allowed_stride; int allowed_rows_n;
    const int* allowed_rows;
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

template <bool VECTORS>
__global__ void __launch_bounds__(LC_THREADS) constrain_kernel(const Constrain a) {
    __shared__ __align__(16) uint32_t count[LC_COLUMNS];
    pdl_wait();
    const int tid = threadIdx.x, r = blockIdx.y;
    const int col0 = blockIdx.x * LC_COLUMNS;
    const int n_cols = min(LC_COLUMNS, a.vocab - col0);
    const float* src = a.logits + (size_t)r * a.in_stride + col0;
    float* dst = a.out + (size_t)r * a.out_stride + col0;
    const bool in_place = a.logits == a.out;
    const int q = a.owner ? a.owner[r] : r;
    const bool owned = q >= 0 && q < a.requests;
    float4 x[LC_VPT];
    if (VECTORS && !in_place) {
#pragma unroll
        for (int i = 0; i < LC_VPT; ++i) {
            const int c = (i * LC_THREADS + tid) * 4;
            if (c + 3 < n_cols) x[i] = __ldcs((const float4*)(src + c));
        }
    }
#pragma unroll
    for (int i = 0; i < LC_VPT; ++i) ((uint4*)count)[i * LC_THREADS + tid] = make_uint4(0u, 0u, 0u, 0u);
    const uint32_t* words = nullptr;
    if (a.allowed) {
        const int w = a.allowed_rows ? a.allowed_rows[r] : r;
        if (w >= 0 && w < a.allowed_rows_n) words = a.allowed + (size_t)w * a.allowed_stride + (col0 >> 5);
    }
    float rep = 1.f, presence = 0.f, frequency = 0.f;
    int b_lo = 0, b_hi = 0;
    bool counts = false;
    if (owned && a.bias_start) { b_lo = a.bias_start[q]; b_hi = a.bias_start[q + 1]; }
    if (owned && a.penalties) {
        rep = a.penalties[3 * q]; presence = a.penalties[3 * q + 1]; frequency = a.penalties[3 * q + 2];
        counts = (rep != 0.f && rep != 1.f) || presence != 0.f || frequency != 0.f;
    }
    __syncthreads();
    if (counts) {
        int room = a.windows ? a.windows[q] : 0;
        if (room <= 0) room = 0x7fffffff;
        if (a.seen) {
            unsigned long long path = a.seen[r];
            const int t0 = a.draft_start[q], n = min(a.draft_start[q + 1] - t0, DR_NODES);
            path &= n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
            const int length = __popcll(path);
            if (tid < DR_NODES && path >> tid & 1ull && __popcll(path >> tid) <= room) {
                const int c = a.draft_tokens[t0 + tid] - col0;
                if (c >= 0 && c < n_cols) atomicAdd(&count[c], 1u);
            }
            room -= min(room, length);
        }
        if (a.history_start) {
            int lo = a.history_start[q];
            const int hi = a.history_start[q + 1];
            if (hi - lo > room) lo = hi - room;
#pragma unroll 4
            for (int i = lo + tid; i < hi; i += LC_THREADS) {
                const int c = a.history[i] - col0;
                if (c >= 0 && c < n_cols) atomicAdd(&count[c], 1u);
            }
        }
    }
    for (int i = b_lo + tid; i < b_hi; i += LC_THREADS) {
        const int c = a.bias_ids[i] - col0;
        if (c >= 0 && c < n_cols) atomicOr(&count[c], LC_BIASED);
    }
    __syncthreads();
    auto value = [&](float v, uint32_t n, uint32_t allowed) {
        if (n & LC_BIASED) return v;
        if (!(allowed & 1u)) return -INFINITY;
        return lc_edit(v, n, rep, presence, frequency);
    };
    if (VECTORS) {
#pragma unroll
        for (int i = 0; i < LC_VPT; ++i) {
            const int g = i * LC_THREADS + tid, c = g * 4;
            if (c >= n_cols) break;
            const uint4 n = ((const uint4*)count)[g];
            const uint32_t bits = words ? words[c >> 5] >> (c & 31) : 0xfu;
            if (in_place && (bits & 0xfu) == 0xfu && !((n.x | n.y | n.z | n.w) & ~LC_BIASED)) continue;
            if (c + 3 < n_cols) {
                float4 v;
                if (in_place) v = *(const float4*)(src + c); else v = x[i];
                v.x = value(v.x, n.x, bits); v.y = value(v.y, n.y, bits >> 1);
                v.z = value(v.z, n.z, bits >> 2); v.w = value(v.w, n.w, bits >> 3);
                __stcs((float4*)(dst + c), v);
            } else {
                for (int k = 0; c + k < n_cols; ++k) dst[c + k] = value(src[c + k], count[c + k], bits >> k);
            }
        }
    } else {
        for (int c = tid; c < n_cols; c += LC_THREADS) {
            const uint32_t bits = words ? words[c >> 5] >> (c & 31) : 1u;
            if (in_place && (bits & 1u) && !(count[c] & ~LC_BIASED)) continue;
            dst[c] = value(src[c], count[c], bits);
        }
    }
    if (b_hi > b_lo) {
        __syncthreads();
        for (int i = b_lo + tid; i < b_hi; i += LC_THREADS) {
            const int c = a.bias_ids[i] - col0;
            if (c < 0 || c >= n_cols) continue;
            const bool ok = !words || words[c >> 5] >> (c & 31) & 1u;
            dst[c] = ok ? lc_edit(src[c] + a.bias[i], count[c] & ~LC_BIASED, rep, presence, frequency) : -INFINITY;
        }
    }
}

// Addresses that are null leave their stage out. strides in elements (words for `allowed`).
TGO_API int tgo_logits_constrain(const float* logits, long long in_stride, float* out, long long out_stride, int rows, int vocab,
                                 int requests, const int* owner, const int* bias_start, const int* bias_ids, const float* bias,
                                 const int* history_start, const int* history, const float* penalties, const int* windows,
                                 const int* draft_start, const int* draft_tokens, const void* seen, const void* allowed,
                                 long long allowed_stride, int allowed_rows_n, const int* allowed_rows, cudaStream_t stream) {
    if (rows <= 0 || vocab <= 0) return 0;
    const int slices = (vocab + LC_COLUMNS - 1) / LC_COLUMNS;
    if (rows > 65535 || (rows > 1 && (in_stride < vocab || out_stride < vocab)) || requests < 0 ||
        (allowed && allowed_stride < (vocab + 31) / 32))
        return TGO_E_BAD_ARG;
    Constrain a = {logits, out, in_stride, out_stride, rows, vocab, requests, owner, bias_start, bias_ids, bias, history_start, history,
                   penalties, windows, draft_start, draft_tokens, (const unsigned long long*)seen, (const uint32_t*)allowed,
                   allowed_stride, allowed_rows_n, allowed_rows};
    const bool vectors = ((uintptr_t)logits % 16 == 0 && (uintptr_t)out % 16 == 0) && (rows == 1 || (in_stride % 4 == 0 && out_stride % 4 == 0));
    if (vectors) return tgo_launch_pdl(constrain_kernel<true>, dim3(slices, rows), dim3(LC_THREADS), 0, stream, a);
    return tgo_launch_pdl(constrain_kernel<false>, dim3(slices, rows), dim3(LC_THREADS), 0, stream, a);
}

// --------------------------------------------------------------------------- tree_accept
// A warp a request; a lane holds nodes `lane` and `lane + 32`. From the node it stands on, the request goes on to the first
// later node that is its child and holds the token chosen at it.
__global__ void __launch_bounds__(32) accept_kernel(const int* __restrict__ tokens, const int* __restrict__ parents,
                                                    const int* __restrict__ chosen, const int* __restrict__ q_start,
                                                    int* __restrict__ path, int* __restrict__ counts, int* __restrict__ following) {
    pdl_wait();
    const int b = blockIdx.x, lane = threadIdx.x;
    const int t0 = q_start[b], all = q_start[b + 1] - t0;
    const int n = min(all, DR_NODES);
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
                            int* path, int* counts, int* following, cudaStream_t stream) {
    if (requests <= 0) return 0;
    return tgo_launch_pdl(accept_kernel, dim3(requests), dim3(32), 0, stream, tokens, parents, chosen, q_start, path, counts, following);
}

// ----------------------------------------------------------------------------- tree_keep
// Row slots[q_start + j] <- row slots[q_start + path[j]] for the accepted nodes j of a request, in place, in every tensor of
// pages [outer][pages][heads][page_size][row]. A path ascends, path[j] >= j: a row is only written when every
// earlier place has its own and no later one wants it, so a thread that goes along the path with one piece of
// all the rows, reading some before it writes them, needs no other thread.
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
                                                          const int* __restrict__ q_start, const int* __restrict__ path,
                                                          const int* __restrict__ counts) {
    __shared__ int from[DR_NODES], to[DR_NODES];
    pdl_wait();
    const int b = blockIdx.y, t = blockIdx.z, tid = threadIdx.x;
    const int t0 = q_start[b], n = min(q_start[b + 1] - t0, DR_NODES);
    const int count = min(counts[b], n);
    if (count <= 1) return;
    const long long rows = (long long)a.pages[t] * a.page_size;
    if (tid < count) {
        const int p = path[t0 + tid];
        int s = p >= tid && p < n ? slots[t0 + p] : -1, d = slots[t0 + tid];
        if (s < 0 || d < 0 || s >= rows || d >= rows || p == tid) s = d = -1;
        from[tid] = s;
        to[tid] = d;
    }
    __syncthreads();
    const int pieces = a.row_bytes[t] / (int)sizeof(V);
    const long long total = (long long)a.outer[t] * a.heads[t] * pieces;
    const long long i = (long long)blockIdx.x * TK_THREADS + tid;
    if (i >= total) return;
    const int piece = (int)(i % pieces);
    const long long oh = i / pieces;
    char* base = a.base[t] + oh / a.heads[t] * a.outer_stride[t] + oh % a.heads[t] * a.head_stride[t] + (size_t)piece * sizeof(V);
    auto at = [&](int slot) {
        return (V*)(base + (long long)(slot / a.page_size) * a.page_stride[t] + (long long)(slot % a.page_size) * a.row_bytes[t]);
    };
    for (int j = 0; j < count; j += TK_AHEAD) {
        V v[TK_AHEAD];
#pragma unroll
        for (int k = 0; k < TK_AHEAD; ++k)
            if (j + k < count && from[j + k] >= 0) v[k] = *at(from[j + k]);
#pragma unroll
        for (int k = 0; k < TK_AHEAD; ++k)
            if (j + k < count && from[j + k] >= 0) *at(to[j + k]) = v[k];
    }
}

template <typename V>
static int keep_launch(const KeepRows& a, int n, int requests, long long blocks, const int* slots, const int* q_start,
                       const int* path, const int* counts, cudaStream_t stream) {
    return tgo_launch_pdl(keep_kernel<V>, dim3((unsigned)blocks, requests, n), dim3(TK_THREADS), 0, stream, a, slots, q_start, path, counts);
}

// desc: per tensor five numbers: address, outer count, pages, heads, bytes of a row; all contiguous
// [outer][pages][heads][page_size][row].
TGO_API int tgo_tree_keep(const long long* desc, int tensors, int page_size, const int* slots, const int* q_start, int requests,
                          const int* path, const int* counts, cudaStream_t stream) {
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
        if (blocks > 0x7fffff00) return TGO_E_BAD_ARG;
        int rc;
        if (width == 16) rc = keep_launch<uint4>(a, n, requests, blocks, slots, q_start, path, counts, stream);
        else if (width == 8) rc = keep_launch<uint2>(a, n, requests, blocks, slots, q_start, path, counts, stream);
        else if (width == 4) rc = keep_launch<uint32_t>(a, n, requests, blocks, slots, q_start, path, counts, stream);
        else if (width == 2) rc = keep_launch<uint16_t>(a, n, requests, blocks, slots, q_start, path, counts, stream);
        else return TGO_E_BAD_ARG;
        if (rc) return rc;
    }
    return 0;
}
