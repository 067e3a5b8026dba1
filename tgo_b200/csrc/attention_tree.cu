// Attention of trees of drafted tokens over the paged cache.
//
// Request b brings n_b <= 64 nodes (tokens q_start[b] .. q_start[b+1]); node i's key and value lie at position
// base_b + i of its cache, base_b = context_lens[b] - n_b. seen[t] says by its bits which nodes of its request node t sees;
// its position is p = base + (bits set) - 1. With x = scale q . k,
//   out = sum_k e^x v / sum_k e^x  over  { cached k < base, k > p - window (window 0: all) } and { base + j : bit j of seen },
// zeros where that is nothing.
//
// How the work is shared out. An item is a tile of query rows (node, query head of the group) of one request and kv head; it
// walks the request's keys tile by tile, and the K and V of a kv head serve all its rows. The items of all requests, laid
// end to end, are cut into equally long pieces, one a worker, whatever the requests' lengths: a worker has the rest of an
// item, some whole ones, and the beginning of another. (An item counts TREE_OVERHEAD tiles more than it has: its start
// and its end take time too.) Every worker finds its piece from the lengths on the device, so nothing of it depends on the host
// and a captured call fits every step. What is cut leaves an unnormalised sum, a maximum and a sum of exponentials per
// row in the workspace, at most two of them a worker, and a second kernel joins them, in the order of the keys: equal
// calls give equal bits.
#include "common.cuh"

#define TREE_NODES 64
#define TREE_OVERHEAD 1

struct TreeWork {
    const int *context_lens, *q_start;
    int B, H, Hkv, window, max_keys;          // max_keys: what a block table can name
    int rows_per_tile, tokens_per_tile;       // a tile holds so many rows, or (if not 0) so many whole tokens
    int key_tile, min_units;
    int workers;                              // at most
};

struct TreeRequest {
    int tok0, n, base, len, t_lo, tiles, row_tiles;
    long long units;                          // of all its items
};

__device__ __forceinline__ TreeRequest tree_request(const TreeWork& w, int b) {
    TreeRequest r;
    r.tok0 = w.q_start[b];
    r.n = min(max(w.q_start[b + 1] - r.tok0, 0), TREE_NODES);
    r.len = w.context_lens[b];
    r.base = r.len - r.n;
    const bool none = r.base < 0;             // a padded request: its rows get zeros
    const int hi = none ? 0 : min(r.len, w.max_keys);
    const int lo = w.window > 0 && r.base - w.window > 0 ? r.base - w.window : 0;
    r.t_lo = none ? 0 : lo / w.key_tile;
    r.tiles = max((hi + w.key_tile - 1) / w.key_tile - r.t_lo, 1);
    const int G = w.H / w.Hkv;
    r.row_tiles = w.tokens_per_tile ? (r.n + w.tokens_per_tile - 1) / w.tokens_per_tile
                                    : (r.n * G + w.rows_per_tile - 1) / w.rows_per_tile;
    r.units = (long long)r.row_tiles * w.Hkv * (r.tiles + TREE_OVERHEAD);
    return r;
}

// All units, by one warp.
__device__ __forceinline__ long long tree_total(const TreeWork& w) {
    long long sum = 0;
    for (int b = threadIdx.x & 31; b < w.B; b += 32) sum += tree_request(w, b).units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
__device__ __forceinline__ int tree_workers(const TreeWork& w, long long total) {
    const long long most = total / w.min_units;
    return most < 1 ? 1 : most < w.workers ? (int)most : w.workers;
}
__device__ __forceinline__ long long tree_begin(long long total, int workers, int i) {
    return total / workers * i + (total % workers) * i / workers;
}
// The request that unit u lies in and its first unit, by one warp; u < the total.
__device__ __forceinline__ int tree_find(const TreeWork& w, long long u, long long& first) {
    const int lane = threadIdx.x & 31;
    long long before = 0;
    for (int b0 = 0; b0 < w.B; b0 += 32) {
        const long long mine = b0 + lane < w.B ? tree_request(w, b0 + lane).units : 0;
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const uint32_t in = __ballot_sync(0xffffffffu, u < before + upto);
        if (in) {
            const int l = __ffs(in) - 1;
            first = before + __shfl_sync(0xffffffffu, upto - mine, l);
            return b0 + l;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    first = before;
    return w.B;
}

// A worker's walk over its pieces: `next` gives them one after the other.
struct TreeWalk {
    long long u, end, first;                  // where it stands, where its piece ends, where request b begins
    int b;
    TreeRequest r;
    // of the piece
    int kvh, row_tile, from, to;              // key tiles from .. to - 1 of the item
    __device__ __forceinline__ bool next(const TreeWork& w) {
        while (u < end) {
            while (u >= first + r.units) {
                first += r.units;
                if (++b >= w.B) return false;
                r = tree_request(w, b);
            }
            const int item_units = r.tiles + TREE_OVERHEAD;
            const int item = (int)((u - first) / item_units);
            const long long s = first + (long long)item * item_units;
            from = max((int)(u - s) - TREE_OVERHEAD, 0);
            to = end - s >= item_units ? r.tiles : max((int)(end - s) - TREE_OVERHEAD, 0);
            kvh = item / r.row_tiles;
            row_tile = item % r.row_tiles;
            u = s + item_units;
            if (to > from) return true;
        }
        return false;
    }
};
// The walk of worker i, found by one warp.
__device__ __forceinline__ TreeWalk tree_walk(const TreeWork& w, long long total, int workers, int i) {
    TreeWalk k;
    k.u = tree_begin(total, workers, i);
    k.end = tree_begin(total, workers, i + 1);
    k.b = tree_find(w, k.u, k.first);
    k.r = tree_request(w, min(k.b, w.B - 1));
    return k;
}

// What a row may see of its request's keys.
struct TreeRow {
    int lo;                                   // cached keys from here on
    unsigned long long bits;
    __device__ __forceinline__ bool sees(int key, int base, int n) const {
        return key < base ? key >= lo : key - base < n && (bits >> (key - base) & 1ull);
    }
};
__device__ __forceinline__ TreeRow tree_row(const TreeWork& w, const TreeRequest& r, const unsigned long long* seen, int token) {
    TreeRow t;
    t.bits = seen[r.tok0 + token] & (r.n >= 64 ? ~0ull : (1ull << r.n) - 1ull);
    const int lo = r.base + __popcll(t.bits) - w.window;
    t.lo = w.window > 0 && lo > 0 ? lo : 0;
    return t;
}

#define TREE_LOG2E 1.44269504088896341f

// ------------------------------------------------------------------------- plain products
// float32, and bfloat16 where the tensor cores' kernel has no instance: 32 rows and 64 keys a tile on the FMA units, sixteen
// threads a pair of rows. A thread makes 2 x 4 scores, then 2 x (width / 16) outputs; rows lie in shared memory 4 floats
// further apart than they are wide, so that eight threads' 16-byte reads meet no bank twice.
// A masked score becomes the weight -0, which no exponential gives: in tiles that not every row sees whole, such
// a weight is left out of the sum, so that what lies in a masked place (an infinity, a NaN) does not reach it.
#define TP_ROWS 32
#define TP_KEYS 64
#define TP_THREADS 256

__device__ __forceinline__ float4 tp_load4(const float* p) { return *(const float4*)p; }
__device__ __forceinline__ float4 tp_load4(const bf16* p) {
    const uint2 u = *(const uint2*)p;
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

template <typename T, int DP>
__global__ void __launch_bounds__(TP_THREADS) tree_plain_kernel(
    const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const T* __restrict__ k_cache,
    const T* __restrict__ v_cache, int n_pages, int page_size, const int* __restrict__ block_tables, int max_blocks,
    const unsigned long long* __restrict__ seen, int dh, float scale, const TreeWork w, float* __restrict__ part_o,
    float* __restrict__ part_ml) {
    constexpr int LD = DP + 4, LS = TP_KEYS + 4, J = DP / 64;
    extern __shared__ __align__(16) float tp_smem[];
    float* sq = tp_smem;                          // [TP_ROWS][LD]
    float* sk = sq + TP_ROWS * LD;                // [TP_KEYS][LD]
    float* sv = sk + TP_KEYS * LD;                // [TP_KEYS][LD]
    float* ss = sv + TP_KEYS * LD;                // [TP_ROWS][LS]
    __shared__ TreeWalk s_walk;
    __shared__ int s_workers;
    pdl_wait();
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    if (tid < 32) {
        const long long total = tree_total(w);
        const int workers = total > 0 ? tree_workers(w, total) : 0;
        TreeWalk k;
        if ((int)blockIdx.x < workers) k = tree_walk(w, total, workers, blockIdx.x);
        if (tid == 0) { s_workers = workers; if ((int)blockIdx.x < workers) s_walk = k; }
    }
    __syncthreads();
    if ((int)blockIdx.x >= s_workers) return;
    TreeWalk walk = s_walk;
    const int G = w.H / w.Hkv;
    const float c = scale * TREE_LOG2E;
    const bool vectors = dh % 4 == 0 && ((uintptr_t)k_cache | (uintptr_t)v_cache) % (4 * sizeof(T)) == 0;
    while (walk.next(w)) {
        const TreeRequest r = walk.r;
        const int row0 = walk.row_tile * TP_ROWS, n_rows = min(r.n * G - row0, TP_ROWS);
        const int kvh = walk.kvh;
        __syncthreads();                          // the last piece's rows have been read
        for (int i = tid; i < TP_ROWS * DP; i += TP_THREADS) {
            const int row = i / DP, d = i % DP, f = row0 + row;
            sq[row * LD + d] = row < n_rows && d < dh
                ? to_f32(q[(size_t)(r.tok0 + f / G) * q_stride + (size_t)(kvh * G + f % G) * dh + d]) : 0.f;
        }
        TreeRow see[2];
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float o[2][J * 4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = ty * 2 + i;
            if (row < n_rows) see[i] = tree_row(w, r, seen, (row0 + row) / G);
            else { see[i].lo = 0x7fffffff; see[i].bits = 0; }
#pragma unroll
            for (int d = 0; d < J * 4; ++d) o[i][d] = 0.f;
        }
        const int hi = r.base < 0 ? 0 : min(r.len, w.max_keys);
        const int* bt = block_tables + (size_t)walk.b * max_blocks;
        for (int t = walk.from; t < walk.to; ++t) {
            const int key0 = (r.t_lo + t) * TP_KEYS;
            __syncthreads();                      // the last tile's K and V have been read
            for (int i = tid; i < TP_KEYS * (DP / 4); i += TP_THREADS) {
                const int row = i / (DP / 4), d = i % (DP / 4) * 4, key = key0 + row;
                float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
                const int page = key < hi ? bt[key / page_size] : -1;
                if (page >= 0 && page < n_pages && d < dh) {
                    const size_t at = (((size_t)page * w.Hkv + kvh) * page_size + key % page_size) * dh + d;
                    if (vectors) {
                        a = tp_load4(k_cache + at);
                        b = tp_load4(v_cache + at);
                    } else {
                        float ka[4], va[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ka[e] = d + e < dh ? to_f32(k_cache[at + e]) : 0.f;
                            va[e] = d + e < dh ? to_f32(v_cache[at + e]) : 0.f;
                        }
                        a = make_float4(ka[0], ka[1], ka[2], ka[3]);
                        b = make_float4(va[0], va[1], va[2], va[3]);
                    }
                }
                *(float4*)(sk + row * LD + d) = a;
                *(float4*)(sv + row * LD + d) = b;
            }
            __syncthreads();
            float x[2][4] = {};
#pragma unroll 8
            for (int d = 0; d < DP; d += 4) {
                float4 a[2], b[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) a[i] = *(const float4*)(sq + (ty * 2 + i) * LD + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = *(const float4*)(sk + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[i][j] = fmaf(a[i].x, b[j].x, x[i][j]);
                        x[i][j] = fmaf(a[i].y, b[j].y, x[i][j]);
                        x[i][j] = fmaf(a[i].z, b[j].z, x[i][j]);
                        x[i][j] = fmaf(a[i].w, b[j].w, x[i][j]);
                    }
            }
            bool ok[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = key0 + tx + 16 * j;
                    ok[i][j] = key < hi && see[i].sees(key, r.base, r.n);
                    if (ok[i][j]) mx = fmaxf(mx, x[i][j]);
                }
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                const float m_new = fmaxf(m[i], mx * c);
                const float corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                m[i] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p = ok[i][j] ? exp2f(fmaf(x[i][j], c, -ref)) : -0.f;
                    sum += p;
                    ss[(ty * 2 + i) * LS + tx + 16 * j] = p;
                }
                l[i] = l[i] * corr + sum;
#pragma unroll
                for (int d = 0; d < J * 4; ++d) o[i][d] *= corr;
            }
            __syncwarp();                         // a pair of rows belongs to half a warp
            // all of the tile's keys are seen by every row: cached, behind every window's beginning
            const bool whole = key0 + TP_KEYS <= min(hi, r.base) && (w.window <= 0 || key0 >= r.base + r.n - w.window);
            if (whole) {
#pragma unroll 2
                for (int k = 0; k < TP_KEYS; k += 4) {
                    const float4 p0 = *(const float4*)(ss + (ty * 2) * LS + k), p1 = *(const float4*)(ss + (ty * 2 + 1) * LS + k);
                    const float pa[4] = {p0.x, p0.y, p0.z, p0.w}, pb[4] = {p1.x, p1.y, p1.z, p1.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            const float4 v = *(const float4*)(sv + (k + e) * LD + tx * 4 + 64 * j);
                            o[0][4 * j] = fmaf(pa[e], v.x, o[0][4 * j]); o[0][4 * j + 1] = fmaf(pa[e], v.y, o[0][4 * j + 1]);
                            o[0][4 * j + 2] = fmaf(pa[e], v.z, o[0][4 * j + 2]); o[0][4 * j + 3] = fmaf(pa[e], v.w, o[0][4 * j + 3]);
                            o[1][4 * j] = fmaf(pb[e], v.x, o[1][4 * j]); o[1][4 * j + 1] = fmaf(pb[e], v.y, o[1][4 * j + 1]);
                            o[1][4 * j + 2] = fmaf(pb[e], v.z, o[1][4 * j + 2]); o[1][4 * j + 3] = fmaf(pb[e], v.w, o[1][4 * j + 3]);
                        }
                }
            } else {
#pragma unroll 2
                for (int k = 0; k < TP_KEYS; ++k) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float p = ss[(ty * 2 + i) * LS + k];
                        if (__float_as_uint(p) == 0x80000000u) continue;
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            const float4 v = *(const float4*)(sv + k * LD + tx * 4 + 64 * j);
                            o[i][4 * j] = fmaf(p, v.x, o[i][4 * j]); o[i][4 * j + 1] = fmaf(p, v.y, o[i][4 * j + 1]);
                            o[i][4 * j + 2] = fmaf(p, v.z, o[i][4 * j + 2]); o[i][4 * j + 3] = fmaf(p, v.w, o[i][4 * j + 3]);
                        }
                    }
                }
            }
        }
        const bool whole_item = walk.from == 0 && walk.to == r.tiles;
        const size_t slot = (size_t)blockIdx.x * 2 + (walk.from == 0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float sum = l[i];
#pragma unroll
            for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            const int row = ty * 2 + i, f = row0 + row;
            if (row >= n_rows) continue;
            if (whole_item) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                T* dst = out + (size_t)(r.tok0 + f / G) * out_stride + (size_t)(kvh * G + f % G) * dh;
#pragma unroll
                for (int d = 0; d < J * 4; ++d) {
                    const int col = tx * 4 + 64 * (d >> 2) + (d & 3);
                    if (col < dh) dst[col] = from_f32<T>(o[i][d] * inv);
                }
            } else {
                float* dst = part_o + (slot * TP_ROWS + row) * dh;
#pragma unroll
                for (int d = 0; d < J * 4; ++d) {
                    const int col = tx * 4 + 64 * (d >> 2) + (d & 3);
                    if (col < dh) dst[col] = o[i][d];
                }
                if (tx == 0) {
                    part_ml[(slot * TP_ROWS + row) * 2] = m[i];
                    part_ml[(slot * TP_ROWS + row) * 2 + 1] = sum;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------- the join
// Block (j, y): the item that the boundary between workers j and j + 1 is the first to cut, eight of its rows, a warp a
// row. Its parts are worker j's second slot and the following workers' first ones.
#define TJ_WARPS 8
template <typename T>
__global__ void __launch_bounds__(TJ_WARPS * 32) tree_join_kernel(T* __restrict__ out, long long out_stride, int dh, const TreeWork w,
                                                                  const float* __restrict__ part_o, const float* __restrict__ part_ml) {
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, j = blockIdx.x;
    const long long total = tree_total(w);
    const int workers = total > 0 ? tree_workers(w, total) : 0;
    if (j + 1 >= workers) return;
    const long long u = tree_begin(total, workers, j + 1);
    long long first;
    const int b = tree_find(w, u, first);
    if (b >= w.B) return;
    const TreeRequest r = tree_request(w, b);
    const int item_units = r.tiles + TREE_OVERHEAD;
    const int item = (int)((u - first) / item_units);
    const long long s = first + (long long)item * item_units;
    if (u - s <= TREE_OVERHEAD) return;                                       // between items
    if (tree_begin(total, workers, j) - s > TREE_OVERHEAD) return;            // cut before
    int parts = 2;
    while (tree_begin(total, workers, j + parts) < s + item_units) ++parts;
    const int G = w.H / w.Hkv, kvh = item / r.row_tiles, row_tile = item % r.row_tiles;
    const int per_tile = w.tokens_per_tile ? w.tokens_per_tile * G : w.rows_per_tile;
    const int row0 = row_tile * per_tile, n_rows = min(r.n * G - row0, per_tile);
    const int row = blockIdx.y * TJ_WARPS + warp, f = row0 + row;
    if (row >= n_rows) return;
    auto at = [&](int p) { return (size_t)(p == 0 ? 2 * j + 1 : 2 * (j + p)) * w.rows_per_tile + row; };
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 32) m = fmaxf(m, part_ml[at(p) * 2]);
    m = warp_max(m);
    float sum = 0.f, o[8] = {};
    const float ref = m == -INFINITY ? 0.f : m;
    for (int p0 = 0; p0 < parts; p0 += 32) {
        float weight = 0.f, l = 0.f;
        if (p0 + lane < parts) {
            weight = exp2f(part_ml[at(p0 + lane) * 2] - ref);
            l = part_ml[at(p0 + lane) * 2 + 1];
        }
        sum += weight * l;
        const int n = min(32, parts - p0);
#pragma unroll 4
        for (int p = 0; p < n; ++p) {
            const float f_p = __shfl_sync(0xffffffffu, weight, p);
            const float* src = part_o + at(p0 + p) * dh;
#pragma unroll
            for (int d = 0; d < 8; ++d)
                if (lane + 32 * d < dh) o[d] = fmaf(f_p, src[lane + 32 * d], o[d]);
        }
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* dst = out + (size_t)(r.tok0 + f / G) * out_stride + (size_t)(kvh * G + f % G) * dh;
#pragma unroll
    for (int d = 0; d < 8; ++d)
        if (lane + 32 * d < dh) dst[lane + 32 * d] = from_f32<T>(o[d] * inv);
}

// ------------------------------------------------------------------------------------ host
// Floats of workspace that a call wants.
TGO_API int tgo_attention_tree_work(int dtype, int dh) {
    return 2 * tgo_multiprocessors() * 2 * TP_ROWS * (dh + 2);
}

template <typename T, int DP>
static int tree_plain_go(const void* q, long long q_stride, void* out, long long out_stride, const void* k, const void* v,
                         int n_pages, int page_size, const int* tables, int max_blocks, const void* seen, int dh, float scale,
                         const TreeWork& w, float* part_o, float* part_ml, cudaStream_t stream) {
    constexpr size_t smem = (size_t)((TP_ROWS + 2 * TP_KEYS) * (DP + 4) + TP_ROWS * (TP_KEYS + 4)) * sizeof(float);
    static bool set[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(tree_plain_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        set[dev] = true;
    }
    int rc = tgo_launch_pdl(tree_plain_kernel<T, DP>, dim3(w.workers), dim3(TP_THREADS), smem, stream, (const T*)q, q_stride, (T*)out,
                            out_stride, (const T*)k, (const T*)v, n_pages, page_size, tables, max_blocks,
                            (const unsigned long long*)seen, dh, scale, w, part_o, part_ml);
    if (rc) return rc;
    if (w.workers == 1) return 0;
    return tgo_launch_pdl(tree_join_kernel<T>, dim3(w.workers - 1, (w.rows_per_tile + TJ_WARPS - 1) / TJ_WARPS), dim3(TJ_WARPS * 32), 0,
                          stream, (T*)out, out_stride, dh, w, (const float*)part_o, (const float*)part_ml);
}

// work: tgo_attention_tree_work() floats.
TGO_API int tgo_attention_tree(const void* q, long long q_stride, void* out, long long out_stride, int dtype, const void* k_cache,
                               const void* v_cache, int n_pages, int page_size, const int* block_tables, int max_blocks,
                               const int* context_lens, const int* q_start, const void* seen, int B, int H, int Hkv, int dh,
                               int window, float* work, cudaStream_t stream, float scale) {
    if (B <= 0) return 0;
    if (H <= 0 || Hkv <= 0 || H % Hkv || dh <= 0 || dh > 256 || n_pages <= 0 || page_size <= 0 || max_blocks <= 0 || window < 0 ||
        (long long)max_blocks * page_size > 0x7fffff00ll || (dtype != TGO_F32 && dtype != TGO_BF16))
        return TGO_E_BAD_ARG;
    TreeWork w = {context_lens, q_start, B, H, Hkv, window, max_blocks * page_size, TP_ROWS, 0, TP_KEYS, 2, 2 * tgo_multiprocessors()};
    float* part_ml = work + (size_t)w.workers * 2 * TP_ROWS * dh;
#define TP_GO(T, DP) return tree_plain_go<T, DP>(q, q_stride, out, out_stride, k_cache, v_cache, n_pages, page_size, block_tables, \
                                                 max_blocks, seen, dh, scale, w, work, part_ml, stream)
    if (dtype == TGO_F32) { if (dh <= 64) TP_GO(float, 64); if (dh <= 128) TP_GO(float, 128); TP_GO(float, 256); }
    if (dh <= 64) TP_GO(bf16, 64);
    if (dh <= 128) TP_GO(bf16, 128);
    TP_GO(bf16, 256);
#undef TP_GO
}
