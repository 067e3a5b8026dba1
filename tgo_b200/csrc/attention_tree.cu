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
#include <mutex>
#include <unordered_map>

#include "tcgen.cuh"

#define TREE_NODES 64
#define TREE_OVERHEAD 1

struct TreeWork {
    const int *context_lens, *q_start;
    int B, T, H, Hkv, window, max_nodes, max_keys;      // max_keys: what a block table can name
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
    r.n = min(min(max(w.q_start[b + 1] - r.tok0, 0), w.max_nodes), r.tok0 < 0 ? 0 : max(w.T - r.tok0, 0));
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

// -------------------------------------------------------------------------- tensor cores
// bfloat16, heads of 64 or 128, pages of 8 to 128 places: tcgen05. A tile is 128 query rows (128 / G whole nodes, row r =
// node r / G, head r % G; rows that a short tree leaves empty cost their warps nothing) and 128 keys. One CTA an SM walks its
// pieces with everything double-buffered: tensor memory holds S0, S1 (P lies over S) and O0, O1, shared memory two Q, two K
// and two V tiles.
//   warp 0        walks, asks TMA for an item's Q rows and publishes a record of the item in a ring of four;
//   warps 12, 10  follow the records and ask TMA for the K and for the V pages;
//   warps 1, 11   issue S = Q K^T and O += P V, a thread each;
//   warps 2-9     softmax, two threads a row, a half of the tile's keys each.
// The running maximum moves only when a row has outgrown it by 2^8: then the rows of O are rescaled. P is rounded to
// bfloat16, at most 2^-8 of a weight, as the storage's own rounding is; its sum is not.
// Rows of V that nobody sees are zeroed before the product, the cache may hold anything there. Where only some rows see
// a key (the nodes, and the cached keys at the windows' edges), a value that is no finite number is zeroed too, and its
// key noted: at the item's end the rows that see it get it added (rows are read from the cache again then).
// Waits have a limit of about two seconds, after which a code is left, what is under way is waited for, and the CTA ends.
#define TT_ROWS 128
#define TT_KEYS 128
#define TT_THREADS 416
#define TT_BLOCK (128 * 64 * 2)               // 128 rows x 64 columns of bfloat16
#define TT_TILE (2 * TT_BLOCK)
#define TT_PAGES 1024                         // pages of a piece whose numbers are kept in shared memory

__device__ int tree_error_flag = 0;

struct TreeItem {
    int valid;                                // 0: no more
    int tok0, n_rows, kvh, seq;               // its tile's first token
    int first_token;                          // its request's
    int key_tile, n_it;                       // key tiles from .. on, 0: zeros out
    int base, n, lo, hi;                      // of the request; keys lo .. hi - 1 are somebody's
    int whole, slot;                          // the item's result, or a part of it
    int pad[2];
};

// Both warps of a quarter of the rows; everyone gets the OR.
__device__ __forceinline__ bool tt_both(int quarter, bool pred) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
                 "bar.red.or.pred q, %2, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)pred), "r"(quarter + 1) : "memory");
    return r != 0;
}
__device__ __forceinline__ float tt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tt_load_3d(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(tg_smem(dst)), "l"(map), "r"(tg_smem(bar)), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// bits lo .. hi - 1
__device__ __forceinline__ unsigned long long tt_range(int lo, int hi) {
    lo = max(lo, 0);
    hi = min(hi, 64);
    if (hi <= lo) return 0ull;
    return (hi == 64 ? ~0ull : (1ull << hi) - 1ull) & ~((1ull << lo) - 1ull);
}
__device__ __forceinline__ unsigned long long tt_shift(unsigned long long x, int left) {
    return left >= 64 || left <= -64 ? 0ull : left >= 0 ? x << left : x >> -left;
}
// Two bfloat16 numbers, zero for one that is not finite.
__device__ __forceinline__ uint32_t tt_finite(uint32_t x) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
    return x;
}

template <int DH>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_tc_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
    const bf16* __restrict__ v_cache, int n_pages, bf16* __restrict__ out, long long out_stride, int page_size, int page_shift,
    const int* __restrict__ block_tables, int max_blocks, const unsigned long long* __restrict__ seen, float scale_log2,
    const TreeWork w, float* __restrict__ part_o, float* __restrict__ part_ml) {
    constexpr int NH = DH / 64, OC = DH / 2;
    extern __shared__ unsigned char tt_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)tt_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;                                   // [2][2 column halves][128 rows][128 bytes]
    unsigned char* sK = sQ + 2 * TT_TILE;
    unsigned char* sV = sK + 2 * TT_TILE;
    uint64_t* bars = (uint64_t*)(sV + 2 * TT_TILE);
    uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = bars + 6, *v_full = bars + 8, *v_empty = bars + 10,
             *s_full = bars + 12, *p_full = bars + 14, *o_free = bars + 16, *p_free = bars + 18, *o_done = bars + 20, *settled = bars + 21;
    unsigned long long* odd_nodes = (unsigned long long*)(bars + 23);       // [4 items]: nodes, and keys lo + i, whose values
    unsigned long long* odd_edge = odd_nodes + 4;                           // are not all finite
    uint32_t* tmem_slot = (uint32_t*)(bars + 31);
    TreeItem* ring = (TreeItem*)(bars + 32);                    // [4]
    float* s_m = (float*)(ring + 4);                            // [2][2 halves][128 rows]
    float* s_l = s_m + 512;                                     // [2 halves][128 rows]
    int* s_pages_k = (int*)(s_l + 256);
    int* s_pages_v = s_pages_k + TT_PAGES;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = w.H / w.Hkv;
    const int pages_per_tile = TT_KEYS >> page_shift;
    int* const err = &tree_error_flag;
    // rows of the Q tiles that no box writes must not hold NaN by chance
    for (int i = tid; i < 2 * TT_TILE / 16; i += TT_THREADS) ((uint4*)sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid < 8) odd_nodes[tid] = 0;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            tg_init(&q_full[i], 1); tg_init(&q_empty[i], 12);
            tg_init(&k_full[i], 1); tg_init(&k_empty[i], 1);
            tg_init(&v_full[i], 1); tg_init(&v_empty[i], 1);
            tg_init(&s_full[i], 1); tg_init(&p_full[i], 8);
            tg_init(&o_free[i], 8); tg_init(&p_free[i], 1);
            tg_init(&settled[i], 1);
        }
        tg_init(o_done, 1);
    }
    tg_init_done();
    if (warp == 1) tg_alloc512(tmem_slot);
    tg_before();
    __syncthreads();
    tg_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    if (warp == 0) {
        // ------------------------------------------------------------- pieces and Q
        const long long total = tree_total(w);
        const int workers = total > 0 ? tree_workers(w, total) : 0;
        TreeWalk walk;
        bool more = (int)blockIdx.x < workers;
        if (more) walk = tree_walk(w, total, workers, blockIdx.x);
        const int box_rows = w.tokens_per_tile * G;
        for (uint32_t n = 0;; ++n) {
            TreeItem* rec = &ring[n & 3];
            const uint32_t qb = n & 1u, qph = (n >> 1) & 1u;
            if (more) more = walk.next(w);
            if (!__all_sync(0xffffffffu, tg_wait(&q_empty[qb], qph ^ 1u, err, 1))) {
                tg_settle_copies(q_full, 2, n, err, 1);
                break;
            }
            if (!more) {
                if (lane == 0) { rec->valid = 0; tg_arrive(&q_full[qb]); }
                break;
            }
            if (lane == 0) {
                const TreeRequest& r = walk.r;
                const int token = walk.row_tile * w.tokens_per_tile;
                rec->valid = 1;
                rec->tok0 = r.tok0 + token;
                rec->n_rows = min(r.n - token, w.tokens_per_tile) * G;
                rec->kvh = walk.kvh; rec->seq = walk.b; rec->first_token = r.tok0;
                rec->key_tile = r.t_lo + walk.from;
                rec->base = r.base; rec->n = r.n;
                rec->hi = min(r.len, w.max_keys);
                rec->lo = w.window > 0 && r.base > w.window ? r.base - w.window : 0;
                rec->n_it = r.base < 0 || rec->hi <= rec->lo ? 0 : walk.to - walk.from;
                rec->whole = walk.from == 0 && walk.to == r.tiles;
                rec->slot = (int)blockIdx.x * 2 + (walk.from == 0 ? 1 : 0);
                if (rec->n_it > 0) {
                    // the G heads of a full tile's tokens: tokens behind this tile's are others' rows, whose results are
                    // not stored, tokens behind the last zeros
                    unsigned char* dq = sQ + qb * TT_TILE;
                    tg_expect(&q_full[qb], (uint32_t)(NH * box_rows) * 128u);
                    tt_load_3d(dq, &map_q, 0, walk.kvh * G, rec->tok0, &q_full[qb]);
                    if (NH > 1) tt_load_3d(dq + TT_BLOCK, &map_q, 64, walk.kvh * G, rec->tok0, &q_full[qb]);
                } else {
                    tg_arrive(&q_full[qb]);
                }
            }
            __syncwarp();
        }
    } else if (warp == 10 || warp == 12) {
        // ------------------------------------------------------------- V (warp 10), K (warp 12)
        const bool is_k = warp == 12;
        int* s_pages = is_k ? s_pages_k : s_pages_v;
        unsigned char* tiles = is_k ? sK : sV;
        uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
        const CUtensorMap* map = is_k ? &map_k : &map_v;
        bool ok = true;
        uint32_t g = 0;
        for (uint32_t n = 0; ok; ++n) {
            const uint32_t qb = n & 1u;
            ok = __all_sync(0xffffffffu, tg_wait(&q_full[qb], (n >> 1) & 1u, err, 1));
            if (!ok) break;
            const TreeItem rec = ring[n & 3];
            if (!rec.valid) break;
            __syncwarp();
            if (lane == 0) tg_arrive(&q_empty[qb]);
            const int* bt = block_tables + (size_t)rec.seq * max_blocks;
            const int pg_lo = rec.key_tile * pages_per_tile;
            const int pg_hi = min(min(pg_lo + rec.n_it * pages_per_tile, max_blocks), pg_lo + TT_PAGES);
            for (int i = pg_lo + lane; i < pg_hi; i += 32) s_pages[i - pg_lo] = bt[i];
            __syncwarp();
            for (int it = 0; it < rec.n_it; ++it, ++g) {
                const uint32_t s = g & 1u, ph = (g >> 1) & 1u;
                // the tile's pages that hold a key of somebody's
                const int p0 = (rec.key_tile + it) * pages_per_tile;
                const int first = max(p0, rec.lo >> page_shift), last = min(p0 + pages_per_tile, ((rec.hi - 1) >> page_shift) + 1);
                ok = __all_sync(0xffffffffu, tg_wait(&empty[s], ph ^ 1u, err, 1));
                if (!ok) break;
                if (lane == 0) tg_expect(&full[s], (uint32_t)max(last - first, 0) * (uint32_t)page_size * (uint32_t)(DH * 2));
                __syncwarp();
                for (int pi = first + lane; pi < last; pi += 32) {
                    const int page = pi - pg_lo < TT_PAGES ? s_pages[pi - pg_lo] : bt[pi];
                    // a number that names no page reads zeros: rows behind the last
                    const int row = page >= 0 && page < n_pages ? (page * w.Hkv + rec.kvh) * page_size : n_pages * w.Hkv * page_size;
                    unsigned char* dst = tiles + s * TT_TILE + (pi - p0) * page_size * 128;
                    tg_load_2d(dst, map, 0, row, &full[s]);
                    if (NH > 1) tg_load_2d(dst + TT_BLOCK, map, 64, row, &full[s]);
                }
            }
            __syncwarp();
        }
        if (!ok) tg_settle_copies(full, 2, g, err, 1);
    } else if (warp == 1) {
        // ------------------------------------------------------------- S = Q K^T
        if (lane == 0) {
            const uint32_t idesc = tg_idesc(128);
            uint32_t g = 0;
            bool ok = true;
            for (uint32_t n = 0; ok; ++n) {
                const uint32_t qb = n & 1u;
                ok = tg_wait(&q_full[qb], (n >> 1) & 1u, err, 2);
                if (!ok) break;
                const TreeItem* rec = &ring[n & 3];
                if (!rec->valid) break;
                const int n_it = rec->n_it;
                const unsigned char* qt = sQ + qb * TT_TILE;
                const uint64_t dq0 = tg_desc(qt), dq1 = tg_desc(qt + TT_BLOCK);
                for (int it = 0; it < n_it; ++it, ++g) {
                    const uint32_t s = g & 1u, ph = (g >> 1) & 1u;
                    ok = tg_wait(&k_full[s], ph, err, 2) && tg_wait(&p_free[s], ph ^ 1u, err, 2);
                    if (!ok) break;
                    tg_after();
                    const uint64_t dk0 = tg_desc(sK + s * TT_TILE), dk1 = tg_desc(sK + s * TT_TILE + TT_BLOCK);
#pragma unroll
                    for (int k = 0; k < 4; ++k) tg_mma(tmem + 128u * s, dq0 + 2 * k, dk0 + 2 * k, idesc, k > 0 ? 1u : 0u);
                    if (NH > 1)
#pragma unroll
                        for (int k = 0; k < 4; ++k) tg_mma(tmem + 128u * s, dq1 + 2 * k, dk1 + 2 * k, idesc, 1u);
                    tg_commit(&k_empty[s]);
                    tg_commit(&s_full[s]);
                }
                tg_commit(&q_empty[qb]);
            }
            if (!ok) tg_settle_products(&settled[0], err, 2);
        }
    } else if (warp == 11) {
        // ------------------------------------------------------------- O += P V
        if (lane == 0) {
            const uint32_t idesc = tg_idesc(DH, true);
            uint32_t g = 0;
            bool ok = true;
            for (uint32_t n = 0; ok; ++n) {
                ok = tg_wait(&q_full[n & 1u], (n >> 1) & 1u, err, 2);
                if (!ok) break;
                const TreeItem* rec = &ring[n & 3];
                if (!rec->valid) break;
                const int n_it = rec->n_it;
                tg_arrive(&q_empty[n & 1u]);
                const uint32_t ob = n & 1u, tm_o = tmem + 256u + 128u * ob;
                for (int it = 0; it < n_it && ok; ++it, ++g) {
                    const uint32_t s = g & 1u, ph = (g >> 1) & 1u;
                    if (it == 0) ok = tg_wait(&o_free[ob], ((n >> 1) & 1u) ^ 1u, err, 2);
                    ok = ok && tg_wait(&p_full[s], ph, err, 2) && tg_wait(&v_full[s], ph, err, 2);
                    if (!ok) break;
                    tg_after();
                    const uint64_t dv = NH > 1 ? tg_desc_mn(sV + s * TT_TILE, TT_BLOCK) : tg_desc(sV + s * TT_TILE);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        tg_mma_ts(tm_o, tmem + 128u * s + 8u * k, dv + (uint64_t)(128 * k), idesc, (it > 0 || k > 0) ? 1u : 0u);
                    tg_commit(&v_empty[s]);
                    tg_commit(&p_free[s]);
                    tg_commit(o_done);
                }
            }
            if (!ok) tg_settle_products(&settled[1], err, 2);
        }
    } else {
        // ------------------------------------------------------------- softmax
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        bool ok = true;
        uint32_t g = 0, walked = 0;                             // key tiles, items with any
        for (uint32_t n = 0;; ++n) {
            if (ok) ok = tg_wait(&q_full[n & 1u], (n >> 1) & 1u, err, 3);
            if (tt_both(quarter, !ok)) break;                   // both warps of the rows leave together
            const TreeItem rec = ring[n & 3];
            if (!rec.valid) break;
            __syncwarp();
            if (lane == 0) tg_arrive(&q_empty[n & 1u]);
            const uint32_t ob = n & 1u, tm_o = tmem + 256u + 128u * ob;
            const bool row_ok = row < rec.n_rows;
            const bool live = quarter * 32 < rec.n_rows;        // a row of the warp's is somebody's
            const int token = (row_ok ? row : 0) / G, head = rec.kvh * G + (row_ok ? row : 0) % G;
            bf16* dst = out + (size_t)(rec.tok0 + token) * out_stride + (size_t)head * DH + OC * half;
            if (rec.n_it == 0) {
                if (row_ok)
#pragma unroll
                    for (int i = 0; i < OC / 8; ++i) *(uint4*)(dst + i * 8) = make_uint4(0u, 0u, 0u, 0u);
                __syncwarp();
                if (lane == 0) tg_arrive(&o_free[ob]);
                continue;
            }
            unsigned long long bits = 0;
            int lo = 0x7fffffff;
            if (row_ok) {
                bits = seen[rec.tok0 + token] & (rec.n >= 64 ? ~0ull : (1ull << rec.n) - 1ull);
                lo = w.window > 0 ? max(rec.base + __popcll(bits) - w.window, 0) : 0;
            }
            const bool warp_rows_ok = quarter * 32 + 31 < rec.n_rows;
            // keys whole_lo .. base - 1 are seen by every row
            const int whole_lo = w.window > 0 ? rec.base + rec.n - w.window : 0;
            float m_used = -INFINITY, l = 0.f;
            bool left = false;                                  // decided at a barrier: the same for both warps
            for (int it = 0; it < rec.n_it; ++it, ++g) {
                const uint32_t s = g & 1u, ph = (g >> 1) & 1u;
                const uint32_t tm_s = tmem + 128u * s;
                const int tile_lo = (rec.key_tile + it) * TT_KEYS, kbase = tile_lo + 64 * half;
                float corr = 1.f;
                bool rescale = false;
                if (live) {
                    if (ok) ok = tg_wait(&s_full[s], ph, err, 3);
                    tg_after();
                    float sc[64];
                    {
                        uint32_t r0[32], r1[32];
                        tg_ld32(tm_s + lane_base + 64u * half, r0);
                        tg_ld32(tm_s + lane_base + 64u * half + 32u, r1);
                        tg_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) { sc[i] = __uint_as_float(r0[i]); sc[32 + i] = __uint_as_float(r1[i]); }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (!(warp_rows_ok && kbase + 64 <= rec.base && kbase >= whole_lo && kbase + 64 <= rec.hi)) {
                        const unsigned long long see = (tt_range(lo - kbase, rec.base - kbase) | tt_shift(bits, rec.base - kbase)) &
                                                       tt_range(0, rec.hi - kbase);
                        const uint32_t see0 = (uint32_t)see, see1 = (uint32_t)(see >> 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sc[i] = see0 >> i & 1u ? sc[i] : -INFINITY;
                            sc[32 + i] = see1 >> i & 1u ? sc[32 + i] : -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 64; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], sc[i]);
                    float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
                    float* xm = s_m + (g & 1u) * 256;
                    xm[half * 128 + row] = mx;
                    // both halves have read their S (P is written over it)
                    if (tt_both(quarter, !ok)) { left = true; break; }
                    mx = fmaxf(mx, xm[(half ^ 1) * 128 + row]);
                    const float m_new = fmaxf(m_used, mx);
                    const bool grow = m_new > m_used + 8.f || (m_used == -INFINITY && m_new != -INFINITY);
                    rescale = __any_sync(0xffffffffu, grow);
                    if (rescale) {
                        corr = m_new == -INFINITY ? 1.f : exp2f(m_used - m_new);
                        m_used = m_new;
                    }
                    const float ref = m_used == -INFINITY ? 0.f : m_used;
                    float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t r[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float a = tt_exp2(fmaf(sc[2 * i], scale_log2, -ref));
                        const float b = tt_exp2(fmaf(sc[2 * i + 1], scale_log2, -ref));
                        sum4[i & 3] += a + b;
                        r[i] = tg_pack(a, b);
                    }
                    tg_st32(tm_s + lane_base + 32u * half, r);
                    l = l * corr + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
                }
                if (tile_lo + TT_KEYS > min(rec.base, rec.hi) || (w.window > 0 && tile_lo < rec.lo + 64)) {
                    // places that nobody sees, and values that are no numbers where only some rows see them
                    if (ok) ok = tg_wait(&v_full[s], ph, err, 3);
                    const int key = tile_lo + row;
                    unsigned char* vrow = sV + s * TT_TILE + row * 128 + (NH > 1 ? half * TT_BLOCK : half * 64);
                    const bool nobody = key >= rec.hi || key < rec.lo;
                    if (nobody || key >= rec.base || key < whole_lo) {
#pragma unroll
                        for (int c = 0; c < 4 * NH; ++c) {
                            uint4* at = (uint4*)(vrow + c * 16);
                            uint4 v = make_uint4(0u, 0u, 0u, 0u);
                            if (!nobody) {
                                const uint4 u = *at;
                                v = make_uint4(tt_finite(u.x), tt_finite(u.y), tt_finite(u.z), tt_finite(u.w));
                                if (v.x == u.x && v.y == u.y && v.z == u.z && v.w == u.w) continue;
                                if (key >= rec.base) atomicOr(&odd_nodes[walked & 3u], 1ull << (key - rec.base));
                                else atomicOr(&odd_edge[walked & 3u], 1ull << (key - rec.lo));
                            }
                            *at = v;
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (live) {
                    if (it > 0) {
                        if (ok) ok = tg_wait(o_done, (g - 1u) & 1u, err, 3);
                        tg_after();
                        if (rescale) {
                            uint32_t r[32];
#pragma unroll
                            for (int c = 0; c < NH; ++c) {
                                tg_ld32(tm_o + lane_base + (uint32_t)(OC * half) + 32u * c, r);
                                tg_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
                                tg_st32(tm_o + lane_base + (uint32_t)(OC * half) + 32u * c, r);
                            }
                        }
                    }
                    tg_wait_st();
                    tg_before();
                } else if (it > 0) {
                    // not a phase further than the others: an arrival for this tile may not run into the last one's
                    if (ok) ok = tg_wait(o_done, (g - 1u) & 1u, err, 3);
                }
                const bool warp_ok = __all_sync(0xffffffffu, ok);
                if (lane == 0 && warp_ok) tg_arrive(&p_full[s]);
                if (!live && tt_both(quarter, !warp_ok)) { left = true; break; }
            }
            if (left) break;
            if (ok) ok = tg_wait(o_done, (g - 1u) & 1u, err, 3);
            tg_after();
            s_l[half * 128 + row] = l;
            if (tt_both(quarter, !ok)) break;
            l += s_l[(half ^ 1) * 128 + row];
            const unsigned long long nodes = odd_nodes[walked & 3u] & bits;
            const unsigned long long edge = odd_edge[walked & 3u] & tt_range(lo - rec.lo, rec.base - rec.lo);
            // for the item after the next: nobody is past that one, which wants this thread's arrivals, or before this one
            if (tid == 64) odd_nodes[(walked + 2u) & 3u] = odd_edge[(walked + 2u) & 3u] = 0;
            ++walked;
            if (live) {
                const float factor = rec.whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                const size_t at = (size_t)rec.slot * w.rows_per_tile + row;
                if (!rec.whole && row_ok && half == 0) {
                    part_ml[at * 2] = m_used;
                    part_ml[at * 2 + 1] = l;
                }
#pragma unroll
                for (int c = 0; c < NH; ++c) {
                    uint32_t r[32];
                    tg_ld32(tm_o + lane_base + (uint32_t)(OC * half) + 32u * c, r);
                    tg_wait_ld();
                    if (row_ok) {
                        float o[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(r[i]) * factor;
                        if (nodes | edge) {
                            for (int k = 0; k < 128; ++k) {
                                if (!((k < 64 ? nodes >> k : edge >> (k - 64)) & 1ull)) continue;
                                const int key = k < 64 ? rec.base + k : rec.lo + k - 64;
                                const int page = block_tables[(size_t)rec.seq * max_blocks + (key >> page_shift)];
                                const bf16* v = v_cache + (((size_t)page * w.Hkv + rec.kvh) * page_size + (key & (page_size - 1))) * DH +
                                                OC * half + 32 * c;
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float x = __bfloat162float(v[i]);
                                    if (!isfinite(x)) o[i] += x;
                                }
                            }
                        }
                        if (rec.whole) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                *(uint4*)(dst + c * 32 + i * 8) = make_uint4(tg_pack(o[8 * i], o[8 * i + 1]), tg_pack(o[8 * i + 2], o[8 * i + 3]),
                                                                             tg_pack(o[8 * i + 4], o[8 * i + 5]), tg_pack(o[8 * i + 6], o[8 * i + 7]));
                        } else {
                            float* po = part_o + at * DH + OC * half + 32 * c;
#pragma unroll
                            for (int i = 0; i < 8; ++i) *(float4*)(po + i * 4) = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }
                }
            }
            tg_before();
            __syncwarp();
            if (lane == 0) tg_arrive(&o_free[ob]);
        }
    }
    tg_before();
    __syncthreads();
    if (warp == 1) {
        tg_after();
        tg_free512(tmem);
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
// Whether the tensor cores' kernel takes calls of this layout (in bfloat16).
TGO_API int tgo_attention_tree_tc_supports(int dh, int group, int page_size) {
    return (dh == 64 || dh == 128) && group >= 1 && group <= TT_ROWS && page_size >= 8 && page_size <= TT_KEYS &&
           (page_size & (page_size - 1)) == 0;
}
// The code that a wait of that kernel left when it ran out (1 copies, 2 products, 3 softmax), or 0. Synchronises.
TGO_API int tgo_attention_tree_error(int* value) { return (int)cudaMemcpyFromSymbol(value, tree_error_flag, sizeof(int)); }

static int tree_force = 0;                    // for tests: 1 plain products, 2 tensor cores where they take the call
TGO_API int tgo_attention_tree_force(int way) { tree_force = way; return 0; }

// Floats of workspace that a call wants.
TGO_API int tgo_attention_tree_work(int dtype, int dh, int group, int page_size, int max_nodes) {
    const int sms = tgo_multiprocessors();
    int rows = 2 * TP_ROWS;
    if (dtype == TGO_BF16 && tgo_attention_tree_tc_supports(dh, group, page_size)) {
        const int mine = max_nodes * group < TT_ROWS ? max_nodes * group : TT_ROWS;
        rows = mine > rows ? mine : rows;
    }
    return sms * 2 * rows * (dh + 2);
}

// The tensor map of a layer's K or V pages, kept by address, rows, page size and width.
static const CUtensorMap* tree_map_kv(const void* pages, long long rows, int page_size, int dh) {
    struct Key {
        const void* pages; long long rows; int page_size, dh;
        bool operator==(const Key& o) const { return pages == o.pages && rows == o.rows && page_size == o.page_size && dh == o.dh; }
    };
    struct Hash {
        size_t operator()(const Key& k) const {
            return (size_t)(uintptr_t)k.pages ^ ((size_t)k.rows * 0x9e3779b97f4a7c15ull) ^ ((size_t)k.page_size << 56) ^ ((size_t)k.dh << 48);
        }
    };
    static std::mutex lock;
    static std::unordered_map<Key, CUtensorMap, Hash> maps;
    std::lock_guard<std::mutex> hold(lock);
    const Key key{pages, rows, page_size, dh};
    auto it = maps.find(key);
    if (it != maps.end()) return &it->second;
    CUtensorMap map;
    if (!tg_map(&map, pages, rows, dh, dh, page_size)) return nullptr;
    return &maps.emplace(key, map).first->second;
}
// ... of query rows [tokens][heads][dh], `stride` apart, in boxes of 64 columns of G heads of box_tokens tokens.
static const CUtensorMap* tree_map_q(const void* q, long long stride, int tokens, int H, int G, int dh) {
    struct Key {
        const void* q; long long stride; int tokens, H, G, dh;
        bool operator==(const Key& o) const {
            return q == o.q && stride == o.stride && tokens == o.tokens && H == o.H && G == o.G && dh == o.dh;
        }
    };
    struct Hash {
        size_t operator()(const Key& k) const {
            return (size_t)(uintptr_t)k.q * 0x9e3779b97f4a7c15ull ^ ((size_t)k.stride << 32) ^ ((size_t)k.tokens << 12) ^
                   ((size_t)k.H << 6) ^ (size_t)k.G ^ ((size_t)k.dh << 56);
        }
    };
    static std::mutex lock;
    static std::unordered_map<Key, CUtensorMap, Hash> maps;
    std::lock_guard<std::mutex> hold(lock);
    const Key key{q, stride, tokens, H, G, dh};
    auto it = maps.find(key);
    if (it != maps.end()) return &it->second;
    const TgEncodeFn encode = tg_encode();
    if (!encode) return nullptr;
    CUtensorMap map;
    const cuuint64_t dims[3] = {(cuuint64_t)dh, (cuuint64_t)H, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)dh * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(TT_ROWS / G)};
    const cuuint32_t elem[3] = {1, 1, 1};
    if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return nullptr;
    if (maps.size() > 4096) maps.clear();
    return &maps.emplace(key, map).first->second;
}

template <typename T>
static int tree_join_go(void* out, long long out_stride, int dh, const TreeWork& w, const float* part_o, const float* part_ml,
                        cudaStream_t stream) {
    if (w.workers == 1) return 0;
    return tgo_launch_pdl(tree_join_kernel<T>, dim3(w.workers - 1, (w.rows_per_tile + TJ_WARPS - 1) / TJ_WARPS), dim3(TJ_WARPS * 32), 0,
                          stream, (T*)out, out_stride, dh, w, part_o, part_ml);
}

template <int DH>
static int tree_tc_go(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const void* v, int n_pages, void* out,
                      long long out_stride, int page_size, const int* tables, int max_blocks, const void* seen, float scale,
                      const TreeWork& w, float* part_o, float* part_ml, cudaStream_t stream) {
    constexpr size_t smem = 1024 + 6 * (size_t)TT_TILE + 32 * 8 + 4 * sizeof(TreeItem) + 768 * sizeof(float) + 2 * TT_PAGES * sizeof(int);
    static bool set[64] = {};
    int dev = 0, shift = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(tree_tc_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        set[dev] = true;
    }
    while ((1 << shift) < page_size) ++shift;
    const int rc = tgo_launch_pdl(tree_tc_kernel<DH>, dim3(w.workers), dim3(TT_THREADS), smem, stream, mk, mv, mq, (const bf16*)v, n_pages,
                                  (bf16*)out, out_stride, page_size, shift, tables, max_blocks, (const unsigned long long*)seen,
                                  scale * TREE_LOG2E, w, part_o, part_ml);
    if (rc) return rc;
    return tree_join_go<bf16>(out, out_stride, DH, w, part_o, part_ml, stream);
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
    return tree_join_go<T>(out, out_stride, dh, w, part_o, part_ml, stream);
}

// work: tgo_attention_tree_work() floats. scale > 0.
TGO_API int tgo_attention_tree(const void* q, long long q_stride, void* out, long long out_stride, int dtype, int T, const void* k_cache,
                               const void* v_cache, int n_pages, int page_size, const int* block_tables, int max_blocks,
                               const int* context_lens, const int* q_start, const void* seen, int B, int H, int Hkv, int dh,
                               int window, int max_nodes, float* work, cudaStream_t stream, float scale) {
    if (B <= 0 || T <= 0 || max_nodes <= 0) return 0;
    if (H <= 0 || Hkv <= 0 || H % Hkv || dh <= 0 || dh > 256 || n_pages <= 0 || page_size <= 0 || max_blocks <= 0 || window < 0 ||
        max_nodes > TREE_NODES || (long long)max_blocks * page_size > 0x7fffff00ll || (dtype != TGO_F32 && dtype != TGO_BF16) || !(scale > 0.f))
        return TGO_E_BAD_ARG;
    const int sms = tgo_multiprocessors(), G = H / Hkv;
    const long long rows = (long long)n_pages * Hkv * page_size;
    TreeWork w = {context_lens, q_start, B, T, H, Hkv, window, max_nodes, max_blocks * page_size, 0, 0, 0, 2, 0};
    if (dtype == TGO_BF16 && tree_force != 1 && tgo_attention_tree_tc_supports(dh, G, page_size) && q_stride % 8 == 0 && out_stride % 8 == 0 &&
        (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)k_cache % 128 == 0 && (uintptr_t)v_cache % 128 == 0 &&
        rows + page_size <= 0x7fffffffll) {
        w.tokens_per_tile = TT_ROWS / G;
        w.rows_per_tile = max_nodes * G < TT_ROWS ? max_nodes * G : TT_ROWS;      // of a part
        w.key_tile = TT_KEYS;
        w.workers = sms;
        const CUtensorMap* mk = tree_map_kv(k_cache, rows, page_size, dh);
        const CUtensorMap* mv = tree_map_kv(v_cache, rows, page_size, dh);
        const CUtensorMap* mq = tree_map_q(q, q_stride, T, H, G, dh);
        if (!mk || !mv || !mq) return TGO_E_BAD_ARG;
        float* part_ml = work + (size_t)w.workers * 2 * w.rows_per_tile * dh;
        if (dh == 128) return tree_tc_go<128>(*mk, *mv, *mq, v_cache, n_pages, out, out_stride, page_size, block_tables, max_blocks, seen, scale, w, work, part_ml, stream);
        return tree_tc_go<64>(*mk, *mv, *mq, v_cache, n_pages, out, out_stride, page_size, block_tables, max_blocks, seen, scale, w, work, part_ml, stream);
    }
    w.rows_per_tile = TP_ROWS;
    w.key_tile = TP_KEYS;
    w.workers = 2 * sms;
    float* part_ml = work + (size_t)w.workers * 2 * TP_ROWS * dh;
#define TP_GO(T, DP) return tree_plain_go<T, DP>(q, q_stride, out, out_stride, k_cache, v_cache, n_pages, page_size, block_tables, \
                                                 max_blocks, seen, dh, scale, w, work, part_ml, stream)
    if (dtype == TGO_F32) { if (dh <= 64) TP_GO(float, 64); if (dh <= 128) TP_GO(float, 128); TP_GO(float, 256); }
    if (dh <= 64) TP_GO(bf16, 64);
    if (dh <= 128) TP_GO(bf16, 128);
    TP_GO(bf16, 256);
#undef TP_GO
}
