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

#include "tcgen.cuh"

#define TREE_NODES 64
#define TREE_E_WORK 1001                      // returned, nothing done: the call wants a workspace
#define TREE_OVERHEAD 1

struct TreeWork {
    const int *context_lens, *q_start;
    int B, T, H, Hkv, window, max_nodes, max_keys;      // max_keys: what a block table can name
    int rows_per_tile, tokens_per_tile;       // a tile holds so many rows, or (if not 0) so many whole tokens
    int min_units, workers;                   // of a piece at least, in all at most
    int whole;                                // items are not cut: each is a unit
};

struct TreeRequest {
    int tok0, n, base, len, t_lo, tiles, row_tiles;
    int units;                                // of all its items
};

// KT: keys of a tile.
template <int KT> __device__ __forceinline__ TreeRequest tree_request(const TreeWork& w, int b) {
    TreeRequest r;
    r.tok0 = w.q_start[b];
    r.n = min(min(max(w.q_start[b + 1] - r.tok0, 0), w.max_nodes), r.tok0 < 0 ? 0 : max(w.T - r.tok0, 0));
    r.len = w.context_lens[b];
    r.base = r.len - r.n;
    const bool none = r.base < 0;             // a padded request: its rows get zeros
    const int hi = none ? 0 : min(r.len, w.max_keys);
    const int lo = w.window > 0 && r.base - w.window > 0 ? r.base - w.window : 0;
    r.t_lo = none ? 0 : lo / KT;
    r.tiles = max((hi + KT - 1) / KT - r.t_lo, 1);
    r.row_tiles = w.tokens_per_tile ? (r.n + w.tokens_per_tile - 1) / w.tokens_per_tile
                                    : (r.n * (w.H / w.Hkv) + w.rows_per_tile - 1) / w.rows_per_tile;
    r.units = r.row_tiles * w.Hkv * (w.whole ? 1 : r.tiles + TREE_OVERHEAD);
    return r;
}

// How all units are cut: worker i begins at i * each + min(i, more).
struct TreeCut {
    int workers, each, more;
    __device__ __forceinline__ int begin(int i) const { return i * each + min(i, more); }
};

// A worker's walk over its pieces: `next` gives them one after the other.
template <int KT> struct TreeWalk {
    TreeCut cut;
    int u, end, first;                        // where it stands, where its piece ends, where request b begins
    int b;
    TreeRequest r;
    // of the piece
    int kvh, row_tile, from, to;              // key tiles from .. to - 1 of the item
    // Worker i's, by one warp; no pieces if there are fewer workers.
    __device__ __forceinline__ void find(const TreeWork& w, int i) {
        const int lane = threadIdx.x & 31;
        TreeRequest mine;
        mine.units = 0;
        if (lane < w.B) mine = tree_request<KT>(w, lane);
        auto scan = [&](int x) {                   // the sum of the lanes up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += other;
            }
            return x;
        };
        int upto = scan(mine.units);
        int total = __shfl_sync(0xffffffffu, upto, 31);
        if (w.B > 32) {
            int rest = 0;
            for (int c = lane + 32; c < w.B; c += 32) rest += tree_request<KT>(w, c).units;
            total += __shfl_sync(0xffffffffu, scan(rest), 31);
        }
        const int most = total / w.min_units;
        cut.workers = total == 0 ? 0 : most < 1 ? 1 : min(most, w.workers);
        u = end = first = b = 0;
        if (i >= cut.workers) return;
        cut.each = total / cut.workers;
        cut.more = total - cut.each * cut.workers;
        u = cut.begin(i);
        end = cut.begin(i + 1);
        int before = 0;
        for (int b0 = 0; b0 < w.B; b0 += 32) {
            if (b0) {
                mine.units = 0;
                if (b0 + lane < w.B) mine = tree_request<KT>(w, b0 + lane);
                upto = scan(mine.units);
            }
            const uint32_t in = __ballot_sync(0xffffffffu, u < before + upto);
            if (in) {
                const int l = __ffs(in) - 1;
                b = b0 + l;
                first = before + __shfl_sync(0xffffffffu, upto - mine.units, l);
                r.tok0 = __shfl_sync(0xffffffffu, mine.tok0, l);
                r.n = __shfl_sync(0xffffffffu, mine.n, l);
                r.base = __shfl_sync(0xffffffffu, mine.base, l);
                r.len = __shfl_sync(0xffffffffu, mine.len, l);
                r.t_lo = __shfl_sync(0xffffffffu, mine.t_lo, l);
                r.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
                r.row_tiles = __shfl_sync(0xffffffffu, mine.row_tiles, l);
                r.units = __shfl_sync(0xffffffffu, mine.units, l);
                return;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __device__ __forceinline__ bool next(const TreeWork& w) {
        while (u < end) {
            while (u >= first + r.units) {
                first += r.units;
                if (++b >= w.B) return false;
                r = tree_request<KT>(w, b);
            }
            const int item_units = w.whole ? 1 : r.tiles + TREE_OVERHEAD;
            const int item = w.whole ? u - first : (u - first) / item_units;
            const int s = first + item * item_units;
            from = max(u - s - TREE_OVERHEAD, 0);
            to = end - s >= item_units ? r.tiles : max(end - s - TREE_OVERHEAD, 0);
            kvh = r.row_tiles == 1 ? item : item / r.row_tiles;
            row_tile = item - kvh * r.row_tiles;
            u = s + item_units;
            if (to > from) return true;
        }
        return false;
    }
};

// What worker i leaves for the join about an item that it begins and does not end; n_rows is 0 where there is none.
struct TreeNote {
    int parts, n_rows, row0, tok0, kvh;       // workers with a part; rows row0 .. of the request that begins at token tok0
};
template <int KT> __device__ __forceinline__ TreeNote tree_note(const TreeWork& w, const TreeWalk<KT>& k, int i) {
    TreeNote t = {0, 0, 0, 0, 0};
    if (k.from > 0 || k.to == k.r.tiles) return t;
    t.parts = 2;
    while (k.cut.begin(i + t.parts) < k.u) ++t.parts;          // u is where the item ends
    const int G = w.H / w.Hkv, per_tile = w.tokens_per_tile ? w.tokens_per_tile * G : w.rows_per_tile;
    t.row0 = k.row_tile * per_tile;
    t.n_rows = min(k.r.n * G - t.row0, per_tile);
    t.tok0 = k.r.tok0;
    t.kvh = k.kvh;
    return t;
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
// float32, and bfloat16 where the tensor cores' kernel has no instance: 16, 32 or 64 rows (R = 1, 2, 4 a thread) and 64 keys a
// tile on the FMA units, sixteen threads R rows. A thread makes R x 4 scores, then R x (width / 16) outputs; rows lie in
// shared memory 4 floats further apart than they are wide, so that eight threads' 16-byte reads meet no bank twice. Four rows a
// thread read 12 times 128 bytes for 64 products of a warp and are bound by these, fewer by the reads. The next K is
// copied while this tile's weights and sums are made, the next V while its scores are.
// A masked score becomes the weight -0, which no exponential gives: in tiles that not every row sees whole and that hold an
// infinity or a NaN, such a weight is left out of the sum, so that what lies in a masked place does not reach it.
//   MEASURED, in a graph of calls: 3 requests of 12 nodes over up to 1513 keys, 16 heads over 4 of 128: 30.5 us with the join. A tile
// of 64 keys takes 13 thousand cycles, 8 at the FMA units' rate (64 rows, of which 48 are somebody's), most blocks have two
// and some none; a block is at its first product after 12 thousand cycles (its piece, pages, copies). Tiles of 32 keys
// and two blocks an SM took 36.0 us with 2 x 4 scores a thread and 34.6 with 8 x 4 by quarters of the width.
#define TP_KEYS 64
#define TP_THREADS 256

// Four numbers of the cache into shared memory, or zeros; bfloat16 by way of registers.
__device__ __forceinline__ void tp_copy4(float* dst, const float* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tg_smem(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void tp_copy4(float* dst, const bf16* src, bool there) {
    uint2 u = make_uint2(0u, 0u);
    if (there) u = *(const uint2*)src;
    *(float4*)dst = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                                __uint_as_float(u.y & 0xffff0000u));
}

// The same, or one by one where four do not lie together; `left` of them belong to the row.
template <typename T>
__device__ __forceinline__ void tp_row4(float* dst, const T* src, bool there, bool vectors, int left) {
    if (vectors) tp_copy4(dst, src, there);
    else
#pragma unroll 1
        for (int e = 0; e < 4; ++e) dst[e] = there && e < left ? to_f32(src[e]) : 0.f;
}

template <typename T, int DP, int R>
__global__ void __launch_bounds__(TP_THREADS) tree_plain_kernel(
    const T* __restrict__ q, long long q_stride, T* __restrict__ out, long long out_stride, const T* __restrict__ k_cache,
    const T* __restrict__ v_cache, int n_pages, int page_size, int page_shift, const int* __restrict__ block_tables, int max_blocks,
    const unsigned long long* __restrict__ seen, int dh, float scale, const TreeWork w, float* __restrict__ part_o,
    float* __restrict__ part_ml, TreeNote* __restrict__ notes) {
    constexpr int ROWS = 16 * R, LD = DP + 4, LS = TP_KEYS + 4, J = DP / 64;
    constexpr int FOURS = DP / 4, EACH = TP_THREADS / FOURS, PASSES = TP_KEYS / EACH;
    extern __shared__ __align__(16) float tp_smem[];
    float* sq = tp_smem;                          // [ROWS][LD]
    float* sk = sq + ROWS * LD;                   // [TP_KEYS][LD]
    float* sv = sk + TP_KEYS * LD;                // [TP_KEYS][LD]
    float* ss = sv + TP_KEYS * LD;                // [ROWS][LS]
    __shared__ TreeWalk<TP_KEYS> s_walk;
    pdl_wait();
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    if (tid < 32) {
        TreeWalk<TP_KEYS> k;
        k.find(w, blockIdx.x);
        if (tid == 0) {
            s_walk = k;
            if (!w.whole) notes[blockIdx.x].n_rows = 0;
        }
    }
    __syncthreads();
    TreeWalk<TP_KEYS> walk = s_walk;
    const int G = w.H / w.Hkv;
    // r / G: r < 64 G, and r G < 2^32
    const uint32_t by_g = G > 1 ? (uint32_t)((0x100000000ull + G - 1) / G) : 0;
    auto node_of = [&](int r) { return G > 1 ? (int)__umulhi((uint32_t)r, by_g) : r; };
    const float c = scale * TREE_LOG2E;
    const bool vectors = dh % 4 == 0 && ((uintptr_t)k_cache | (uintptr_t)v_cache) % (4 * sizeof(T)) == 0;
    const bool q_vectors = dh % 4 == 0 && q_stride % 4 == 0 && (uintptr_t)q % (4 * sizeof(T)) == 0;
    const int my_d = tid % FOURS * 4, my_row = tid / FOURS;
    while (walk.next(w)) {
        const TreeRequest r = walk.r;
        const int row0 = walk.row_tile * ROWS, n_rows = min(r.n * G - row0, ROWS);
        const int kvh = walk.kvh;
        const int hi = r.base < 0 ? 0 : min(r.len, w.max_keys);
        const int* bt = block_tables + (size_t)walk.b * max_blocks;
        // A tile of K or V, a thread the same four columns of every EACH-th row: where its rows lie, and their copies. 32-bit
        // numbers are copied past the registers.
        int page[PASSES], place[PASSES];
        auto look = [&](int t) {
            const int key0 = (r.t_lo + t) * TP_KEYS;
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const int key = key0 + my_row + i * EACH, nth = page_shift >= 0 ? key >> page_shift : key / page_size;
                place[i] = key - nth * page_size;
                page[i] = key < hi ? bt[nth] : -1;
            }
        };
        auto copy = [&](float* dst, const T* cache) {
#pragma unroll
            for (int i = 0; i < PASSES; ++i) {
                const bool there = page[i] >= 0 && page[i] < n_pages && my_d < dh;
                const T* at = cache + (there ? (((size_t)page[i] * w.Hkv + kvh) * page_size + place[i]) * dh + my_d : 0);
                tp_row4(dst + (my_row + i * EACH) * LD + my_d, at, there, vectors, dh - my_d);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncthreads();                          // the last piece's rows have been read
        look(walk.from);
        for (int row = my_row; row < ROWS; row += EACH) {
            const int f = row0 + row, node = node_of(f);
            const bool there = row < n_rows && my_d < dh;
            const T* at = q + (there ? (size_t)(r.tok0 + node) * q_stride + (size_t)(kvh * G + f - node * G) * dh + my_d : 0);
            tp_row4(sq + row * LD + my_d, at, there, q_vectors, dh - my_d);
        }
#pragma unroll 1
        for (int i = 0; i < 2; ++i) copy(i ? sv : sk, i ? v_cache : k_cache);
        TreeRow see[R];
        float m[R], l[R], o[R][J * 4];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int row = ty * R + i;
            if (row < n_rows) see[i] = tree_row(w, r, seen, node_of(row0 + row));
            else { see[i].lo = 0x7fffffff; see[i].bits = 0; }
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int d = 0; d < J * 4; ++d) o[i][d] = 0.f;
        }
        for (int t = walk.from; t < walk.to; ++t) {
            const int key0 = (r.t_lo + t) * TP_KEYS;
            asm volatile("cp.async.wait_group 1;" ::: "memory");         // K is there
            __syncthreads();
            float x[R][4] = {};
#pragma unroll 4
            for (int d = 0; d < DP; d += 4) {
                float4 a[R], b[4];
#pragma unroll
                for (int i = 0; i < R; ++i) a[i] = *(const float4*)(sq + (ty * R + i) * LD + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = *(const float4*)(sk + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[i][j] = fmaf(a[i].x, b[j].x, x[i][j]);
                        x[i][j] = fmaf(a[i].y, b[j].y, x[i][j]);
                        x[i][j] = fmaf(a[i].z, b[j].z, x[i][j]);
                        x[i][j] = fmaf(a[i].w, b[j].w, x[i][j]);
                    }
            }
            __syncthreads();                      // K has been read
            if (t + 1 < walk.to) {
                look(t + 1);
                copy(sk, k_cache);
            } else {
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
            // all of the tile's keys are seen by every row: cached, behind every window's beginning
            const bool whole = key0 + TP_KEYS <= min(hi, r.base) && (w.window <= 0 || key0 >= r.base + r.n - w.window);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                uint32_t ok = ty * R + i < n_rows ? 15u : 0u;
                if (!whole)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = key0 + tx + 16 * j;
                        if (!(key < hi && see[i].sees(key, r.base, r.n))) ok &= ~(1u << j);
                    }
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (ok >> j & 1u) mx = fmaxf(mx, x[i][j]);
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, s));
                const float m_new = fmaxf(m[i], mx * c);
                const float corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                m[i] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float p = ok >> j & 1u ? exp2f(fmaf(x[i][j], c, -ref)) : -0.f;
                    sum += p;
                    ss[(ty * R + i) * LS + tx + 16 * j] = p;
                }
                l[i] = l[i] * corr + sum;
#pragma unroll
                for (int d = 0; d < J * 4; ++d) o[i][d] *= corr;
            }
            asm volatile("cp.async.wait_group 1;" ::: "memory");         // V is there
            bool odd = false;                     // values that are no finite numbers where not every row sees them
            if (!whole)
#pragma unroll
                for (int i = 0; i < PASSES; ++i) {
                    const float4 v = *(const float4*)(sv + (my_row + i * EACH) * LD + my_d);
                    odd |= !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
                }
            if (!__syncthreads_or(odd)) {
#pragma unroll 2
                for (int k = 0; k < TP_KEYS; k += 4) {
                    float p[R][4];
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float4 u = *(const float4*)(ss + (ty * R + i) * LS + k);
                        p[i][0] = u.x; p[i][1] = u.y; p[i][2] = u.z; p[i][3] = u.w;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < J; ++j) {
                            const float4 v = *(const float4*)(sv + (k + e) * LD + tx * 4 + 64 * j);
#pragma unroll
                            for (int i = 0; i < R; ++i) {
                                o[i][4 * j] = fmaf(p[i][e], v.x, o[i][4 * j]);
                                o[i][4 * j + 1] = fmaf(p[i][e], v.y, o[i][4 * j + 1]);
                                o[i][4 * j + 2] = fmaf(p[i][e], v.z, o[i][4 * j + 2]);
                                o[i][4 * j + 3] = fmaf(p[i][e], v.w, o[i][4 * j + 3]);
                            }
                        }
                }
            } else {
#pragma unroll 1
                for (int k = 0; k < TP_KEYS; ++k) {
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float p = ss[(ty * R + i) * LS + k];
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
            __syncthreads();                      // V has been read
            if (t + 1 < walk.to) {
                look(t + 1);
                copy(sv, v_cache);
            } else {
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        const bool whole_item = walk.from == 0 && walk.to == r.tiles;
        if (tid == 0 && walk.from == 0 && !whole_item) notes[blockIdx.x] = tree_note(w, walk, blockIdx.x);
        const size_t slot = (size_t)blockIdx.x * 2 + (walk.from == 0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float sum = l[i];
#pragma unroll
            for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            const int row = ty * R + i, f = row0 + row;
            if (row >= n_rows) continue;
            if (whole_item) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const int node = node_of(f);
                T* dst = out + (size_t)(r.tok0 + node) * out_stride + (size_t)(kvh * G + f - node * G) * dh;
#pragma unroll
                for (int d = 0; d < J * 4; ++d) {
                    const int col = tx * 4 + 64 * (d >> 2) + (d & 3);
                    if (col < dh) dst[col] = from_f32<T>(o[i][d] * inv);
                }
            } else {
                const int fours = (dh + 3) / 4;
                float4* dst = (float4*)part_o + slot * fours * w.rows_per_tile + row;
#pragma unroll
                for (int j = 0; j < J; ++j)
                    if (tx + 16 * j < fours) dst[(tx + 16 * j) * w.rows_per_tile] = make_float4(o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]);
                if (tx == 0) *(float2*)(part_ml + (slot * w.rows_per_tile + row) * 2) = make_float2(m[i], sum);
            }
        }
    }
    pdl_launch_late();
}

// -------------------------------------------------------------------------- tensor cores
// bfloat16, heads of 64 or 128, pages of 8 to 128 places: tcgen05, tiles of 128 keys. An item's query rows (row r = node
// r / G, head r % G) make one tile of 128 rows or, for wide trees, two, which share the item's K and V. One persistent CTA an
// SM walks its pieces.
//
// The softmax of a tile takes longer than its two products: a warp's line of scores read, maxima found, exponentials, sums and
// weights stored, each behind the other (fewer exponentials for the special-function unit changed nothing). So there are two streams, each with scores S, sums O, a running
// maximum and a sum of exponentials of its own, and four softmax warps, a thread a row, that need nothing of each other:
// two row tiles, or, where there is one, the first and the second half of every key tile, put together at the item's end. A
// step of a stream is 64 keys, and its scores have two buffers: the next step's are made while this one's exponentials run.
//   warp 0        walks, publishes a record of every item in a ring and asks TMA for its Q rows and its K pages;
//   warp 3        walks too, and asks for the V pages (two tiles of each are in flight; a warp starts a copy about every
//                 80 cycles, 16 copies a tile of 16-place pages);
//   warp 1        issues S = Q K^T, warp 2 O += P V, a thread each;
//   warps 4-7, 8-11   softmax of stream 0 and of stream 1; P lies over its scores;
//   warps 12-15   clean V's tiles where that is needed, and take an item's result out of tensor memory.
// The running maximum moves only when a row has outgrown it by 2^8: then, when the product before has run, O is rescaled. P
// is rounded to bfloat16, at most 2^-8 of a weight, as the storage's own rounding is; its sum is not.
// Rows of V that nobody sees are zeroed before the product, the cache may hold anything there. Where only some rows see
// a key (the nodes, and the cached keys at the windows' edges), a value that is no finite number is zeroed too, and its
// key noted: at the item's end the rows that see it get it added (it is read from the cache again then).
// Waits have a limit of about two seconds, after which a code is left, what is under way is waited for, and the CTA ends.
//   MEASURED, in a graph of calls, with the join: 8 requests of 16 nodes, 4099 to 1230 keys, 8 kv heads of 4 query heads of 128: 27.5 us (90
// MB of K and V; 1.3 us a tile of 128 keys, which is the copy rate, beside 11.5 of beginnings, ends and the join); 2 requests of
// 64 nodes over 32703 keys: 78 us, 0.85 PFLOP/s, the softmax threads; one request of 8 nodes over 497 keys 11.4 us: a chain of
// reads (lengths, pages, K), a masked tile, its result. Taken back: the four softmax warps of a stream as eight with two threads a row
// (29 and 92 us for 27.5 and 79), a quarter of the exponentials as cubics on the FMA units (the same), K and V asked for by
// one warp (a copy every 80 cycles, 32 a tile), pages into the L2 ahead of them (33 and 92).
#define TT_ROWS 128
#define TT_KEYS 128
#define TT_THREADS 512
#define TT_BLOCK (128 * 64 * 2)               // 128 rows x 64 columns of bfloat16
#define TT_TILE (2 * TT_BLOCK)

__device__ int tree_error_flag = 0;

struct TreeItem {
    int valid;                                // 0: no more
    int tok0, n_rows, kvh, seq;               // its first token
    int key_tile, n_it;                       // key tiles from .. on, 0: zeros out
    int base, n, lo, hi;                      // of the request; keys lo .. hi - 1 are somebody's
    int whole, slot;                          // the item's result, or a part of it
    int pad[3];
};

__device__ __forceinline__ float tt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two numbers at a time.
__device__ __forceinline__ unsigned long long tt_pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void tt_unpair(unsigned long long p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ unsigned long long tt_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long tt_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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
__device__ __forceinline__ int tt_low(const TreeWork& w, int base) { return w.window > 0 && base > w.window ? base - w.window : 0; }
// Whether V's tile that begins at this key holds places that not every row sees.
__device__ __forceinline__ bool tt_mixed(int key, int base, int lo, int hi, int window) {
    return key + TT_KEYS > min(base, hi) || (window > 0 && key < lo + TREE_NODES);
}

// The pages of a piece's key tiles: a lane asks for those whose place in the piece is its number, 32 at a time; the next 32
// numbers are read meanwhile.
struct TreePages {
    const int* table;
    int lo, hi, n_it;                         // keys of somebody's, key tiles
    int first, end, per_tile, shift;          // of the piece: its first page, behind its last
    int group, page, next_page;
    __device__ __forceinline__ TreePages() { n_it = 0; }
    __device__ __forceinline__ TreePages(const TreeWork& w, const TreeWalk<TT_KEYS>& k, const int* tables, int max_blocks, int page_shift) {
        lo = tt_low(w, k.r.base);
        hi = min(k.r.len, w.max_keys);
        n_it = k.r.base < 0 || hi <= lo ? 0 : k.to - k.from;
        shift = page_shift;
        per_tile = TT_KEYS >> page_shift;
        table = tables + (size_t)k.b * max_blocks;
        first = group = (k.r.t_lo + k.from) * per_tile;
        end = min(first + n_it * per_tile, max_blocks);
        const int mine = group + (int)(threadIdx.x & 31);
        page = mine < end ? table[mine] : -1;
        next_page = -1;
    }
    __device__ __forceinline__ void turn(int it) {
        const int p0 = first + it * per_tile;
        if (p0 >= group + 32) {
            group += 32;
            page = next_page;
        }
        const int mine = group + 32 + (int)(threadIdx.x & 31);
        if (p0 == group) next_page = mine < end ? table[mine] : -1;
    }
    // tile `it`, of which only pages that hold a key of somebody's; a page is two boxes of 64 columns, or one
    template <int NH>
    __device__ __forceinline__ void load(const CUtensorMap* map, unsigned char* tile, uint64_t* bar, int it, int Hkv, int kvh, int n_pages) {
        const int p0 = first + it * per_tile, from = max(p0, lo >> shift), to = min(p0 + per_tile, ((hi - 1) >> shift) + 1);
        const int lane = threadIdx.x & 31, mine = group + lane;
        if (lane == 0) tg_expect(bar, (uint32_t)max(to - from, 0) << (shift + 7) << (NH - 1));
        __syncwarp();
        if (mine >= from && mine < to) {
            // a number that names no page reads zeros: rows behind the last
            const int row = (page >= 0 && page < n_pages ? page * Hkv + kvh : n_pages * Hkv) << shift;
            unsigned char* dst = tile + ((mine - p0) << (shift + 7));
            tg_load_2d(dst, map, 0, row, bar);
            if (NH > 1) tg_load_2d(dst + TT_BLOCK, map, 64, row, bar);
        }
    }
};

// DH: head size. RT: row tiles of an item (at most).
template <int DH, int RT>
__global__ void __launch_bounds__(TT_THREADS, 1) tree_tc_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
    const bf16* __restrict__ v_cache, int n_pages, bf16* __restrict__ out, long long out_stride, int page_size, int page_shift,
    const int* __restrict__ block_tables, int max_blocks, const unsigned long long* __restrict__ seen, float scale_log2,
    const TreeWork w, float* __restrict__ part_o, float* __restrict__ part_ml, TreeNote* __restrict__ notes) {
    constexpr int NH = DH / 64;
    extern __shared__ unsigned char tt_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)tt_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = base;                                   // [2][2 column halves][128 rows][128 bytes]
    unsigned char* sK = sQ + 2 * TT_TILE;
    unsigned char* sV = sK + 2 * TT_TILE;
    uint64_t* bars = (uint64_t*)(sV + 2 * TT_TILE);
    uint64_t *q_full = bars, *q_empty = bars + 2, *k_full = bars + 4, *k_empty = bars + 6, *v_full = bars + 8, *v_empty = bars + 10,
             *told = bars + 12, *bits_told = bars + 14,         // an item's record, what its nodes see
             *v_raw = bars + 16, *v_clean = bars + 18,          // mixed tiles: landed, cleaned
             *o_full = bars + 20, *l_full = bars + 22, *o_free = bars + 24,         // of an item
             *settled = bars + 26, *s_full = bars + 28, *p_full = bars + 32, *p_free = bars + 36;       // [stream][buffer]
    unsigned long long* odd_nodes = (unsigned long long*)(bars + 40);       // [8 items]: nodes, and keys lo + i, whose values
    unsigned long long* odd_edge = odd_nodes + 8;                           // are not all finite
    unsigned long long* s_bits = odd_edge + 8;                  // [2][64 nodes of the item]
    TreeItem* ring = (TreeItem*)(s_bits + 128);                 // [4]
    float* s_m = (float*)(ring + 4);                            // [2 items][2 streams][128 rows]
    float* s_l = s_m + 512;
    uint4* s_stage = (uint4*)(s_l + 512);                       // [4 warps][32 rows][64 bytes]
    uint32_t* tmem_slot = (uint32_t*)(s_stage + 512);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = w.H / w.Hkv;
    const int tile_tokens = TT_ROWS / G, tile_rows = tile_tokens * G;       // of a row tile
    const uint32_t by_g = (65535u + (uint32_t)G) / (uint32_t)G;             // r / G for r < 256
    auto node_of = [&](int r) { return (int)((uint32_t)r * by_g >> 16); };
    int* const err = &tree_error_flag;
    // rows of the Q tiles that no box writes must not hold NaN by chance
    if (tile_rows != TT_ROWS) for (int i = tid; i < 2 * TT_TILE / 16; i += TT_THREADS) ((uint4*)sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid < 16) odd_nodes[tid] = 0;
    if (tid == 64) {
        for (int i = 0; i < 2; ++i) {
            tg_init(&q_full[i], 1); tg_init(&q_empty[i], 14);   // products 1 + 1, softmax 8, results 4
            tg_init(&k_full[i], 1); tg_init(&k_empty[i], 1);
            tg_init(&v_full[i], 1); tg_init(&v_empty[i], 1);
            tg_init(&told[i], 1); tg_init(&bits_told[i], 1);
            tg_init(&v_raw[i], 1); tg_init(&v_clean[i], 4);
            tg_init(&s_full[i], 1); tg_init(&p_full[i], 4); tg_init(&p_free[i], 1);
            tg_init(&s_full[2 + i], 1); tg_init(&p_full[2 + i], 4); tg_init(&p_free[2 + i], 1);
            tg_init(&o_full[i], 1); tg_init(&l_full[i], 8); tg_init(&o_free[i], 4);
            tg_init(&settled[i], 1);
        }
    }
    tg_init_done();
    if (warp == 1) tg_alloc512(tmem_slot);
    pdl_wait();
    // The two warps that ask for copies find their pieces first; they wait for what the others have laid out, and nobody for them.
    TreeWalk<TT_KEYS> walk;
    if (warp == 0 || warp == 3) {
        walk.find(w, blockIdx.x);
        __syncwarp();
        asm volatile("barrier.cta.sync.aligned 1, %0;" ::"n"(TT_THREADS) : "memory");
    } else {
        __syncwarp();
        tg_before();
        asm volatile("barrier.cta.arrive.aligned 1, %0;" ::"n"(TT_THREADS) : "memory");
        asm volatile("barrier.cta.sync.aligned 2, %0;" ::"n"(TT_THREADS - 64) : "memory");
    }
    tg_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------------- records and Q
        TreeNote note = {0, 0, 0, 0, 0};
        if (lane == 0 && !w.whole) notes[blockIdx.x] = note;
        uint32_t sent = 0, g = 0;                               // items whose Q was asked for, key tiles
        bool ok = true;
        for (uint32_t n = 0;; ++n) {
            // A record lies in n % 4; a buffer of Q and of what nodes see is item n's if n is even, and the other one's
            // otherwise, or both tiles of Q are the item's.
            TreeItem* rec = &ring[n & 3];
            const uint32_t qb = n & 1u, qph = (n >> 1) & 1u;
            const bool more = walk.next(w);
            const TreeRequest& r = walk.r;
            const int token = walk.row_tile * w.tokens_per_tile;
            TreePages pages;
            if (more) pages = TreePages(w, walk, block_tables, max_blocks, page_shift);
            // what its nodes see, read while the buffers come free
            unsigned long long bits[2] = {0, 0};
            if (more)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (lane + 32 * h < w.tokens_per_tile && token + lane + 32 * h < r.n)
                        bits[h] = seen[r.tok0 + token + lane + 32 * h] & (r.n >= 64 ? ~0ull : (1ull << r.n) - 1ull);
            ok = __all_sync(0xffffffffu, tg_wait(&q_empty[qb], qph ^ 1u, err, 1));
            if (RT == 2 && ok && n > 0) ok = __all_sync(0xffffffffu, tg_wait(&q_empty[qb ^ 1u], ((n - 1u) >> 1) & 1u, err, 1));
            if (!ok) break;
            if (!more) {
                if (lane == 0) {
                    rec->valid = 0;
                    tg_arrive(&told[qb]);
                    tg_arrive(&bits_told[qb]);
                    if (!w.whole) notes[blockIdx.x] = note;
                }
                break;
            }
            if (lane == 0) {
                const int tok0 = r.tok0 + token, n_it = pages.n_it;
                const int n_rows = min(r.n - token, w.tokens_per_tile) * G;
                rec->valid = 1;
                rec->tok0 = tok0;
                rec->n_rows = n_rows;
                rec->kvh = walk.kvh; rec->seq = walk.b;
                rec->key_tile = r.t_lo + walk.from;
                rec->n_it = n_it;
                rec->base = r.base; rec->n = r.n;
                rec->lo = pages.lo; rec->hi = pages.hi;
                rec->whole = walk.from == 0 && walk.to == r.tiles;
                rec->slot = (int)blockIdx.x * 2 + (walk.from == 0 ? 1 : 0);
                tg_arrive(&told[qb]);
                if (n_it > 0) {
                    // the G heads of a full tile's tokens: tokens behind this tile's are others' rows, whose results are
                    // not stored, tokens behind the last zeros
                    const int tiles = RT == 2 && n_rows > tile_rows ? 2 : 1;
                    tg_expect(&q_full[qb], (uint32_t)(tiles * NH * tile_rows) * 128u);
                    for (int t = 0; t < tiles; ++t) {
                        unsigned char* dq = sQ + (RT == 2 ? (uint32_t)t : qb) * TT_TILE;
                        tt_load_3d(dq, &map_q, 0, walk.kvh * G, tok0 + t * tile_tokens, &q_full[qb]);
                        if (NH > 1) tt_load_3d(dq + TT_BLOCK, &map_q, 64, walk.kvh * G, tok0 + t * tile_tokens, &q_full[qb]);
                    }
                } else {
                    tg_arrive(&q_full[qb]);
                }
            }
            ++sent;
            s_bits[qb * 64 + lane] = bits[0];
            s_bits[qb * 64 + lane + 32] = bits[1];
            __syncwarp();
            if (lane == 0) tg_arrive(&bits_told[qb]);
            if (walk.from == 0 && walk.to < r.tiles) note = tree_note(w, walk, blockIdx.x);
            for (int it = 0; it < pages.n_it; ++it, ++g) {
                const uint32_t s = g & 1u;
                pages.turn(it);
                ok = __all_sync(0xffffffffu, tg_wait(&k_empty[s], ((g >> 1) & 1u) ^ 1u, err, 1));
                if (!ok) break;
                pages.load<NH>(&map_k, sK + s * TT_TILE, &k_full[s], it, w.Hkv, walk.kvh, n_pages);
            }
            if (!ok) break;
            __syncwarp();
        }
        if (!ok) {                                              // the copies under way
            tg_settle_copies(q_full, 2, sent, err, 1);
            tg_settle_copies(k_full, 2, g, err, 1);
        }
    } else if (warp == 3) {
        // ------------------------------------------------------------- V
        bool ok = true;
        uint32_t g = 0, mixed = 0, plain0 = 0, plain1 = 0;      // tiles; mixed ones, the others by stage
        while (ok && walk.next(w)) {
            TreePages pages(w, walk, block_tables, max_blocks, page_shift);
            for (int it = 0; it < pages.n_it; ++it, ++g) {
                const uint32_t s = g & 1u;
                pages.turn(it);
                ok = __all_sync(0xffffffffu, tg_wait(&v_empty[s], ((g >> 1) & 1u) ^ 1u, err, 1));
                if (!ok) break;
                uint64_t* bar = &v_full[s];
                if (tt_mixed((walk.r.t_lo + walk.from + it) * TT_KEYS, walk.r.base, pages.lo, pages.hi, w.window)) bar = &v_raw[mixed++ & 1u];
                else if (s) ++plain1;
                else ++plain0;
                pages.load<NH>(&map_v, sV + s * TT_TILE, bar, it, w.Hkv, walk.kvh, n_pages);
            }
            __syncwarp();
        }
        if (!ok) {                                              // the copies under way
            tg_settle_copies(v_raw, 2, mixed, err, 1);
            if (plain0) tg_wait(&v_full[0], (plain0 - 1u) & 1u, err, 1);
            if (plain1) tg_wait(&v_full[1], (plain1 - 1u) & 1u, err, 1);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------- S = Q K^T
        if (tg_elect()) {
            const uint32_t idesc = tg_idesc(64);
            uint32_t g = 0, steps[2] = {0, 0};                  // key tiles, steps of each stream
            bool ok = true;
            for (uint32_t n = 0; ok; ++n) {
                const uint32_t qb = n & 1u;
                ok = tg_wait(&told[qb], (n >> 1) & 1u, err, 2);
                if (!ok) break;
                const TreeItem* rec = &ring[n & 3];
                if (!rec->valid) break;
                const int n_it = rec->n_it;
                const bool two = RT == 2 && rec->n_rows > tile_rows;
                ok = tg_wait(&q_full[qb], (n >> 1) & 1u, err, 2);
                if (!ok) break;
                for (int it = 0; it < n_it && ok; ++it, ++g) {
                    const uint32_t s = g & 1u, ph = (g >> 1) & 1u;
                    ok = tg_wait(&k_full[s], ph, err, 2);
#pragma unroll
                    for (int u = 0; u < 2 * RT; ++u) {
                        const int x = u & 1, half = RT == 2 ? u >> 1 : u;          // the stream, and the tile's half
                        if (RT == 2 && x == 1 && !two) continue;
                        const uint32_t step = steps[x]++, b = step & 1u;
                        ok = ok && tg_wait(&p_free[2 * x + b], ((step >> 1) & 1u) ^ 1u, err, 2);     // the product with what lay there has run
                        if (!ok) break;
                        tg_after();
                        const unsigned char* qt = sQ + (RT == 2 ? (uint32_t)x : qb) * TT_TILE;
                        const unsigned char* kt = sK + s * TT_TILE + half * (TT_BLOCK / 2);
                        const uint64_t dq0 = tg_desc(qt), dq1 = tg_desc(qt + TT_BLOCK), dk0 = tg_desc(kt), dk1 = tg_desc(kt + TT_BLOCK);
                        const uint32_t d = tmem + 128u * x + 64u * b;
#pragma unroll
                        for (int k = 0; k < 4; ++k) tg_mma(d, dq0 + 2 * k, dk0 + 2 * k, idesc, k > 0 ? 1u : 0u);
                        if (NH > 1)
#pragma unroll
                            for (int k = 0; k < 4; ++k) tg_mma(d, dq1 + 2 * k, dk1 + 2 * k, idesc, 1u);
                        tg_commit(&s_full[2 * x + b]);
                    }
                    if (ok) tg_commit(&k_empty[s]);
                }
                if (ok) tg_commit(&q_empty[qb]);
            }
            if (!ok) tg_settle_products(&settled[0], err, 2);
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------- O += P V
        if (tg_elect()) {
            const uint32_t idesc = tg_idesc(DH, true);
            uint32_t g = 0, mixed = 0, plain0 = 0, plain1 = 0, steps[2] = {0, 0}, walked = 0;
            bool ok = true;
            for (uint32_t n = 0; ok; ++n) {
                ok = tg_wait(&told[n & 1u], (n >> 1) & 1u, err, 2);
                if (!ok) break;
                const TreeItem* rec = &ring[n & 3];
                if (!rec->valid) break;
                const int n_it = rec->n_it, key_tile = rec->key_tile, r_base = rec->base, lo = rec->lo, hi = rec->hi;
                const bool two = RT == 2 && rec->n_rows > tile_rows;
                tg_arrive(&q_empty[n & 1u]);
                if (n_it == 0) continue;
                // the last item's O is out
                if (walked > 0) ok = tg_wait(&o_free[(walked - 1u) & 1u], ((walked - 1u) >> 1) & 1u, err, 2);
                for (int it = 0; it < n_it && ok; ++it, ++g) {
                    const uint32_t s = g & 1u;
                    if (tt_mixed((key_tile + it) * TT_KEYS, r_base, lo, hi, w.window)) {
                        ok = tg_wait(&v_clean[mixed & 1u], (mixed >> 1) & 1u, err, 2);
                        ++mixed;
                    } else {
                        ok = tg_wait(&v_full[s], (s ? plain1++ : plain0++) & 1u, err, 2);
                    }
#pragma unroll
                    for (int u = 0; u < 2 * RT; ++u) {
                        const int x = u & 1, half = RT == 2 ? u >> 1 : u;
                        if (RT == 2 && x == 1 && !two) continue;
                        const uint32_t step = steps[x]++, b = step & 1u;
                        ok = ok && tg_wait(&p_full[2 * x + b], (step >> 1) & 1u, err, 2);
                        if (!ok) break;
                        tg_after();
                        const unsigned char* vt = sV + s * TT_TILE + half * (TT_BLOCK / 2);
                        const uint64_t dv = NH > 1 ? tg_desc_mn(vt, TT_BLOCK) : tg_desc(vt);
                        const uint32_t more = it > 0 || (RT == 2 && half > 0);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tg_mma_ts(tmem + 256u + 128u * x, tmem + 128u * x + 64u * b + 8u * k, dv + (uint64_t)(128 * k), idesc, k > 0 ? 1u : more);
                        tg_commit(&p_free[2 * x + b]);
                    }
                    if (ok) tg_commit(&v_empty[s]);
                }
                if (ok) tg_commit(&o_full[walked & 1u]);
                ++walked;
            }
            if (!ok) tg_settle_products(&settled[1], err, 2);
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------- softmax
        const int quarter = warp & 3, x = (warp - 4) >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t tm_x = tmem + 128u * x + lane_base, tm_o = tmem + 256u + 128u * x + lane_base;
        const int row_lo = RT == 2 ? x * tile_rows : 0;         // the item's row that is row 0 here
        bool ok = true;
        uint32_t step = 0, walked = 0;                          // this stream's, items with any
        for (uint32_t n = 0;; ++n) {
            ok = __all_sync(0xffffffffu, tg_wait(&bits_told[n & 1u], (n >> 1) & 1u, err, 3));
            if (!ok) break;
            const TreeItem rec = ring[n & 3];
            const int n_rows = min(rec.n_rows - row_lo, tile_rows);
            const bool row_ok = row < n_rows;
            const unsigned long long bits = rec.valid && row_ok ? s_bits[(n & 1u) * 64 + node_of(row_lo + row)] : 0ull;
            if (!rec.valid) break;
            __syncwarp();
            if (lane == 0) tg_arrive(&q_empty[n & 1u]);
            if (rec.n_it == 0) continue;
            const bool live = quarter * 32 < n_rows;            // a row of the warp's is somebody's
            const int lo = !row_ok ? 0x7fffffff : w.window > 0 ? max(rec.base + __popcll(bits) - w.window, 0) : 0;
            const bool warp_rows_ok = quarter * 32 + 31 < n_rows;
            // keys whole_lo .. base - 1 are seen by every row
            const int whole_lo = w.window > 0 ? rec.base + rec.n - w.window : 0;
            float m_used = -INFINITY, l = 0.f;
            const int n_steps = n_rows <= 0 ? 0 : RT * rec.n_it;
            for (int i_step = 0; i_step < n_steps; ++i_step, ++step) {
                const uint32_t b = step & 1u;
                ok = __all_sync(0xffffffffu, tg_wait(&s_full[2 * x + b], (step >> 1) & 1u, err, 3));
                if (!ok) break;
                if (live) {
                    tg_after();
                    const uint32_t tm_s = tm_x + 64u * b;
                    const int kbase = rec.key_tile * TT_KEYS + (RT == 2 ? 64 * i_step : TT_KEYS * i_step + 64 * x);
                    float sc[64];
                    {
                        uint32_t r0[32], r1[32];
                        tg_ld32(tm_s, r0);
                        tg_ld32(tm_s + 32u, r1);
                        tg_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) { sc[i] = __uint_as_float(r0[i]); sc[32 + i] = __uint_as_float(r1[i]); }
                    }
                    if (!(warp_rows_ok && kbase + 64 <= min(rec.base, rec.hi) && kbase >= whole_lo)) {
                        const unsigned long long see = (tt_range(lo - kbase, rec.base - kbase) | tt_shift(bits, rec.base - kbase)) &
                                                       tt_range(0, rec.hi - kbase);
                        const uint32_t see0 = (uint32_t)see, see1 = (uint32_t)(see >> 32);
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            sc[i] = see0 >> i & 1u ? sc[i] : -INFINITY;
                            sc[32 + i] = see1 >> i & 1u ? sc[32 + i] : -INFINITY;
                        }
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], fmaxf(sc[2 * i], sc[2 * i + 1]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
                    const float m_new = fmaxf(m_used, mx);
                    const bool grow = m_new > m_used + 8.f || (m_used == -INFINITY && m_new != -INFINITY);
                    if (__any_sync(0xffffffffu, grow)) {
                        const float corr = m_new == -INFINITY ? 1.f : exp2f(m_used - m_new);
                        m_used = m_new;
                        l *= corr;
                        if (i_step > 0) {
                            // when the product before has run
                            ok = __all_sync(0xffffffffu, tg_wait(&p_free[2 * x + (b ^ 1u)], ((step - 1u) >> 1) & 1u, err, 3));
                            if (!ok) break;
                            tg_after();
#pragma unroll 1
                            for (int c = 0; c < 2 * NH; ++c) {
                                uint32_t r[32];
                                tg_ld32(tm_o + 32u * c, r);
                                tg_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * corr);
                                tg_st32(tm_o + 32u * c, r);
                            }
                        }
                    }
                    const float ref = m_used == -INFINITY ? 0.f : m_used;
                    const unsigned long long scale2 = tt_pair(scale_log2, scale_log2), ref2 = tt_pair(-ref, -ref);
                    unsigned long long sum2[2] = {0ull, 0ull};
                    uint32_t r[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        float y0, y1;
                        tt_unpair(tt_fma2(tt_pair(sc[2 * i], sc[2 * i + 1]), scale2, ref2), y0, y1);
                        y0 = tt_exp2(y0);
                        y1 = tt_exp2(y1);
                        sum2[i & 1] = tt_add2(sum2[i & 1], tt_pair(y0, y1));
                        r[i] = tg_pack(y0, y1);
                    }
                    tg_st32(tm_s, r);
                    float s0, s1;
                    tt_unpair(tt_add2(sum2[0], sum2[1]), s0, s1);
                    l += s0 + s1;
                    tg_wait_st();
                    tg_before();
                }
                __syncwarp();
                if (lane == 0) tg_arrive(&p_full[2 * x + b]);
            }
            if (!ok) break;
            // the row's sums to the warps that take the result out, when they have read those of the item before the last
            if (walked > 1) ok = __all_sync(0xffffffffu, tg_wait(&o_free[walked & 1u], ((walked >> 1) - 1u) & 1u, err, 3));
            if (!ok) break;
            s_m[(walked & 1u) * 256 + x * 128 + row] = m_used;
            s_l[(walked & 1u) * 256 + x * 128 + row] = l;
            __syncwarp();
            if (lane == 0) tg_arrive(&l_full[walked & 1u]);
            ++walked;
        }
    } else {
        // ------------------------------------------------------------- V cleaned, results out
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        uint4* const stage = s_stage + quarter * 128;
        uint32_t g = 0, mixed = 0, walked = 0;                  // key tiles, mixed ones, items with any
        bool ok = true;
        for (uint32_t n = 0;; ++n) {
            ok = __all_sync(0xffffffffu, tg_wait(&bits_told[n & 1u], (n >> 1) & 1u, err, 4));
            if (!ok) break;
            const TreeItem rec = ring[n & 3];
            if (!rec.valid) break;
            unsigned long long bits[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t)
                bits[t] = row < min(rec.n_rows - t * tile_rows, tile_rows) ? s_bits[(n & 1u) * 64 + node_of(t * tile_rows + row)] : 0ull;
            __syncwarp();
            if (lane == 0) tg_arrive(&q_empty[n & 1u]);
            auto result = [&](int r) {
                const int node = node_of(r);
                return out + (size_t)(rec.tok0 + node) * out_stride + (size_t)(rec.kvh * G + r - node * G) * DH;
            };
            if (rec.n_it == 0) {
                for (int r = row; r < rec.n_rows; r += TT_ROWS) {
                    bf16* dst = result(r);
                    for (int i = 0; i < DH / 8; ++i) *(uint4*)(dst + i * 8) = make_uint4(0u, 0u, 0u, 0u);
                }
                continue;
            }
            const int whole_lo = w.window > 0 ? rec.base + rec.n - w.window : 0;
            for (int it = 0; it < rec.n_it; ++it, ++g) {
                const int tile_lo = (rec.key_tile + it) * TT_KEYS;
                if (!tt_mixed(tile_lo, rec.base, rec.lo, rec.hi, w.window)) continue;
                ok = __all_sync(0xffffffffu, tg_wait(&v_raw[mixed & 1u], (mixed >> 1) & 1u, err, 4));
                if (!ok) break;
                const int key = tile_lo + row;
                const bool nobody = key >= rec.hi || key < rec.lo;
                if (nobody || key >= rec.base || key < whole_lo) {
                    unsigned char* vrow = sV + (g & 1u) * TT_TILE + row * 128;
                    bool odd = false;
#pragma unroll
                    for (int c = 0; c < 8 * NH; ++c) {
                        // eight lanes' rows lie 128 bytes apart: each begins at another sixteen of them
                        uint4* at = (uint4*)(vrow + (c >> 3) * TT_BLOCK + ((c ^ lane) & 7) * 16);
                        uint4 v = make_uint4(0u, 0u, 0u, 0u);
                        if (!nobody) {
                            const uint4 u = *at;
                            v = make_uint4(tt_finite(u.x), tt_finite(u.y), tt_finite(u.z), tt_finite(u.w));
                            if (v.x == u.x && v.y == u.y && v.z == u.z && v.w == u.w) continue;
                            odd = true;
                        }
                        *at = v;
                    }
                    if (odd && key >= rec.base) atomicOr(&odd_nodes[walked & 7u], 1ull << (key - rec.base));
                    else if (odd) atomicOr(&odd_edge[walked & 7u], 1ull << (key - rec.lo));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) tg_arrive(&v_clean[mixed & 1u]);
                ++mixed;
            }
            if (!ok) break;
            const uint32_t wb = walked & 1u, turn = (walked >> 1) & 1u;
            ok = __all_sync(0xffffffffu, tg_wait(&l_full[wb], turn, err, 4) && tg_wait(&o_full[wb], turn, err, 4));
            if (!ok) break;
            tg_after();
#pragma unroll 1
            for (int t = 0; t < RT; ++t) {
                const int n_rows = min(rec.n_rows - t * tile_rows, tile_rows);
                if (quarter * 32 >= n_rows) break;
                const bool row_ok = row < n_rows;
                const unsigned long long mine = RT == 2 && t == 1 ? bits[RT - 1] : bits[0];
                const int lo = w.window > 0 ? max(rec.base + __popcll(mine) - w.window, 0) : 0;
                const unsigned long long nodes = odd_nodes[walked & 7u] & mine;
                const unsigned long long edge = row_ok ? odd_edge[walked & 7u] & tt_range(lo - rec.lo, rec.base - rec.lo) : 0ull;
                const float* sm = s_m + wb * 256 + (RT == 2 ? t * 128 : 0) + row;
                const float* sl = s_l + wb * 256 + (RT == 2 ? t * 128 : 0) + row;
                float m = sm[0], l = sl[0], f0 = 1.f, f1 = 0.f;
                if (RT == 1) {
                    const float m0 = m, m1 = sm[128];
                    m = fmaxf(m0, m1);
                    const float ref = m == -INFINITY ? 0.f : m;
                    f0 = exp2f(m0 - ref);
                    f1 = exp2f(m1 - ref);
                    l = l * f0 + sl[128] * f1;
                }
                if (rec.whole) {
                    const float inv = l == 0.f ? 0.f : 1.f / l;
                    f0 *= inv;
                    f1 *= inv;
                }
                const int item_row = t * tile_rows + row;
                if (!rec.whole && row_ok)
                    *(float2*)(part_ml + ((size_t)rec.slot * w.rows_per_tile + item_row) * 2) = make_float2(m, l);
                float4* po = (float4*)part_o + (size_t)rec.slot * (DH / 4) * w.rows_per_tile + item_row;
                const uint32_t tm_o = tmem + 256u + (RT == 2 ? 128u * t : 0u) + lane_base;
                // the rows that this lane stores: four lanes a row of 64 bytes
                bf16* line_out[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) line_out[k] = result(t * tile_rows + quarter * 32 + 8 * k + (lane >> 2)) + (lane & 3) * 8;
                auto emit = [&](bool odd) {
#pragma unroll 1
                    for (int c = 0; c < DH / 32; ++c) {
                        float o[32];
                        if (RT == 2) {
                            uint32_t r[32];
                            tg_ld32(tm_o + 32u * c, r);
                            tg_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(r[i]) * f0;
                        } else {
                            uint32_t r[32], u[32];
                            tg_ld32(tm_o + 32u * c, r);
                            tg_ld32(tm_o + 128u + 32u * c, u);
                            tg_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = fmaf(__uint_as_float(r[i]), f0, __uint_as_float(u[i]) * f1);
                        }
                        if (odd) {
                            for (int k = 0; k < 128; ++k) {
                                if (!((k < 64 ? nodes >> k : edge >> (k - 64)) & 1ull)) continue;
                                const int key = k < 64 ? rec.base + k : rec.lo + k - 64;
                                const int page = block_tables[(size_t)rec.seq * max_blocks + (key >> page_shift)];
                                const bf16* v = v_cache + (((size_t)page * w.Hkv + rec.kvh) * page_size + (key & (page_size - 1))) * DH + 32 * c;
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float y = __bfloat162float(v[i]);
                                    if (!isfinite(y)) o[i] += y;
                                }
                            }
                        }
                        if (rec.whole) {
                            // by way of shared memory
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                stage[lane * 4 + ((i ^ (lane >> 1)) & 3)] = make_uint4(tg_pack(o[8 * i], o[8 * i + 1]), tg_pack(o[8 * i + 2], o[8 * i + 3]),
                                                                             tg_pack(o[8 * i + 4], o[8 * i + 5]), tg_pack(o[8 * i + 6], o[8 * i + 7]));
                            __syncwarp();
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const int line = 8 * k + (lane >> 2);
                                if (quarter * 32 + line < n_rows) *(uint4*)(line_out[k] + 32 * c) = stage[line * 4 + ((lane ^ (line >> 1)) & 3)];
                            }
                            __syncwarp();
                        } else if (row_ok) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                po[(8 * c + i) * w.rows_per_tile] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                        }
                    }
                };
                if (__any_sync(0xffffffffu, (nodes | edge) != 0)) emit(true);
                else emit(false);
            }
            // these warps are at most two items apart: nobody reads the last item's but three any more, or writes them yet
            if (quarter == 0 && lane == 0) odd_nodes[(walked + 4u) & 7u] = odd_edge[(walked + 4u) & 7u] = 0;
            tg_before();
            __syncwarp();
            if (lane == 0) tg_arrive(&o_free[wb]);
            ++walked;
        }
    }
    pdl_launch_late();
    tg_before();
    __syncthreads();
    if (warp == 1) {
        tg_after();
        tg_free512(tmem);
    }
}

// ------------------------------------------------------------------------------- the join
// A part's sums lie four columns of all its rows after the other, as the workers' threads (a row each) store them. A warp
// joins 32 columns of eight rows of the item that worker j began and others ended, as its note says: its parts are worker
// j's second slot and the following workers' first ones, taken eight at a time. Bound by latency, a note and then its
// parts: about 3 us behind the first kernel.
#define TJ_WARPS 8
#define TJ_AHEAD 8
template <typename T>
__global__ void __launch_bounds__(TJ_WARPS * 32) tree_join_kernel(T* __restrict__ out, long long out_stride, int dh, int G,
                                                                  int rows_per_part, int strips, const TreeNote* __restrict__ notes,
                                                                  const float* __restrict__ part_o, const float* __restrict__ part_ml) {
    pdl_wait();
    const int lane = threadIdx.x & 31, j = blockIdx.x, unit = blockIdx.y * TJ_WARPS + (threadIdx.x >> 5);
    const TreeNote note = notes[j];
    const int row = unit / strips * 8 + (lane & 7), c0 = unit % strips * 8 + (lane >> 3), fours = (dh + 3) / 4;
    if (row >= note.n_rows) return;
    float m = -INFINITY, l = 0.f;
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int p0 = 0; p0 < note.parts; p0 += TJ_AHEAD) {
        float2 ml[TJ_AHEAD];
        float4 v[TJ_AHEAD][2];
#pragma unroll
        for (int p = 0; p < TJ_AHEAD; ++p) {
            ml[p] = make_float2(-INFINITY, 0.f);
            if (p0 + p >= note.parts) continue;
            const size_t slot = p0 + p == 0 ? 2 * j + 1 : 2 * (j + p0 + p);
            ml[p] = *(const float2*)(part_ml + (slot * rows_per_part + row) * 2);
            const float4* src = (const float4*)part_o + slot * fours * rows_per_part + row;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (c0 + 4 * i < fours) v[p][i] = src[(size_t)(c0 + 4 * i) * rows_per_part];
        }
        float m_new = m;
#pragma unroll
        for (int p = 0; p < TJ_AHEAD; ++p) m_new = fmaxf(m_new, ml[p].x);
        const float ref = m_new == -INFINITY ? 0.f : m_new, f = exp2f(m - ref);
        m = m_new;
        l *= f;
#pragma unroll
        for (int i = 0; i < 2; ++i) { o[i].x *= f; o[i].y *= f; o[i].z *= f; o[i].w *= f; }
#pragma unroll
        for (int p = 0; p < TJ_AHEAD; ++p) {
            if (p0 + p >= note.parts) continue;
            const float f_p = exp2f(ml[p].x - ref);
            l = fmaf(f_p, ml[p].y, l);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                o[i].x = fmaf(f_p, v[p][i].x, o[i].x);
                o[i].y = fmaf(f_p, v[p][i].y, o[i].y);
                o[i].z = fmaf(f_p, v[p][i].z, o[i].z);
                o[i].w = fmaf(f_p, v[p][i].w, o[i].w);
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int f = note.row0 + row;
    T* dst = out + (size_t)(note.tok0 + f / G) * out_stride + (size_t)(note.kvh * G + f % G) * dh;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float x[4] = {o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((c0 + 4 * i) * 4 + e < dh) dst[(c0 + 4 * i) * 4 + e] = from_f32<T>(x[e]);
    }
}

// ------------------------------------------------------------------------------------ host
// Whether the tensor cores' kernel takes calls of this layout (in bfloat16).
TGO_API int tgo_attention_tree_tc_supports(int dh, int group, int page_size) {
    return (dh == 64 || dh == 128) && group >= 1 && group <= TT_ROWS && page_size >= 8 && page_size <= TT_KEYS &&
           (page_size & (page_size - 1)) == 0;
}
// The code that a wait of that kernel left when it ran out (1 copies, 2 products, 3 softmax, 4 results), or 0. Synchronises.
TGO_API int tgo_attention_tree_error(int* value) { return (int)cudaMemcpyFromSymbol(value, tree_error_flag, sizeof(int)); }

static int tree_force = 0;                    // for tests: 1 plain products; 2, 3 items of one row tile, whole and cut; 4, 5 of two
TGO_API int tgo_attention_tree_force(int way) { tree_force = way; return 0; }

// The tensor map of query rows [tokens][heads][dh], `stride` apart, in boxes of 64 columns of G heads of a row tile's tokens.
static bool tree_map_q(CUtensorMap* map, const void* q, long long stride, int tokens, int H, int G, int dh) {
    const TgEncodeFn encode = tg_encode();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)dh, (cuuint64_t)H, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)dh * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(TT_ROWS / G)};
    const cuuint32_t elem[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T>
static int tree_join_go(void* out, long long out_stride, int dh, const TreeWork& w, const float* part_o, const float* part_ml,
                        const TreeNote* notes, cudaStream_t stream) {
    if (w.workers == 1 || w.whole) return 0;
    const int strips = (dh + 31) / 32, units = (w.rows_per_tile + 7) / 8 * strips;
    return tgo_launch_pdl(tree_join_kernel<T>, dim3(w.workers - 1, (units + TJ_WARPS - 1) / TJ_WARPS), dim3(TJ_WARPS * 32), 0, stream,
                          (T*)out, out_stride, dh, w.H / w.Hkv, w.rows_per_tile, strips, notes, part_o, part_ml);
}
// The workspace's parts: sums, (maximum, sum of exponentials) pairs, notes.
static float* tree_ml(float* work, const TreeWork& w, int dh) { return work ? work + (size_t)w.workers * 2 * w.rows_per_tile * ((dh + 3) / 4 * 4) : nullptr; }
static TreeNote* tree_notes(float* work, const TreeWork& w, int dh) { return work ? (TreeNote*)(tree_ml(work, w, dh) + (size_t)w.workers * 4 * w.rows_per_tile) : nullptr; }

template <int DH, int RT>
static int tree_tc_go(const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, const void* v, int n_pages, void* out,
                      long long out_stride, int page_size, const int* tables, int max_blocks, const void* seen, float scale,
                      const TreeWork& w, float* work, cudaStream_t stream) {
    constexpr size_t smem = 1024 + 6 * (size_t)TT_TILE + 184 * 8 + 4 * sizeof(TreeItem) + 1024 * sizeof(float) + 512 * 16 + 16;
    static bool set[64] = {};
    int dev = 0, shift = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!set[dev]) {
        e = cudaFuncSetAttribute(tree_tc_kernel<DH, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        set[dev] = true;
    }
    while ((1 << shift) < page_size) ++shift;
    const int rc = tgo_launch_pdl(tree_tc_kernel<DH, RT>, dim3(w.workers), dim3(TT_THREADS), smem, stream, mk, mv, mq, (const bf16*)v, n_pages,
                                  (bf16*)out, out_stride, page_size, shift, tables, max_blocks, (const unsigned long long*)seen,
                                  scale * TREE_LOG2E, w, work, tree_ml(work, w, DH), tree_notes(work, w, DH));
    if (rc) return rc;
    return tree_join_go<bf16>(out, out_stride, DH, w, work, tree_ml(work, w, DH), tree_notes(work, w, DH), stream);
}

// Most key tiles of an item.
static int tree_tiles(const TreeWork& w, int max_context, int keys) {
    const int reach = w.window > 0 && max_context > w.window + w.max_nodes ? w.window + w.max_nodes + keys - 1 : max_context;
    return reach <= keys ? 1 : (reach + keys - 1) / keys;
}

// The tensor cores' four ways, by what they took where they were measured (us; 8 kv heads of 4 query heads, 128 wide, lengths up to 30 %
// apart; "one" and "two": row tiles an item, "whole" and "cut"):
//                                   one whole  one cut  two whole  two cut
//    1 request of  4 nodes,    300       10.6     12.1
//    1             4,         1000       17.0     12.8
//   16             8,         2000       28.2     31.0
//   40             8,         1500       57.7     48.8
//    1            64,         2000       24.8     16.6       41.5     22.1
//    4            64,         1000       17.5     21.1       26.7     23.9
//    4            64,        16000      135.4     81.7      258.8     73.2
//   32            64,         1000       61.4     70.7       54.7     72.4
//    8            40,         8000       73.6     74.5      129.3     69.3
// Whole items run in rounds of one an SM; cutting costs a join and a beginning and an end for every piece, and shares all tiles out
// evenly. Straight lines through 65 such measurements: us for a call, a round or an item of each SM, and a key tile. The cheapest by
// them is within 11 % of the fastest measured (within 3 % in 63 of the 65). The lines know nothing of other layouts and of windows beyond
// the count of items and tiles; they hold for them: in 54 calls (heads of 64, groups of 1, 5 and 8, a window of 1024; 1 to 32 requests of 4 to
// 64 nodes over 300 to 8000 keys) the chosen way is within 3 % of the fastest, e.g.
//   16 over 2 of  64,  8 requests of 16, 4000   35.1     15.6
//   40 over 8 of 128, 16             8,  2000   31.1     33.2
//   64 over 8 of 128, 12            23,  window 35.4     40.8      30.5     39.8
static void tree_choose(TreeWork& w, int max_context, int G, int sms) {
    const int tokens = TT_ROWS / G, t = tree_tiles(w, max_context, TT_KEYS);
    double best = 0;
    int way = 0;
    for (int rt = 1; rt <= 2; ++rt) {
        if (rt == 2 && w.max_nodes <= tokens) break;
        const double items = (double)w.B * w.Hkv * ((w.max_nodes + rt * tokens - 1) / (rt * tokens));
        const double rounds = (double)(long long)((items + sms - 1) / sms);
        const double whole = rt == 1 ? 3.2 + rounds * (4.5 + 1.1 * t) : rounds * (10.8 + 1.95 * t) - 1.8;
        const double each = items * (t + TREE_OVERHEAD) / sms, tiles = each > 1 ? each : 1;
        const double cut = rt == 1 ? 11.5 + items / sms * 2.5 + tiles * 1.3 : 18.3 + items / sms * 5.0 + tiles * 2.1;
        if (!way || whole < best) { best = whole; way = 2 * rt; }
        if (cut < best) { best = cut; way = 2 * rt + 1; }
    }
    if (tree_force >= 2 && (tree_force < 4 || w.max_nodes > tokens)) way = tree_force;
    w.tokens_per_tile = way / 2 * tokens;
    w.rows_per_tile = (w.max_nodes < w.tokens_per_tile ? w.max_nodes : w.tokens_per_tile) * G;      // of a part
    w.whole = way % 2 == 0;
    w.min_units = w.whole ? 1 : 2;
}

static bool tree_plain_whole(const TreeWork& w, int max_context) { return tree_tiles(w, max_context, TP_KEYS) <= 2; }

template <typename T, int DP, int R>
static int tree_plain_go(const void* q, long long q_stride, void* out, long long out_stride, const void* k, const void* v,
                         int n_pages, int page_size, const int* tables, int max_blocks, const void* seen, int dh, float scale,
                         TreeWork w, int max_context, float* work, cudaStream_t stream) {
    constexpr int ROWS = 16 * R;
    constexpr size_t smem = (size_t)((ROWS + 2 * TP_KEYS) * (DP + 4) + ROWS * (TP_KEYS + 4)) * sizeof(float);
    // per device: how many of its blocks an SM holds
    static int held[64] = {};
    int dev = 0, shift = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!held[dev]) {
        e = cudaFuncSetAttribute(tree_plain_kernel<T, DP, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        int n = 0;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, tree_plain_kernel<T, DP, R>, TP_THREADS, smem);
        if (e != cudaSuccess) return (int)e;
        held[dev] = n < 1 ? 1 : n > 2 ? 2 : n;
    }
    while ((1 << shift) < page_size) ++shift;
    if ((1 << shift) != page_size) shift = -1;
    w.rows_per_tile = ROWS;
    w.workers = held[dev] * tgo_multiprocessors();
    w.whole = tree_plain_whole(w, max_context);
    if (w.whole) w.min_units = 1;
    else if (!work) return TREE_E_WORK;
    int rc = tgo_launch_pdl(tree_plain_kernel<T, DP, R>, dim3(w.workers), dim3(TP_THREADS), smem, stream, (const T*)q, q_stride, (T*)out,
                            out_stride, (const T*)k, (const T*)v, n_pages, page_size, shift, tables, max_blocks,
                            (const unsigned long long*)seen, dh, scale, w, work, tree_ml(work, w, dh), tree_notes(work, w, dh));
    if (rc) return rc;
    return tree_join_go<T>(out, out_stride, dh, w, work, tree_ml(work, w, dh), tree_notes(work, w, dh), stream);
}

// Floats of workspace that a call of these sizes wants: none where items stay whole. max_context -1: that any call wants.
TGO_API int tgo_attention_tree_work(int dtype, int B, int H, int Hkv, int dh, int page_size, int window, int max_nodes, int max_context) {
    if (B <= 0 || Hkv <= 0 || H % Hkv || max_nodes <= 0) return 0;
    const int sms = tgo_multiprocessors(), G = H / Hkv;
    const bool tc = dtype == TGO_BF16 && tgo_attention_tree_tc_supports(dh, G, page_size);
    if (max_context >= 0) {
        TreeWork w = {nullptr, nullptr, B, 0, H, Hkv, window, max_nodes, 0, 0, 0, 2, sms, 0};
        if (tc) tree_choose(w, max_context, G, sms);
        else w.whole = tree_plain_whole(w, max_context);
        if (w.whole) return 0;
    }
    int rows = 2 * 64;                        // two blocks an SM with 64 rows a tile
    if (tc) {
        const int mine = max_nodes * G < 2 * TT_ROWS ? max_nodes * G : 2 * TT_ROWS;
        rows = mine > rows ? mine : rows;
    }
    return sms * 2 * rows * ((dh + 3) / 4 * 4 + 2) + 2 * sms * (int)(sizeof(TreeNote) / sizeof(float));
}

// work: tgo_attention_tree_work() floats, or null. TREE_E_WORK, and nothing is done, where it is null and items are cut, as they may be
// although that said none: by the FMA units for want of alignment. scale > 0.
TGO_API int tgo_attention_tree(const void* q, long long q_stride, void* out, long long out_stride, int dtype, int T, const void* k_cache,
                               const void* v_cache, int n_pages, int page_size, const int* block_tables, int max_blocks,
                               const int* context_lens, const int* q_start, const void* seen, int B, int H, int Hkv, int dh,
                               int window, int max_nodes, int max_context, float* work, cudaStream_t stream,
                               float scale) {
    if (B <= 0 || T <= 0 || max_nodes <= 0) return 0;
    if (H <= 0 || Hkv <= 0 || H % Hkv || dh <= 0 || dh > 256 || n_pages <= 0 || page_size <= 0 || max_blocks <= 0 || window < 0 ||
        max_nodes > TREE_NODES || (long long)max_blocks * page_size > 0x7fffff00ll || (dtype != TGO_F32 && dtype != TGO_BF16) || !(scale > 0.f))
        return TGO_E_BAD_ARG;
    const int sms = tgo_multiprocessors(), G = H / Hkv;
    const long long rows = (long long)n_pages * Hkv * page_size;
    TreeWork w = {context_lens, q_start, B, T, H, Hkv, window, max_nodes, max_blocks * page_size, 0, 0, 2, 0, 0};
    // units are counted in 32 bits
    if ((double)B * Hkv * ((double)max_nodes * G / 16 + 1) * ((double)max_blocks * page_size / TP_KEYS + 2 + TREE_OVERHEAD) > 2e9) return TGO_E_BAD_ARG;
    if (dtype == TGO_BF16 && tree_force != 1 && tgo_attention_tree_tc_supports(dh, G, page_size) && q_stride % 8 == 0 &&
        q_stride >= (long long)H * dh && out_stride % 8 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0 &&
        (uintptr_t)k_cache % 128 == 0 && (uintptr_t)v_cache % 128 == 0 &&
        rows + page_size <= 0x7fffffffll) {
        w.workers = sms;
        tree_choose(w, max_context, G, sms);
        if (!w.whole && !work) return TREE_E_WORK;
        const bool two = w.tokens_per_tile > TT_ROWS / G;
        CUtensorMap mk, mv, mq;
        if (!tg_map(&mk, k_cache, rows, dh, dh, page_size) || !tg_map(&mv, v_cache, rows, dh, dh, page_size) ||
            !tree_map_q(&mq, q, q_stride, T, H, G, dh))
            return TGO_E_BAD_ARG;
#define TT_GO(DH, RT) return tree_tc_go<DH, RT>(mk, mv, mq, v_cache, n_pages, out, out_stride, page_size, block_tables, max_blocks, seen, scale, w, work, stream)
        if (dh == 128) { if (two) TT_GO(128, 2); TT_GO(128, 1); }
        if (two) TT_GO(64, 2);
        TT_GO(64, 1);
#undef TT_GO
    }
#define TP_GO(T, DP, R) return tree_plain_go<T, DP, R>(q, q_stride, out, out_stride, k_cache, v_cache, n_pages, page_size, block_tables, \
                                                       max_blocks, seen, dh, scale, w, max_context, work, stream)
    if (dtype == TGO_F32) {
        // as many rows a thread as the widest tree fills
        const int rows = max_nodes * G;
        if (dh <= 64) { if (rows <= 16) TP_GO(float, 64, 1); if (rows <= 32) TP_GO(float, 64, 2); TP_GO(float, 64, 4); }
        if (dh <= 128) { if (rows <= 16) TP_GO(float, 128, 1); if (rows <= 32) TP_GO(float, 128, 2); TP_GO(float, 128, 4); }
        if (rows <= 16) TP_GO(float, 256, 1);
        TP_GO(float, 256, 2);
    }
    if (dh <= 64) TP_GO(bf16, 64, 2);
    if (dh <= 128) TP_GO(bf16, 128, 2);
    TP_GO(bf16, 256, 2);
#undef TP_GO
}
