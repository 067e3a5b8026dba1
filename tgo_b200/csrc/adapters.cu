// Low-rank adapters of many requests beside a shared projection.
//
// Row t of a batch with adapter i = ids[t]:
//   u[t, s, j] = scale_i sum_k x[t, k] A_i[s, j, k],    out[t, n] = y[t, n] + sum_j u[t, s(n), j] B_i[n, j],
// y being the projection's own result and s(n) the slice of its columns that n lies in (q, k and v of a
// joined matrix; gate and up rows in eights): each slice has an A of its own. A row whose id names no
// adapter keeps y. u is held in 32 bits.
#include "mma_sync.cuh"
#include "tcgen.cuh"

#define LR_MAX_SLICES 4

struct LowRankColumns {
    int ends[LR_MAX_SLICES];      // the column after each slice's last
    int slices;
    int interleaved;              // eight columns of slice 0, eight of slice 1, and so on
};

// Four values of u as the second product takes them: each rounded to bfloat16, what that left out rounded too, and, where y
// is float32, what that left out. All parts but the last stay finite: the largest bfloat16 number stands for a value that would round
// to infinity, and an infinity is left for the last part.
template <bool LAST> __device__ __forceinline__ uint2 lr_round(float4& v) {      // v gets what is left out
    if constexpr (LAST) return make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    uint2 r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r.x) : "f"(v.y), "f"(v.x));
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r.y) : "f"(v.w), "f"(v.z));
    v = make_float4(v.x - __uint_as_float(r.x << 16), v.y - __uint_as_float(r.x & 0xffff0000u),
                    v.z - __uint_as_float(r.y << 16), v.w - __uint_as_float(r.y & 0xffff0000u));
    return r;
}
// Parts of u: 2^-17 of it is lost with two (a bfloat16 y's own rounding is 2^-9), 2^-25 with three.
template <typename TY> struct LowRankParts { static constexpr int N = sizeof(TY) == 4 ? 3 : 2; };

__device__ __forceinline__ int lr_slice(const LowRankColumns& c, int n) {
    if (c.interleaved) return (n >> 3) & 1;
    int s = 0;
#pragma unroll
    for (int i = 0; i < LR_MAX_SLICES - 1; ++i) s += (i + 1 < c.slices && n >= c.ends[i]);
    return s;
}

struct LowRank {
    const void *x, *y, *a, *b;
    void* out;
    long long x_stride, y_stride, out_stride;
    const float* scale;
    const int* ids;
    int T, K, N, adapters, rank;
    LowRankColumns columns;
};

// ------------------------------------------------------------------------- the rows of an adapter
// For many rows: which rows have which adapter, in tiles of up to `tile` rows of one adapter (rows without
// one come last, as tiles of adapter -1). perm: the rows by tile; info: the number of tiles, of those with an adapter, and the first
// place in perm of a row without; a tile is (adapter, first place in perm, rows). One block; a warp has a run of rows. With up to 255 adapters each warp
// counts for itself, and an adapter's rows keep their order: the rows of a request then lie together, and a tile of them
// can be fetched as one box. With more, rows take their places as they come, 32 at a time in order.
#define LP_INFO 3
#define LP_THREADS 1024
#define LP_WARPS (LP_THREADS / 32)
#define LP_MAX_ADAPTERS 3071
#define LP_ORDERED 255
#define LP_HELD 8                 // rows a thread holds; more are read twice
static_assert((LP_WARPS + 2) * (LP_ORDERED + 1) <= 3 * (LP_MAX_ADAPTERS + 1), "the plan's shared memory");

// Rows that the kernels after the plan read, for the blocks after the first to ask for into L2 while the first plans and u,
// which does not fill the memory's time, is made: the first `many` of each matrix, x before y. MEASURED (us, without, 32 MB, 64
// MB, 96 MB): 1833 rows, rank 32, gate and up of 12288 53.0, 50.8, 51.3, 51.6; 8192 rows, rank 64, q, k and v 68.8, 67.1, 66.9, 67.5.
#define LP_AHEAD 48000000
#define LP_PIECE 4096             // bytes asked for at once, at most
struct LowRankAhead {
    const char* from[2];
    long long stride[2];          // bytes
    int bytes[2], many[2];        // of a row; rows
    int all;                      // rows without an adapter, too
};

__global__ void __launch_bounds__(LP_THREADS)
low_rank_plan_kernel(const int* __restrict__ ids, int T, int adapters, int tile, int* __restrict__ perm, int* __restrict__ info,
                     int* __restrict__ tiles, const LowRankAhead ahead) {
    __shared__ int pool[3 * (LP_MAX_ADAPTERS + 1)];
    __shared__ int warp_rows[LP_WARPS], warp_tiles[LP_WARPS];
    pdl_wait();
    pdl_launch_late();                                       // the next kernel's blocks may come and wait: 0.8 us
    if (blockIdx.x > 0) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int pieces = (ahead.bytes[m] + LP_PIECE - 1) / LP_PIECE;
            for (int e = threadIdx.x * (gridDim.x - 1) + blockIdx.x - 1; e < ahead.many[m] * pieces; e += (gridDim.x - 1) * LP_THREADS) {
                const int r = e / pieces, at = (e - r * pieces) * LP_PIECE, id = ids[r];
                if (ahead.all || (id >= 0 && id < adapters))
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(ahead.from[m] + r * ahead.stride[m] + at),
                                 "r"(min(LP_PIECE, ahead.bytes[m] - at)));
            }
        }
        return;
    }
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, slots = adapters + 1;
    const bool ordered = adapters <= LP_ORDERED;
    int* const rows_before = pool;
    int* const tiles_before = rows_before + slots;
    int* const counts = tiles_before + slots;                // [warp][adapter], or [adapter] alone
    const int run = (T + LP_THREADS - 1) / LP_THREADS * 32, from = min(warp * run, T), to = min(from + run, T);
    int held[LP_HELD];
    auto slot_of = [&](int r) {                              // -1: no row
        const int id = r < to ? ids[r] : 0;
        return r >= to ? -1 : id >= 0 && id < adapters ? id : adapters;
    };
#pragma unroll
    for (int i = 0; i < LP_HELD; ++i) held[i] = slot_of(from + i * 32 + lane);
    for (int i = t; i < (ordered ? LP_WARPS * slots : slots); i += LP_THREADS) counts[i] = 0;
    __syncthreads();
    int* const mine = ordered ? counts + warp * slots : counts;
    auto each = [&](auto&& take) {                           // 32 rows of the run at a time
#pragma unroll
        for (int i = 0; i < LP_HELD; ++i)
            if (from + i * 32 < to) take(from + i * 32 + lane, held[i]);
        for (int base = from + LP_HELD * 32; base < to; base += 32) take(base + lane, slot_of(base + lane));
    };
    // the lanes with a lane's adapter; a request's rows lie together: mostly all of them
    auto alike = [&](int slot) {
        return __all_sync(0xffffffffu, slot == __shfl_sync(0xffffffffu, slot, 0)) ? 0xffffffffu : __match_any_sync(0xffffffffu, slot);
    };
    // a run of one adapter alone needs no looking at its parts
    const int lead = __shfl_sync(0xffffffffu, held[0], 0);
    bool one = run <= LP_HELD * 32 && from < to;
#pragma unroll
    for (int i = 0; i < LP_HELD; ++i) one = one && (held[i] == lead || held[i] < 0);
    one = __all_sync(0xffffffffu, one);
    if (one) {
        if (lane == 0) {
            if (ordered) mine[lead] = to - from;
            else atomicAdd(&mine[lead], to - from);
        }
    } else each([&](int, int slot) {
        const unsigned same = alike(slot);
        if (slot >= 0 && lane == __ffs(same) - 1) {
            if (ordered) mine[slot] += __popc(same);
            else atomicAdd(&mine[slot], __popc(same));
        }
        __syncwarp();
    });
    __syncthreads();
    // a warp's rows of an adapter come after the earlier warps'
    if (ordered) {
        for (int i = warp; i < slots; i += LP_WARPS) {
            const int c = counts[lane * slots + i];
            int n = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += a;
            }
            counts[lane * slots + i] = n - c;
            if (lane == 31) rows_before[i] = n;
        }
        __syncthreads();
    }
    // exclusive sums of rows and of tiles over the adapters, a thread a run of neighbours
    const int per = (slots + LP_THREADS - 1) / LP_THREADS, first = min(t * per, slots), last = min(first + per, slots);
    int my_rows = 0, my_tiles = 0;
    for (int i = first; i < last; ++i) {
        if (!ordered) {
            rows_before[i] = counts[i];
            counts[i] = 0;
        }
        my_rows += rows_before[i];
        my_tiles += (rows_before[i] + tile - 1) / tile;
    }
    int sum_rows = my_rows, sum_tiles = my_tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, sum_rows, o), b = __shfl_up_sync(0xffffffffu, sum_tiles, o);
        if (lane >= o) { sum_rows += a; sum_tiles += b; }
    }
    if (lane == 31) { warp_rows[warp] = sum_rows; warp_tiles[warp] = sum_tiles; }
    __syncthreads();
    int at_row = sum_rows - my_rows, at_tile = sum_tiles - my_tiles, total = 0;
    {
        const int a = warp_rows[lane], b = warp_tiles[lane];
        at_row += __reduce_add_sync(0xffffffffu, lane < warp ? a : 0);
        at_tile += __reduce_add_sync(0xffffffffu, lane < warp ? b : 0);
        total = __reduce_add_sync(0xffffffffu, b);
    }
    for (int i = first; i < last; ++i) {
        const int n = rows_before[i];
        rows_before[i] = at_row;
        tiles_before[i] = at_tile;
        at_row += n;
        at_tile += (n + tile - 1) / tile;
    }
    __syncthreads();
    if (t == 0) {
        info[0] = total;
        info[1] = tiles_before[adapters];
        info[2] = rows_before[adapters];
    }
    for (int q = t; q < total; q += LP_THREADS) {
        int lo = 0, hi = slots - 1;                          // the last adapter whose tiles begin at q or before
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (tiles_before[mid] <= q) lo = mid; else hi = mid - 1;
        }
        const int begin = rows_before[lo] + (q - tiles_before[lo]) * tile;
        const int end = lo + 1 < slots ? rows_before[lo + 1] : T;
        tiles[3 * q] = lo < adapters ? lo : -1;
        tiles[3 * q + 1] = begin;
        tiles[3 * q + 2] = min(tile, end - begin);
    }
    if (one) {
        int place = 0;
        if (lane == 0) place = ordered ? mine[lead] : atomicAdd(&mine[lead], to - from);
        place = rows_before[lead] + __shfl_sync(0xffffffffu, place, 0);
        for (int r = lane; r < to - from; r += 32) perm[place + r] = from + r;
    } else each([&](int r, int slot) {
        const unsigned same = alike(slot);
        const int leader = __ffs(same) - 1;
        int place = 0;
        if (slot >= 0 && lane == leader) {
            if (ordered) { place = mine[slot]; mine[slot] = place + __popc(same); }
            else place = atomicAdd(&mine[slot], __popc(same));
        }
        place = __shfl_sync(0xffffffffu, place, leader);
        if (slot >= 0) perm[rows_before[slot] + place + __popc(same & ((1u << lane) - 1))] = r;
        __syncwarp();
    });
}

// ---------------------------------------------------------------------- few rows of an adapter
// A cluster of eight blocks takes up to eight rows of one adapter. Each block forms u over an eighth of k,
// the blocks read each other's sums from shared memory, and each then makes an eighth of the columns: one
// launch, and every number of A and B is read once for eight rows. Bound by the adapters' way from memory or
// L2 when many rows have one each, by latency for a handful. MEASURED (us, clusters of 4, 8, 16): one row, rank 16, 2048 x 2048
// 5.1, 4.1, 4.4; 96 rows of 24 adapters, rank 16, q, k and v of width 4096 12.5, 10.0, 18.0; 347 float32 rows of three adapters,
// rank 8, q, k and v of width 2048 12.4, 10.6, 19.1.
//
// bfloat16: the adapter's rows are the 16 rows of mma.sync products, the batch's rows their 8 columns, both
// straight from memory into the operands' registers: which 16 values of k meet in a product does not
// matter as long as both sides agree, so a thread takes eight neighbouring ones (16 bytes). For the second
// product u is two bfloat16 numbers, its value rounded and the rest rounded, or three where y is float32.
// float32: plain sums, a warp four values of u for all eight rows, its lanes over k; u's and the result's
// order of additions depends on K and the rank alone, whatever the batch.
//
// Without a plan (up to 512 rows and 255 adapters) each cluster finds its rows by itself: a thread a row counts the rows of the
// same adapter before it, every eighth begins a group, and the cluster takes the group of its number. Under a microsecond,
// where a plan of its own takes four. (A single row has nothing to look for: 4.2 us, 4.5 with it.)
#define LF_ROWS 8
#define LF_CTAS 8
#define LF_THREADS 256
#define LF_WARPS (LF_THREADS / 32)
#define LF_PASS 64                // values of u a pass, bfloat16
#define LF_TILES 2                // tiles of 16 columns a warp has under way, bfloat16
#define LR_SCAN_TURNS 2           // rows a thread looks at
#define LR_SCAN_ROWS (LR_SCAN_TURNS * LF_THREADS)
#define LR_SCAN_ADAPTERS 255      // their counts' places, and one for none
static_assert(LR_SCAN_ADAPTERS + 1 == LF_THREADS && LR_SCAN_TURNS * LF_WARPS == 16, "sixteen counts of 32 rows a thread's adapter");
static_assert(LF_ROWS == LF_WARPS, "a warp a row");

__device__ __forceinline__ void lf_cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void lf_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ float4 lf_peer(const float* mine, int rank) {
    float4 v;
    asm volatile("{\n\t.reg .u32 p;\n\tmapa.shared::cluster.u32 p, %4, %5;\n\t"
                 "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [p];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(smem_u32(mine)), "r"(rank) : "memory");
    return v;
}

// Floats of shared memory: u of all blocks [8][width + 4], this block's [8][width], then partial sums
// [8 warps][64][8], later u's third parts [8][width / 2 + 4] (bfloat16), or the block's part of x [8][k] (float32).
template <typename T> static inline long long lf_floats(int width, int K) {
    const long long third = (long long)LF_ROWS * (width / 2 + 4), sums = LF_WARPS * LF_PASS * LF_ROWS;
    const long long tail = sizeof(T) == 2 ? (third > sums ? third : sums) : (long long)LF_ROWS * ((((K + LF_CTAS - 1) / LF_CTAS) + 3) / 4 * 4);
    return (long long)LF_ROWS * (2 * width + 4) + tail;
}

template <typename T, typename TY>
__global__ void __launch_bounds__(LF_THREADS, 3)
low_rank_few_kernel(const LowRank p, const int* __restrict__ perm, const int* __restrict__ info, const int* __restrict__ tiles) {
    extern __shared__ __align__(16) float lf_smem[];
    __shared__ int rows[LF_ROWS];
    __shared__ __align__(16) unsigned char counts[LF_THREADS][LR_SCAN_TURNS * LF_WARPS];
    __shared__ int warp_count[LR_SCAN_TURNS * LF_WARPS], group[2];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int item = blockIdx.x / LF_CTAS, cta = blockIdx.x % LF_CTAS;
    pdl_wait();
    int id, n;
    if (tiles) {
        if (item >= info[0]) return;
        id = tiles[3 * item];
        n = tiles[3 * item + 2];
        if (t < n) rows[t] = perm[tiles[3 * item + 1] + t];
        __syncthreads();
    } else if (p.T == 1) {
        id = p.ids[0];
        n = 1;
        if (t == 0) rows[0] = 0;
        __syncthreads();
    } else {
        // LR_SCAN_TURNS rows a thread: which adapter, how many rows of it before (counted by the 32 rows of a warp), and
        // whether it begins a group
        int mine[LR_SCAN_TURNS], before[LR_SCAN_TURNS], all = 0;
        unsigned who[LR_SCAN_TURNS];
        *(uint4*)counts[t] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < LR_SCAN_TURNS; ++h) {
            const int r = h * LF_THREADS + t;
            mine[h] = r < p.T ? p.ids[r] : -2;
            if (r < p.T && (mine[h] < 0 || mine[h] >= p.adapters)) mine[h] = -1;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < LR_SCAN_TURNS; ++h) {
            const unsigned same = __match_any_sync(0xffffffffu, mine[h]);
            before[h] = __popc(same & ((1u << lane) - 1));
            if (mine[h] >= -1 && before[h] == 0) counts[mine[h] & 255][h * LF_WARPS + warp] = (unsigned char)__popc(same);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < LR_SCAN_TURNS; ++h) {
            const uint4 q = *(const uint4*)counts[mine[h] & 255];
            const unsigned word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = h * LF_WARPS + warp - 4 * i;   // bytes of it that count
                before[h] = (int)__dp4a(k >= 4 ? word[i] : k > 0 ? word[i] & ((1u << 8 * k) - 1) : 0u, 0x01010101u, (unsigned)before[h]);
            }
            who[h] = __ballot_sync(0xffffffffu, mine[h] >= -1 && before[h] % LF_ROWS == 0);
            if (lane == 0) warp_count[h * LF_WARPS + warp] = __popc(who[h]);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < LR_SCAN_TURNS; ++h) {
            int place = __popc(who[h] & ((1u << lane) - 1)) + all;
#pragma unroll
            for (int w = 0; w < LF_WARPS; ++w) {
                place += w < warp ? warp_count[h * LF_WARPS + w] : 0;
                all += warp_count[h * LF_WARPS + w];
            }
            if ((who[h] >> lane & 1) && place == item) { group[0] = mine[h]; group[1] = before[h]; }
        }
        if (item >= all) return;
        __syncthreads();
        id = group[0];
        n = 0;
#pragma unroll
        for (int h = 0; h < LR_SCAN_TURNS; ++h) {
            const bool in = mine[h] == id && before[h] >= group[1] && before[h] < group[1] + LF_ROWS;
            if (in) rows[before[h] - group[1]] = h * LF_THREADS + t;
            n += __syncthreads_count(in);
        }
    }
    const TY* const y = (const TY*)p.y;
    TY* const out = (TY*)p.out;
    const int pairs = (p.N + 31) / 32, col0 = min((pairs * cta / LF_CTAS) * 32, p.N), col1 = min((pairs * (cta + 1) / LF_CTAS) * 32, p.N);
    if (id < 0 || id >= p.adapters) {                        // no adapter: y as it is
        if (p.out != p.y && warp < n) {
            const TY* const from = y + (size_t)rows[warp] * p.y_stride;
            TY* const to = out + (size_t)rows[warp] * p.out_stride;
            for (int c = col0 + lane; c < col1; c += 8 * 32) {
                TY v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i * 32 < col1) v[i] = from[c + i * 32];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + i * 32 < col1) to[c + i * 32] = v[i];
            }
        }
        return;
    }
    const int rank = p.rank, width = p.columns.slices * rank, K = p.K;
    const T* const a = (const T*)p.a + (size_t)id * width * K;
    const T* const b = (const T*)p.b + (size_t)id * p.N * rank;
    float* const u = lf_smem;                                // [8][width + 4]
    float* const part = u + LF_ROWS * (width + 4);           // [8][width]
    float* const tail = part + LF_ROWS * width;
    {   // B's rows and y, which are read last, are asked for now
        const char* const from = (const char*)(b + (size_t)col0 * rank);
        const int bytes = (col1 - col0) * rank * (int)sizeof(T);
        for (int o = t * 128; o < bytes; o += LF_THREADS * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + o));
    }

    if constexpr (sizeof(T) == 2) {
        const int g = lane >> 2, tig = lane & 3, blocks = (K + 31) / 32;
        const bf16* const x = (const bf16*)p.x + (size_t)rows[g < n ? g : 0] * p.x_stride;
        float* const red = tail;                             // [warp][value of u][row]
        for (int j0 = 0; j0 < width; j0 += LF_PASS) {
            float acc[LF_PASS / 16][4] = {};
#pragma unroll 2
            for (int kb = cta * LF_WARPS + warp; kb < blocks; kb += LF_CTAS * LF_WARPS) {
                const int k = kb * 32 + tig * 8;
                const uint4 zero = make_uint4(0, 0, 0, 0);
                const uint4 xv = g < n && k < K ? *(const uint4*)(x + k) : zero;
#pragma unroll
                for (int m = 0; m < LF_PASS / 16; ++m) {
                    const int j = j0 + m * 16 + g;
                    if (j0 + m * 16 < width) {
                        const uint4 lo = k < K && j < width ? *(const uint4*)(a + (size_t)j * K + k) : zero;
                        const uint4 hi = k < K && j + 8 < width ? *(const uint4*)(a + (size_t)(j + 8) * K + k) : zero;
                        const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
                        mma_bf16(acc[m], a0, xv.x, xv.y);
                        mma_bf16(acc[m], a1, xv.z, xv.w);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < LF_PASS / 16; ++m) {
                float* const to = red + (warp * LF_PASS + m * 16 + g) * LF_ROWS + 2 * tig;
                *(float2*)to = make_float2(acc[m][0], acc[m][1]);
                *(float2*)(to + 8 * LF_ROWS) = make_float2(acc[m][2], acc[m][3]);
            }
            __syncthreads();
            for (int e = t; e < LF_PASS * LF_ROWS; e += LF_THREADS) {
                const int j = j0 + e / LF_ROWS;
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < LF_WARPS; ++w) s += red[w * LF_PASS * LF_ROWS + e];
                if (j < width) part[(e % LF_ROWS) * width + j] = s;
            }
            __syncthreads();
        }
    } else {
        // x in shared memory, a warp a row. Three blocks a multiprocessor are asked for: 347 rows of three adapters, width
        // 2048, 2048 + 512 + 512 columns, rank 8 14.0 us, with two 18.8 (10.6 since the clusters find their rows).
        const int kc = ((K + LF_CTAS - 1) / LF_CTAS + 3) / 4 * 4, k0 = min(cta * kc, K), k1 = min(k0 + kc, K);
        float* const xs = tail;                              // [row][k of the block]
#pragma unroll 4
        for (int k = lane * 4; k < k1 - k0; k += 128)
            *(float4*)(xs + warp * kc + k) = warp < n ? *(const float4*)((const float*)p.x + (size_t)rows[warp] * p.x_stride + k0 + k)
                                                      : make_float4(0.f, 0.f, 0.f, 0.f);
        __syncthreads();
        for (int j0 = warp * 4; j0 < width; j0 += 4 * LF_WARPS) {
            float v[4 * LF_ROWS] = {};
            for (int k = lane * 4; k < k1 - k0; k += 128) {
                float4 w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    w[j] = j0 + j < width ? *(const float4*)((const float*)a + (size_t)(j0 + j) * K + k0 + k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int r = 0; r < LF_ROWS; ++r) {
                    const float4 q = *(const float4*)(xs + r * kc + k);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j * LF_ROWS + r] = fmaf(q.w, w[j].w, fmaf(q.z, w[j].z, fmaf(q.y, w[j].y, fmaf(q.x, w[j].x, v[j * LF_ROWS + r]))));
                }
            }
            // 32 sums over the lanes: each step halves the sums a lane has, after five lane l has sum l
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < o; ++i) {
                    const float give = lane & o ? v[i] : v[i + o], keep = lane & o ? v[i + o] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
            if (j0 + lane / LF_ROWS < width) part[(lane % LF_ROWS) * width + j0 + lane / LF_ROWS] = v[0];
        }
    }
    lf_cluster_arrive();
    lf_cluster_wait();
    const float scale = p.scale[id];
    for (int e = t * 4; e < LF_ROWS * width; e += LF_THREADS * 4) {
        float4 s = lf_peer(part + e, 0);
#pragma unroll
        for (int r = 1; r < LF_CTAS; ++r) {
            const float4 q = lf_peer(part + e, r);
            s.x += q.x; s.y += q.y; s.z += q.z; s.w += q.w;
        }
        s = make_float4(s.x * scale, s.y * scale, s.z * scale, s.w * scale);
        float* const to = u + (e / width) * (width + 4) + e % width;
        if constexpr (sizeof(T) == 2) {
            const uint2 first = lr_round<false>(s), second = lr_round<LowRankParts<TY>::N == 2>(s);
            *(uint4*)to = make_uint4(first.x, first.y, second.x, second.y);
            if constexpr (LowRankParts<TY>::N == 3) *(uint2*)(tail + (e / width) * (width / 2 + 4) + e % width / 2) = lr_round<true>(s);
        } else *(float4*)to = s;
    }
    lf_cluster_arrive();                                     // waited for at the end: a peer may still be reading `part`
    __syncthreads();

    if constexpr (sizeof(T) == 2) {
        const int g = lane >> 2, tig = lane & 3;
        const int r0 = 2 * tig < n ? rows[2 * tig] : -1, r1 = 2 * tig + 1 < n ? rows[2 * tig + 1] : -1;
        // LF_TILES tiles of 16 columns at a time: what is read of y and B is under way before the first is made (out may be
        // y, so no load passes a store by itself). MEASURED: 96 rows of 24 adapters, width 4096, 6144 columns, rank 16: one at a time 12.7 us, two 11.6,
        // four 12.6: the code is run once, and its fetching shows.
        const int far = p.columns.interleaved ? 16 : 8;      // columns from a product's row g to row g + 8
#pragma unroll 1
        for (int q0 = col0 / 16 + warp; q0 < col1 / 16; q0 += LF_TILES * LF_WARPS) {
            int c[LF_TILES], at_u[LF_TILES], at_third[LF_TILES];
            TY v[LF_TILES][4];
            float acc[LF_TILES][4] = {};
#pragma unroll
            for (int i = 0; i < LF_TILES; ++i) {
                const int q = min(q0 + i * LF_WARPS, col1 / 16 - 1);     // past the end: the last one, and not stored
                c[i] = p.columns.interleaved ? q / 2 * 32 + (q & 1) * 8 + g : q * 16 + g;
                const int first = (p.columns.interleaved ? q & 1 : lr_slice(p.columns, q * 16)) * rank;
                at_u[i] = g * (width + 4) + first;
                at_third[i] = g * (width / 2 + 4) + first / 2;
                const TY* const ya = y + (size_t)max(r0, 0) * p.y_stride + c[i];
                const TY* const yb = y + (size_t)max(r1, 0) * p.y_stride + c[i];
                if (r0 >= 0) { v[i][0] = ya[0]; v[i][2] = ya[far]; }
                if (r1 >= 0) { v[i][1] = yb[0]; v[i][3] = yb[far]; }
            }
#pragma unroll 1
            for (int k = 4 * tig; k - 4 * tig < rank; k += 16) {
                uint2 lo[LF_TILES], hi[LF_TILES];
#pragma unroll
                for (int i = 0; i < LF_TILES; ++i) {
                    lo[i] = hi[i] = make_uint2(0, 0);
                    if (k < rank) {
                        lo[i] = *(const uint2*)(b + (size_t)c[i] * rank + k);
                        hi[i] = *(const uint2*)(b + (size_t)(c[i] + far) * rank + k);
                    }
                }
#pragma unroll
                for (int i = 0; i < LF_TILES; ++i) {
                    const uint4 f = k < rank ? *(const uint4*)(u + at_u[i] + k) : make_uint4(0, 0, 0, 0);
                    const uint32_t m[4] = {lo[i].x, hi[i].x, lo[i].y, hi[i].y};
                    mma_bf16(acc[i], m, f.x, f.y);
                    mma_bf16(acc[i], m, f.z, f.w);
                    if constexpr (LowRankParts<TY>::N == 3) {
                        const uint2 third = k < rank ? *(const uint2*)(tail + at_third[i] + k / 2) : make_uint2(0, 0);
                        mma_bf16(acc[i], m, third.x, third.y);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < LF_TILES; ++i) {
                if (q0 + i * LF_WARPS >= col1 / 16) break;
                if (r0 >= 0) {
                    out[(size_t)r0 * p.out_stride + c[i]] = from_f32<TY>(to_f32(v[i][0]) + acc[i][0]);
                    out[(size_t)r0 * p.out_stride + c[i] + far] = from_f32<TY>(to_f32(v[i][2]) + acc[i][2]);
                }
                if (r1 >= 0) {
                    out[(size_t)r1 * p.out_stride + c[i]] = from_f32<TY>(to_f32(v[i][1]) + acc[i][1]);
                    out[(size_t)r1 * p.out_stride + c[i] + far] = from_f32<TY>(to_f32(v[i][3]) + acc[i][3]);
                }
            }
        }
    } else {
        for (int c = col0 + t; c < col1; c += LF_THREADS) {
            const float* const w = (const float*)b + (size_t)c * rank;
            const float* const us = u + lr_slice(p.columns, c) * rank;
            float acc[LF_ROWS] = {}, v[LF_ROWS];             // y first: out may be y, and no load passes a store
#pragma unroll
            for (int r = 0; r < LF_ROWS; ++r)
                if (r < n) v[r] = to_f32(y[(size_t)rows[r] * p.y_stride + c]);
#pragma unroll 2
            for (int k = 0; k < rank; k += 4) {
                const float4 q = *(const float4*)(w + k);
#pragma unroll
                for (int r = 0; r < LF_ROWS; ++r) {
                    const float4 f = *(const float4*)(us + r * (width + 4) + k);
                    acc[r] = fmaf(f.w, q.w, fmaf(f.z, q.z, fmaf(f.y, q.y, fmaf(f.x, q.x, acc[r]))));
                }
            }
#pragma unroll
            for (int r = 0; r < LF_ROWS; ++r)
                if (r < n) out[(size_t)rows[r] * p.out_stride + c] = from_f32<TY>(v[r] + acc[r]);
        }
    }
    lf_cluster_wait();
}

// ---------------------------------------------------------------------- many rows of an adapter
// Tiles of 128 planned rows, bfloat16. Two kernels, u between them as two or three bfloat16 numbers a value (see above):
//
// u (`low_rank_u_kernel`): X[rows] A^T on tcgen05, a cluster 64 or 128 rows, a part of k a block: TMA brings 64 columns of
// the rows (one box where they lie together, else four rows a request) and of A into a ring, a thread issues the products.
// Each block sends its sums to the blocks that add them, by rows, through their shared memory; these scale u and split it.
// Bound by x's way into the multiprocessors: 26 of the 66 us of 8192 rows, width 4096, rank 64, q, k and v (calls in a graph; 70
// where the host makes each call).
//
// out (`low_rank_out_kernel`): u and 64 columns of B at a time come by TMA, a thread issues the products into four
// accumulators in turn, eight warps add them to y in shared memory, from where TMA stores it. Bound by y's and out's way:
// 36 of the 66 us, 5.6 TB/s.
#define LT_ROWS 128
#define LT_BK 64
#define LT_STAGES 6               // of the ring, at most 8
#define LT_PASS 256               // columns of u that the blocks of a cluster exchange at a time
#define LT_THREADS 224
#define LT_MAX_WIDTH 512          // slices x rank: the columns of tensor memory

__device__ int low_rank_error_flag = 0;

struct LowRankTile {
    int width, cut, cuts, kbs, splits, stages;    // A's rows come in `cuts` boxes of `cut`; `splits` blocks a cluster
    int rows;                                     // of a cluster: 128, or 64 and two clusters a tile
};
// Bytes of the ring, which later holds a pass of sums.
__host__ __device__ static inline int lt_ring(const LowRankTile& g) {
    // with 64 rows the products read on for 64 more, into whatever lies there
    const int ring = g.stages * (g.rows * LT_BK * 2 + g.cuts * g.cut * LT_BK * 2) + (LT_ROWS - g.rows) * LT_BK * 2;
    const int pass = (g.width < LT_PASS ? (g.width + 31) / 32 * 32 : LT_PASS) * g.rows * 4;
    return ring > pass ? ring : pass;
}

template <int N> struct LtParts { static constexpr int value = N; };

template <int COLS>
__global__ void __launch_bounds__(LT_THREADS)
low_rank_u_kernel(const __grid_constant__ CUtensorMap map_row, const __grid_constant__ CUtensorMap map_some,
                  const __grid_constant__ CUtensorMap map_all, const __grid_constant__ CUtensorMap map_a, const LowRankTile g,
                  int rank, int parts, const float* __restrict__ scale, const int* __restrict__ perm, const int* __restrict__ info,
                  const int* __restrict__ tiles, bf16* __restrict__ u) {
    extern __shared__ unsigned char lt_raw[];
    unsigned char* const base = (unsigned char*)(((uintptr_t)lt_raw + 1023) & ~(uintptr_t)1023);
    const int x_bytes = g.rows * LT_BK * 2, stage_bytes = x_bytes + g.cuts * g.cut * LT_BK * 2;
    uint64_t* const full = (uint64_t*)(base + lt_ring(g));
    uint64_t* const empty = full + 8;
    uint64_t* const done = empty + 8;
    uint64_t* const settled = done + 1;                      // after a wait ran out
    uint32_t* const tmem_slot = (uint32_t*)(settled + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tile = blockIdx.y, split = blockIdx.x % g.splits, skip = blockIdx.x / g.splits * g.rows;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 8; ++i) { tg_init(&full[i], 2); tg_init(&empty[i], 1); }
        tg_init(done, 1);
        tg_init(settled, 1);
        tg_init_done();
    }
    pdl_wait();
    pdl_launch_late();                                       // out's blocks come as these leave: 0.7 us of 64
    const int id = tiles[3 * tile], r0 = tiles[3 * tile + 1] + skip, rows = min(tiles[3 * tile + 2] - skip, g.rows);
    if (tile >= info[0] || id < 0 || rows <= 0) return;      // the same for the whole cluster
    if (warp == 1) tg_alloc<COLS>(tmem_slot);
    tg_before();
    __syncthreads();
    tg_after();
    const uint32_t tmem = *tmem_slot;
    const float by = scale[id];
    const int kb0 = g.kbs * split / g.splits, kb1 = g.kbs * (split + 1) / g.splits;
    bool handed = false;                                     // the sums are there

    if (warp == 0 || warp == 6) {
        // ---- rows (warp 0) and A (warp 6)
        uint32_t it = 0;
        bool ok = true;
        int src[4] = {0, 0, 0, 0}, first = 0;
        bool together = true;
        if (warp == 0) {
            first = perm[r0];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = min(4 * lane + j, rows - 1);
                src[j] = perm[r0 + i];
                together = together && src[j] == first + i;
            }
            together = __all_sync(0xffffffffu, together);
        }
        // three quarters and more come as one box: the rows after the tile's give sums that nobody stores
        const bool whole = together && 4 * rows > 3 * g.rows;
        const int groups = !together ? (rows + 3) / 4 : (rows + 31) / 32, group_bytes = !together ? 512 : 4096;
        int s = 0;
        uint32_t phase = 1;
        if (warp == 6 || whole) {                            // one thread asks for everything
            if (tg_elect()) {
                for (int kb = kb0; kb < kb1; ++kb, ++it) {
                    ok = tg_wait(&empty[s], phase, &low_rank_error_flag, 1);
                    if (!ok) break;
                    unsigned char* const st = base + (size_t)s * stage_bytes;
                    if (warp == 6) {
                        tg_expect(&full[s], (uint32_t)(g.cuts * g.cut * LT_BK * 2));
                        tg_load_2d(st + x_bytes, &map_a, kb * LT_BK, id * g.width, &full[s]);
                        if (g.cuts == 2) tg_load_2d(st + x_bytes + g.cut * LT_BK * 2, &map_a, kb * LT_BK, id * g.width + g.cut, &full[s]);
                    } else {
                        tg_expect(&full[s], (uint32_t)x_bytes);
                        tg_load_2d(st, &map_all, kb * LT_BK, first, &full[s]);
                    }
                    if (++s == g.stages) { s = 0; phase ^= 1; }
                }
                if (!ok) tg_settle_copies(full, g.stages, it, &low_rank_error_flag, 1);
            }
        } else {
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                ok = __all_sync(0xffffffffu, tg_wait(&empty[s], phase, &low_rank_error_flag, 1));
                if (!ok) break;
                unsigned char* const st = base + (size_t)s * stage_bytes;
                if (lane == 0) tg_expect(&full[s], (uint32_t)(groups * group_bytes));
                __syncwarp();
                if (together) {
                    if (lane < groups) tg_load_2d(st + lane * 4096, &map_some, kb * LT_BK, first + 32 * lane, &full[s]);
                } else if (lane < groups) {
                    tg_gather4(st + lane * 512, &map_row, kb * LT_BK, src[0], src[1], src[2], src[3], &full[s]);
                }
                if (++s == g.stages) { s = 0; phase ^= 1; }
            }
            if (!ok) tg_settle_copies(full, g.stages, it, &low_rank_error_flag, 1);
        }
    } else if (warp == 1) {
        if (tg_elect()) {
            const uint32_t idesc = tg_idesc(g.cut);
            int s = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; ++kb) {
                ok = tg_wait(&full[s], phase, &low_rank_error_flag, 2);
                if (!ok) break;
                tg_after();
                unsigned char* const st = base + (size_t)s * stage_bytes;
                const uint64_t dx = tg_desc(st), da = tg_desc(st + x_bytes);
#pragma unroll
                for (int k = 0; k < LT_BK / 16; ++k) tg_mma(tmem, dx + 2 * k, da + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                if (g.cuts == 2) {
                    const uint64_t db = da + (uint64_t)(g.cut * LT_BK * 2 >> 4);
#pragma unroll
                    for (int k = 0; k < LT_BK / 16; ++k) tg_mma(tmem + g.cut, dx + 2 * k, db + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                }
                tg_commit(&empty[s]);
                if (++s == g.stages) { s = 0; phase ^= 1; }
            }
            if (ok) tg_commit(done);
            else tg_settle_products(settled, &low_rank_error_flag, 2);
        }
    } else {
        handed = __all_sync(0xffffffffu, tg_wait(done, 0, &low_rank_error_flag, 3));
    }
    __syncwarp();
    tg_before();
    __syncthreads();
    tg_after();
    // The rings are free: each block of the cluster has an equal share of the rows, and is handed all blocks' sums of
    // those, LT_PASS columns a pass ([block][32 columns][row of the share], a row's 16-byte pieces swapped by its place
    // among eight). It adds them in the blocks' order. Rank by rank the values are filled up to whole sixteens with zeros.
    const int padded = (rank + 15) / 16 * 16, slices = g.width / rank, quads = padded / 4;
    const int share = g.rows / g.splits, blocks = (min(g.width, LT_PASS) + 31) / 32;
    for (int c0 = 0; c0 < g.width; c0 += LT_PASS) {
        const int c1 = min(c0 + LT_PASS, g.width);
        lf_cluster_arrive();
        lf_cluster_wait();
        if (warp >= 2 && warp < 6 && handed && (warp & 3) * 32 < rows) {
            const int quarter = warp & 3;                    // tensor-memory lanes this warp may read
            const int row = quarter * 32 + lane, in = row % share;
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(tg_smem(base) + (uint32_t)(split * blocks * share * 128 + in * 128)), "r"(row / share));
            for (int c = c0; c < c1; c += 32, to += share * 128) {
                uint32_t a[32];
                tg_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, a);
                tg_wait_ld();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + ((q ^ (in & 7)) << 4)), "r"(a[4 * q]), "r"(a[4 * q + 1]),
                                 "r"(a[4 * q + 2]), "r"(a[4 * q + 3]) : "memory");
            }
        }
        lf_cluster_arrive();
        lf_cluster_wait();
        // a lane four values of a slice, a warp a row at a time
        const int s0 = c0 / rank, s1 = (c1 + rank - 1) / rank;   // slices that this pass touches
        auto add = [&](auto blocks_of, auto parts_of) {
            constexpr int BLOCKS = decltype(blocks_of)::value, PARTS = decltype(parts_of)::value;
            for (int e = lane; e < (s1 - s0) * quads; e += 32) {
                const int s = s0 + e / quads, k = e % quads * 4, c = s * rank + k;
                // the zeros behind a slice are written with its last value
                if (k < rank ? c < c0 || c >= c1 : (s + 1) * rank <= c0 || (s + 1) * rank > c1) continue;
                const unsigned char* const from = base + (c - c0) / 32 * (share * 128);
                const int piece = (c - c0) % 32 / 4, step = blocks * share * 128;
                bf16* to = u + ((size_t)(r0 + split * share + warp) * slices + s) * PARTS * padded + k;
#pragma unroll 4
                for (int row = warp; row < min(share, rows - split * share); row += LT_THREADS / 32, to += (size_t)(LT_THREADS / 32) * slices * PARTS * padded) {
                    const unsigned char* const at = from + row * 128 + ((piece ^ (row & 7)) << 4);
                    float4 v = *(const float4*)at;
#pragma unroll
                    for (int i = 1; i < BLOCKS; ++i) {
                        const float4 q = *(const float4*)(at + i * step);
                        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
                    }
                    if (k >= rank) v = make_float4(0.f, 0.f, 0.f, 0.f);     // what lies behind a slice is the next one's
                    v.x *= by; v.y *= by; v.z *= by; v.w *= by;
                    *(uint2*)to = lr_round<false>(v);
                    *(uint2*)(to + padded) = lr_round<PARTS == 2>(v);
                    if constexpr (PARTS == 3) *(uint2*)(to + 2 * padded) = lr_round<true>(v);
                }
            }
        };
        auto add_of = [&](auto parts_of) {
            if (g.splits == 1) add(LtParts<1>(), parts_of);
            else if (g.splits == 2) add(LtParts<2>(), parts_of);
            else if (g.splits == 4) add(LtParts<4>(), parts_of);
            else add(LtParts<8>(), parts_of);
        };
        if (parts == 2) add_of(LtParts<2>());
        else add_of(LtParts<3>());
    }
    tg_before();
    __syncthreads();
    if (warp == 1) {
        tg_after();
        tg_free<COLS>(tmem);
    }
}

// 64 columns a turn. In eights the rows of B that a turn brings, eight of slice 0 and eight of slice 1 in turn,
// are two operands of 32 rows whose groups of eight lie twice as far apart: nothing is moved.
//
// y and out go through shared memory, asynchronously: each of eight warps has 32 rows (the ones whose sums it can read
// from tensor memory, a lane a row) of every other turn and a ring of its own of 32 x 64 tiles; it adds the sums where
// y lies and has the tile stored from there. Rows that lie together are one box either way; others come four at a time and are written by
// the warp, as are part tiles. As many blocks as fit share all tiles' turns out evenly, so that a block's first reads are waited
// for once. MEASURED (the call, us): 1833 rows, rank 32, gate and up of 12288, blocks of eight turns each 63, these 57, with the next
// tile of y asked for before this one is made, not after, 53. Reading y into registers two steps ahead and writing from them, through
// a transposing buffer, took 68 us for 8192 rows of 6144 columns, rank 64, where the kernel takes 36.
#define LO_COLS 64
#define LO_HANDS 8                // warps that hand on; the one after them asks for copies and products
#define LO_THREADS (LO_HANDS * 32 + 32)
#define LO_U_BOX (LT_ROWS * 128)  // bytes of 64 values of k: of 128 rows of u,
#define LO_B_BOX (LO_COLS * 128)  // of a turn's rows of B

__device__ __forceinline__ void lo_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(tg_smem(src)), "r"(x), "r"(y) : "memory");
}
// Operand tile as tg_desc, the groups of eight rows `apart` bytes from each other.
__device__ __forceinline__ uint64_t lo_desc(const void* tile, uint32_t apart) {
    return (tg_desc(tile) & ~((uint64_t)0x3fff << 32)) | ((uint64_t)(apart >> 4) << 32);
}

// BOXES: of 64 values of the rank. PAIRED (rank up to 32, for a float32 y up to 16): all parts of a row share a box.
template <int BOXES, bool PAIRED, bool EIGHTS, typename TY> struct LowRankOut {
    static constexpr int SLICES = EIGHTS ? 2 : 1, PARTS = PAIRED ? 1 : LowRankParts<TY>::N;
    static constexpr int A_BYTES = SLICES * PARTS * BOXES * LO_U_BOX, B_BYTES = BOXES * LO_B_BOX;
    static constexpr int Y_BOXES = (int)sizeof(TY) / 2, Y_BYTES = Y_BOXES * 32 * 128;     // a warp's tile: boxes of 128 bytes a row
    static constexpr int SLOTS = A_BYTES + 2 * B_BYTES + LO_HANDS * 2 * Y_BYTES <= 224 * 1024 ? 2 : 1;
    static constexpr int BYTES = A_BYTES + 2 * B_BYTES + LO_HANDS * SLOTS * Y_BYTES + 512;
    static constexpr int BLOCKS = 2 * (BYTES + 1024) <= 228 * 1024 ? 2 : 1;      // of a multiprocessor
    static_assert(BYTES <= 227 * 1024, "shared memory of a block");
};

template <int BOXES, bool PAIRED, bool EIGHTS, typename TY>
__global__ void __launch_bounds__(LO_THREADS, (LowRankOut<BOXES, PAIRED, EIGHTS, TY>::BLOCKS))
low_rank_out_kernel(const __grid_constant__ CUtensorMap map_u, const __grid_constant__ CUtensorMap map_b,
                    const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_row,
                    const __grid_constant__ CUtensorMap map_out, const LowRank p, const int tile_turns, const int* __restrict__ perm,
                    const int* __restrict__ info, const int* __restrict__ tiles) {
    typedef LowRankOut<BOXES, PAIRED, EIGHTS, TY> L;
    extern __shared__ __align__(1024) unsigned char lo_raw[];
    unsigned char* const a_smem = lo_raw;                    // [slice][part][box][128 rows][128]
    unsigned char* const b_ring = a_smem + L::A_BYTES;       // [2][box][64 columns][128]
    unsigned char* const y_ring = b_ring + 2 * L::B_BYTES;   // [warp][slot][box][32 rows][128]
    uint64_t* const full = (uint64_t*)(y_ring + LO_HANDS * L::SLOTS * L::Y_BYTES);       // [2] B's turn is there
    uint64_t* const u_full = full + 2;
    uint64_t* const acc_full = u_full + 1;                   // [4] a turn's products are done: the accumulator, and B's slot free
    uint64_t* const acc_empty = acc_full + 4;                // [4] the accumulator has been read
    uint64_t* const y_full = acc_empty + 4;                  // [warp][slot]
    uint64_t* const settled = y_full + LO_HANDS * L::SLOTS;         // after a wait ran out
    uint32_t* const tmem_slot = (uint32_t*)(settled + 1);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (t == 0) {
        for (int i = 0; i < 2; ++i) tg_init(&full[i], 1);
        tg_init(u_full, 1);
        for (int i = 0; i < 4; ++i) { tg_init(&acc_full[i], 1); tg_init(&acc_empty[i], 4); }
        for (int i = 0; i < LO_HANDS * L::SLOTS; ++i) tg_init(&y_full[i], 1);
        tg_init(settled, 1);
        tg_init_done();
    }
    __syncthreads();
    pdl_wait();
    // this block's turns: an even share of those of all tiles with an adapter, one after the other
    const int all = info[1] * tile_turns, least = all / (int)gridDim.x, more = all - least * (int)gridDim.x;
    const int begin = blockIdx.x * least + min((int)blockIdx.x, more), turns = least + ((int)blockIdx.x < more);
    // where the w-th turn of a tile lies
    auto columns = [&](int w, int& slice, int& col, int& end) {
        int from = 0;
        slice = 0;
        end = EIGHTS ? p.N : p.columns.ends[0];
        if constexpr (!EIGHTS) {
#pragma unroll
            for (int i = 1; i < LR_MAX_SLICES; ++i) {
                const int n = (end - from + LO_COLS - 1) / LO_COLS;
                if (slice == i - 1 && w >= n) {
                    w -= n;
                    slice = i;
                    from = end;
                    end = p.columns.ends[i];
                }
            }
        }
        col = from + w * LO_COLS;
    };
    TY* const out = (TY*)p.out;
    constexpr int PER = 16 / (int)sizeof(TY);                // columns of a 16-byte piece
    const int steps_all = (p.rank + 15) / 16;
    if (warp == LO_HANDS) {
        struct Turn {
            int row, r0, slice;                              // of B; of u
            bool fresh;                                      // another u than the turn before
        };
        int tile = begin / tile_turns, w = begin - tile * tile_turns, id = 0, r0 = 0, last = 0;
        bool moved = true;
        auto look = [&]() {                                  // the next turn
            Turn q;
            int col, end;
            if (moved) {
                id = tiles[3 * tile];
                r0 = tiles[3 * tile + 1];
            }
            columns(w, q.slice, col, end);
            q.row = id * p.N + col;
            q.r0 = r0;
            q.fresh = moved || q.slice != last;
            last = q.slice;
            moved = ++w == tile_turns;
            if (moved) {
                w = 0;
                ++tile;
            }
            return q;
        };
        auto fetch_u = [&](const Turn& q) {                  // one thread; the rows after the tile's come along: their sums are never stored
            tg_expect(u_full, L::A_BYTES);
#pragma unroll
            for (int i = 0; i < L::SLICES * L::PARTS * BOXES; ++i) {
                const int x = i % BOXES, rest = i / BOXES % L::PARTS, h = i / BOXES / L::PARTS;
                tg_load_2d(a_smem + i * LO_U_BOX, &map_u, ((q.slice + h) * LowRankParts<TY>::N + rest) * steps_all * 16 + x * 64, q.r0, u_full);
            }
        };
        auto fetch = [&](const Turn& q, int s) {             // one thread
            tg_expect(&full[s], L::B_BYTES);
#pragma unroll
            for (int x = 0; x < BOXES; ++x) tg_load_2d(b_ring + s * L::B_BYTES + x * LO_B_BOX, &map_b, x * 64, q.row, &full[s]);
        };
        Turn two[2] = {};                                    // a turn and the next
        if (turns > 0) two[0] = look();
        if (turns > 1) two[1] = look();
        if (lane == 0) {
            if (turns > 0) {
                fetch_u(two[0]);
                fetch(two[0], 0);
            }
            if (turns > 1) fetch(two[1], 1);
        }
        __syncwarp();
        tg_alloc<4 * LO_COLS>(tmem_slot);
        tg_before();
        __syncthreads();
        tg_after();
        const uint32_t tmem = *tmem_slot;
        if (tg_elect()) {
            const uint32_t idesc = tg_idesc(EIGHTS ? LO_COLS / 2 : LO_COLS);
            uint32_t sent = min(turns, 2), u_sent = min(turns, 1);
            bool ok = true;
            for (int i = 0; i < turns; ++i) {
                const int s = i & 1, acc = i & 3;
                const Turn q = s ? two[1] : two[0];
                if (q.fresh) {
                    if (i > 0) {                             // u's place again, once the products before are done
                        ok = tg_wait(&acc_full[(i - 1) & 3], ((i - 1) >> 2) & 1, &low_rank_error_flag, 6);
                        if (!ok) break;
                        fetch_u(q);
                        ++u_sent;
                    }
                    ok = tg_wait(u_full, (u_sent - 1) & 1, &low_rank_error_flag, 4);
                }
                if (ok) ok = tg_wait(&full[s], (i >> 1) & 1, &low_rank_error_flag, 4);
                if (ok) ok = tg_wait(&acc_empty[acc], ((i >> 2) & 1) ^ 1, &low_rank_error_flag, 5);
                if (!ok) break;
                tg_after();
#pragma unroll
                for (int h = 0; h < L::SLICES; ++h) {
                    const uint32_t d = tmem + acc * LO_COLS + h * (LO_COLS / 2);
                    bool first = true;
#pragma unroll
                    for (int x = 0; x < BOXES; ++x) {
                        const unsigned char* const bx = b_ring + s * L::B_BYTES + x * LO_B_BOX + (EIGHTS ? h * 1024 : 0);
                        const uint64_t db = lo_desc(bx, EIGHTS ? 2048 : 1024);
                        const uint64_t da = tg_desc(a_smem + (h * L::PARTS * BOXES + x) * LO_U_BOX);
                        const uint64_t part = PAIRED ? 2 * steps_all : BOXES * (LO_U_BOX >> 4);      // from a part to the next
                        const int steps = min(steps_all - 4 * x, 4);
                        for (int k = 0; k < steps; ++k) {
                            tg_mma(d, da + 2 * k, db + 2 * k, idesc, first ? 0u : 1u);
#pragma unroll
                            for (int r = 1; r < LowRankParts<TY>::N; ++r) tg_mma(d, da + r * part + 2 * k, db + 2 * k, idesc, 1u);
                            first = false;
                        }
                    }
                }
                tg_commit(&acc_full[acc]);
                if (i + 2 < turns) {                         // the slot again, once its products are done
                    const Turn next = look();
                    if (s) two[1] = next;
                    else two[0] = next;
                    ok = tg_wait(&acc_full[acc], (i >> 2) & 1, &low_rank_error_flag, 6);
                    if (!ok) break;
                    fetch(next, s);
                    ++sent;
                }
            }
            if (!ok) {
                tg_settle_copies(full, 2, sent, &low_rank_error_flag, 4);
                tg_settle_copies(u_full, 1, u_sent, &low_rank_error_flag, 4);
                tg_settle_products(settled, &low_rank_error_flag, 6);
            }
        }
        __syncwarp();
    } else {
        // its rows of a tile, from q0 on, none or fewer than 32 perhaps; its turns are set, set + 2, ... of the block's
        const int q0 = (warp & 3) * 32, set = warp >> 2, turns_mine = (turns - set + 1) / 2;
        struct Rows {
            int place, first, count, col, end;               // in perm; in y; columns
            bool together;
        };
        int tile = (begin + set) / tile_turns, w = begin + set - tile * tile_turns, gather[4] = {};
        Rows next = {};
        bool moved = true;
        unsigned char* const ring = y_ring + warp * L::SLOTS * L::Y_BYTES;
        uint64_t* const there = y_full + warp * L::SLOTS;
        auto load = [&](int i) {                             // of this warp's turns; the whole warp
            if (moved) {
                const int r0 = tiles[3 * tile + 1], n = tiles[3 * tile + 2], row = perm[r0 + min(q0 + lane, n - 1)];
                next.place = r0 + q0;
                next.count = min(n - q0, 32);
                next.first = __shfl_sync(0xffffffffu, row, 0);
                next.together = __all_sync(0xffffffffu, lane >= next.count || row == next.first + lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) gather[j] = __shfl_sync(0xffffffffu, row, (4 * lane + j) & 31);
            }
            int slice;
            columns(w, slice, next.col, next.end);
            const int s = i % L::SLOTS;
            if (lane == 0) {
                if (next.count > 0) tg_expect(&there[s], next.together ? L::Y_BYTES : (next.count + 3) / 4 * 4 * 128 * L::Y_BOXES);
                else tg_arrive(&there[s]);
            }
            __syncwarp();
#pragma unroll
            for (int x = 0; x < L::Y_BOXES; ++x) {
                unsigned char* const to = ring + s * L::Y_BYTES + x * 4096;
                if (next.together) {
                    if (lane == 0 && next.count > 0) tg_load_2d(to, &map_y, next.col + x * 32, next.first, &there[s]);
                } else if (4 * lane < next.count) {
                    tg_gather4(to + lane * 512, &map_row, next.col + x * 32, gather[0], gather[1], gather[2], gather[3], &there[s]);
                }
            }
            w += 2;
            moved = w >= tile_turns;
            while (w >= tile_turns) {
                w -= tile_turns;
                ++tile;
            }
        };
        uint32_t sent = 0;
        Rows slots[2] = {};
        for (; sent < min(turns_mine, L::SLOTS); ++sent) {
            load(sent);
            if (sent) slots[1] = next;
            else slots[0] = next;
        }
        auto load_next = [&]() {                             // once what was stored has been read
            if (sent >= turns_mine) return;
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            load(sent);
            if (sent % L::SLOTS) slots[1] = next;
            else slots[0] = next;
            ++sent;
        };
        tg_before();
        __syncthreads();
        tg_after();
        const uint32_t lanes = *tmem_slot + ((uint32_t)q0 << 16);
        bool ok = true;
        for (int i = 0; i < turns_mine && ok; ++i) {
            const int slot = i % L::SLOTS, buf = (2 * i + set) & 3;
            const Rows now = slot ? slots[1] : slots[0];
            const int mine = now.count, c = now.col;
            const uint32_t sums = lanes + buf * LO_COLS;
            ok = __all_sync(0xffffffffu, tg_wait(&acc_full[buf], (i >> 1) & 1, &low_rank_error_flag, 7));
            if (ok) ok = __all_sync(0xffffffffu, tg_wait(&there[slot], (i / L::SLOTS) & 1, &low_rank_error_flag, 8));
            if (!ok) break;
            if (L::SLOTS == 2 && i > 0) load_next();         // where the turn before lay
            tg_after();
            unsigned char* const at = ring + slot * L::Y_BYTES;
            // a row of 128 bytes a lane, its 16-byte pieces swapped by the row's place among eight
#pragma unroll
            for (int v = 0; v < 2 && mine > 0; ++v) {        // 32 columns
                uint32_t acc[32];
                if constexpr (EIGHTS) {                      // 16 of each slice
                    uint32_t a0[16], a1[16];
                    tg_ld16(sums + v * 16, a0);
                    tg_ld16(sums + LO_COLS / 2 + v * 16, a1);
                    tg_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        acc[j / 8 * 16 + j % 8] = a0[j];
                        acc[j / 8 * 16 + 8 + j % 8] = a1[j];
                    }
                } else {
                    tg_ld32(sums + v * 32, acc);
                    tg_wait_ld();
                }
                unsigned char* const line = at + lane * 128 + (L::Y_BOXES == 2 ? v * 4096 : 0);
#pragma unroll
                for (int j = 0; j < 32 / PER; ++j) {
                    uint4* const piece = (uint4*)(line + (((j + (L::Y_BOXES == 1 ? v * 4 : 0)) ^ (lane & 7)) << 4));
                    uint4 w = *piece;
                    uint32_t* const e = (uint32_t*)&w;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (sizeof(TY) == 2)
                            e[k] = pack_bf16(__uint_as_float(e[k] << 16) + __uint_as_float(acc[j * 8 + 2 * k]),
                                             __uint_as_float(e[k] & 0xffff0000u) + __uint_as_float(acc[j * 8 + 2 * k + 1]));
                        else
                            e[k] = __float_as_uint(__uint_as_float(e[k]) + __uint_as_float(acc[j * 4 + k]));
                    }
                    *piece = w;
                }
            }
            tg_before();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tg_arrive(&acc_empty[buf]);
            if (now.together && mine == 32 && c + LO_COLS <= now.end) {
                if (lane == 0) {
#pragma unroll
                    for (int x = 0; x < L::Y_BOXES; ++x) lo_store_2d(&map_out, c + x * 32, now.first, at + x * 4096);
                }
            } else {
#pragma unroll
                for (int x = 0; x < L::Y_BOXES; ++x)
                    for (int r = lane >> 3; r < mine; r += 4) {
                        const int col = c + x * 32 + (lane & 7) * PER, row = now.together ? now.first + r : perm[now.place + r];
                        if (col < now.end)
                            *(uint4*)(out + (size_t)row * p.out_stride + col) = *(const uint4*)(at + x * 4096 + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                    }
            }
            if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");     // with or without a store: a group a turn
            if (L::SLOTS == 1) load_next();
        }
        if (!ok && lane == 0) tg_settle_copies(there, L::SLOTS, sent, &low_rank_error_flag, 8);
        // rows without an adapter: y as it is, 128 vectors of a row a warp and turn
        if (p.out != p.y) {
            const int vectors = p.N / PER, pieces = (vectors + 127) / 128, place = info[2];
            for (long long e = (long long)blockIdx.x * LO_HANDS + warp; e < (long long)(p.T - place) * pieces; e += (long long)gridDim.x * LO_HANDS) {
                const int r = (int)(e / pieces), row = perm[place + r], v = (int)(e - (long long)r * pieces) * 128 + lane;
                const uint4* const from = (const uint4*)((const TY*)p.y + (size_t)row * p.y_stride);
                uint4* const to = (uint4*)(out + (size_t)row * p.out_stride);
                uint4 held[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v + 32 * j < vectors) held[j] = from[v + 32 * j];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v + 32 * j < vectors) to[v + 32 * j] = held[j];
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    tg_before();
    __syncthreads();
    if (warp == LO_HANDS) {
        tg_after();
        tg_free<4 * LO_COLS>(*tmem_slot);
    }
}

// --------------------------------------------------------------------------- any sizes
// A warp a (row, slice, j): lanes go over k, so the sum's order depends on K alone.
template <typename T>
__global__ void __launch_bounds__(256)
low_rank_down_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ a, const float* __restrict__ scale,
                     const int* __restrict__ ids, int adapters, int width, int K, float* __restrict__ u) {
    pdl_wait();
    const int t = blockIdx.x, i = ids[t];
    if (i < 0 || i >= adapters) return;
    const T* const row = x + (size_t)t * x_stride;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int j = blockIdx.y * 8 + warp; j < width; j += 8 * gridDim.y) {
        const T* const col = a + ((size_t)i * width + j) * K;
        float acc = 0.f;
        for (int k = lane; k < K; k += 32) acc = fmaf(to_f32(row[k]), to_f32(col[k]), acc);
        acc = warp_sum(acc);
        if (lane == 0) u[(size_t)t * width + j] = acc * scale[i];
    }
}

// A thread a column.
template <typename T, typename TY>
__global__ void __launch_bounds__(256)
low_rank_up_kernel(const float* __restrict__ u, const T* __restrict__ b, const int* __restrict__ ids, int adapters, int rank,
                   LowRankColumns columns, int N, const TY* y, long long y_stride, TY* out, long long out_stride) {
    pdl_wait();
    const int t = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x, i = ids[t];
    if (n >= N) return;
    float v = to_f32(y[(size_t)t * y_stride + n]);
    if (i < 0 || i >= adapters) {
        if (out != y) out[(size_t)t * out_stride + n] = from_f32<TY>(v);
        return;
    }
    const float* const row = u + ((size_t)t * columns.slices + lr_slice(columns, n)) * rank;
    const T* const col = b + ((size_t)i * N + n) * rank;
    float acc = 0.f;
    for (int j = 0; j < rank; ++j) acc = fmaf(row[j], to_f32(col[j]), acc);
    out[(size_t)t * out_stride + n] = from_f32<TY>(v + acc);
}

// Whether the vectors of the kernels above find their boundaries: rows of x, A and B on 16 bytes, ranks of whole
// vectors, slices of whole products.
template <typename T> static bool lr_vectors(const LowRank& p) {
    const int v = 16 / (int)sizeof(T);
    if (p.K % v || p.x_stride % v || p.rank % 4 || ((uintptr_t)p.x | (uintptr_t)p.a | (uintptr_t)p.b) & 15) return false;
    if (p.columns.interleaved) return p.N % 32 == 0;
    for (int i = 0; i < p.columns.slices; ++i)
        if (p.columns.ends[i] % 16) return false;
    return true;
}

// Whether each cluster of the kernel for few rows finds its rows by itself; a call with more rows or more adapters is planned.
static bool lr_scanned(const LowRank& p) { return p.T <= LR_SCAN_ROWS && p.adapters <= LR_SCAN_ADAPTERS; }
template <typename T> static bool lr_few_takes(const LowRank& p) {
    return lr_vectors<T>(p) && lf_floats<T>(p.columns.slices * p.rank, p.K) * 4 <= 200 * 1024 && p.T <= (1 << 24) &&
           (lr_scanned(p) || p.adapters <= LP_MAX_ADAPTERS);
}

// Tiles there are at most: with an adapter's first row comes one, with every `tile` further ones another.
static long long lr_tiles(const LowRank& p, int tile) {
    const long long adapters = p.T < p.adapters + 1 ? p.T : p.adapters + 1;
    return adapters + (p.T - adapters) / tile;
}

template <typename T, typename TY> static int low_rank_few(const LowRank& p, int* plan, cudaStream_t stream) {
    static bool sized[64] = {};                              // per device
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!sized[dev]) {
        err = cudaFuncSetAttribute(low_rank_few_kernel<T, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (err != cudaSuccess) return (int)err;
        sized[dev] = true;
    }
    const long long items = lr_tiles(p, LF_ROWS);
    int *perm = nullptr, *info = nullptr, *tiles = nullptr;
    if (!lr_scanned(p)) {
        perm = plan;
        info = perm + p.T;
        tiles = info + LP_INFO;
        const int rc = tgo_launch_pdl(low_rank_plan_kernel, dim3(1), dim3(LP_THREADS), 0, stream, p.ids, p.T, p.adapters, LF_ROWS, perm, info, tiles, LowRankAhead{});
        if (rc) return rc;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * LF_CTAS));
    cfg.blockDim = dim3(LF_THREADS);
    cfg.dynamicSmemBytes = (size_t)lf_floats<T>(p.columns.slices * p.rank, p.K) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = LF_CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tgo_pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, low_rank_few_kernel<T, TY>, p, (const int*)perm, (const int*)info, (const int*)tiles);
}

// ---- tiles of 128 rows
// Whether the kernels for many rows take a call: what they read and write on 16 bytes, A's columns in tensor memory.
template <typename TY> static bool lr_tile_takes(const LowRank& p) {
    const int v = 16 / (int)sizeof(TY), width = p.columns.slices * p.rank;
    if (lr_tiles(p, LT_ROWS) > 65535) return false;          // u's grid has a tile a place of its second extent
    if (p.x_stride < p.K || p.y_stride < p.N || p.out_stride < p.N) return false;      // rows over each other (an expanded x)
    if (!lr_vectors<bf16>(p) || p.rank % 8 || p.rank > 128 || width > LT_MAX_WIDTH || p.adapters > LP_MAX_ADAPTERS ||
        p.T > (1 << 24) || (long long)p.adapters * width > 0x7fffffff || (long long)p.adapters * p.N > 0x7fffffff || p.y_stride % v || p.out_stride % v ||
        ((uintptr_t)p.y | (uintptr_t)p.out) & 15)
        return false;
    if (p.columns.interleaved) return p.N % 32 == 0 && (sizeof(TY) == 2 || p.rank <= 64);       // u's parts in shared memory
    for (int i = 0; i < p.columns.slices; ++i)
        if (p.columns.ends[i] % 32) return false;
    return true;
}

static int lt_stage(const LowRankTile& g) { return (g.rows + g.cuts * g.cut) * LT_BK * 2; }
static LowRankTile lt_tile(int width, int K, int rows, int splits) {
    LowRankTile g;
    g.rows = rows;
    g.splits = splits;
    g.width = width;
    g.cuts = width > 256 ? 2 : 1;
    g.cut = ((width + g.cuts - 1) / g.cuts + 15) / 16 * 16;
    g.kbs = (K + LT_BK - 1) / LT_BK;
    const int most = 168 * 1024 / lt_stage(g);
    g.stages = most < LT_STAGES ? most : LT_STAGES;
    return g;
}
static int lt_columns(const LowRankTile& g) {               // of tensor memory
    const int cols = g.cuts * g.cut;
    return cols <= 32 ? 32 : cols <= 64 ? 64 : cols <= 128 ? 128 : cols <= 256 ? 256 : 512;
}
// Shared memory of a block, and no less than its part of the multiprocessor's 228 KB (1 KB a block is the system's) as it has a part of
// the 512 columns: clusters of two calls, on two streams, could otherwise each hold tensor memory on one multiprocessor that the
// other waits for there, and neither would end. (Only the blocks with 512 columns have to be enlarged for it: their clusters ran one block a
// multiprocessor anyway.)
static int lt_bytes(const LowRankTile& g) {
    const int needed = lt_ring(g) + 1024 + 256, part = lt_columns(g) * (228 * 1024 / 512) - 1024;
    return needed > part ? needed : part;
}
// How a tile's u is made: the rows of a cluster and the parts of k, its blocks, that are cheapest by a small model in
// cycles. The blocks run in rounds of as many as the multiprocessors hold. 64 columns cost a block their way into the
// multiprocessor (70 bytes a cycle) or its part of the way of all blocks' rows from memory (3400); to begin and end
// takes 6000, to exchange sums 1500 and a cycle for four. (The tiles that the rows make at least, and one: how many more is
// the device's to know.) MEASURED, all three kernels, us, 1, 2, 4 and 8 parts: 8192 rows, rank 64, q, k and v, clusters of
// 128 rows 74, 67 (taken), 78, 112, of 64 69, 76, 93, 135; 1833 rows, rank 32, gate and up, 128 rows 60, 54, 51, 56, 64 rows
// 60, 53, 51 (taken), 51.
static LowRankTile lr_plan(const LowRank& p) {
    LowRankTile best = {};
    long long least = -1;
    for (int rows = LT_ROWS; rows >= LT_ROWS / 2; rows /= 2)
        for (int s = 1; s <= 8; s *= 2) {
            const LowRankTile g = lt_tile(p.columns.slices * p.rank, p.K, rows, s);
            if (s > 1 && s * 4 > g.kbs) break;
            const int x = rows * LT_BK * 2, stage = lt_stage(g);
            const int slots = tgo_multiprocessors() * (2 * lt_bytes(g) <= 226 * 1024 && g.cuts * g.cut <= 256 ? 2 : 1);
            const long long blocks = ((p.T + LT_ROWS - 1) / LT_ROWS + 1ll) * (LT_ROWS / rows) * s;
            const long long feed = stage / 70, memory = (blocks < slots ? blocks : slots) * x / 3400, each = feed > memory ? feed : memory;
            const long long cost = (blocks + slots - 1) / slots * ((g.kbs + s - 1) / s * each + 6000 + (s > 1 ? 1500 + rows * g.width / 4 : 0));
            if (least < 0 || cost < least) { least = cost; best = g; }
        }
    return best;
}

template <int COLS> static int low_rank_u(const LowRank& p, const LowRankTile& g, int parts, const int* perm, const int* info, const int* tiles, bf16* u,
                                          cudaStream_t stream) {
    static bool sized[64] = {};                              // per device
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!sized[dev]) {
        err = cudaFuncSetAttribute(low_rank_u_kernel<COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (err != cudaSuccess) return (int)err;
        sized[dev] = true;
    }
    CUtensorMap row, some, all, a;
    if (!tg_map(&row, p.x, p.T, p.K, p.x_stride, 1) || !tg_map(&some, p.x, p.T, p.K, p.x_stride, 32) ||
        !tg_map(&all, p.x, p.T, p.K, p.x_stride, g.rows) || !tg_map(&a, p.a, (long long)p.adapters * g.width, p.K, p.K, g.cut))
        return TGO_E_BAD_ARG;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(LT_ROWS / g.rows * g.splits, (unsigned)lr_tiles(p, LT_ROWS));
    cfg.blockDim = dim3(LT_THREADS);
    cfg.dynamicSmemBytes = (size_t)lt_bytes(g);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = g.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tgo_pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, low_rank_u_kernel<COLS>, row, some, all, a, g, p.rank, parts, p.scale, perm, info, tiles, u);
}

template <int BOXES, bool PAIRED, bool EIGHTS, typename TY>
static int low_rank_out(const LowRank& p, const bf16* u, const int* perm, const int* info, const int* tiles, cudaStream_t stream) {
    static bool sized[64] = {};                              // per device
    constexpr int bytes = LowRankOut<BOXES, PAIRED, EIGHTS, TY>::BYTES;
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (!sized[dev]) {
        err = cudaFuncSetAttribute(low_rank_out_kernel<BOXES, PAIRED, EIGHTS, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (err != cudaSuccess) return (int)err;
        sized[dev] = true;
    }
    int turns = 0, begin = 0;                                // of a tile
    for (int i = 0; i < (EIGHTS ? 1 : p.columns.slices); ++i) {
        const int end = EIGHTS ? p.N : p.columns.ends[i];
        turns += (end - begin + LO_COLS - 1) / LO_COLS;
        begin = end;
    }
    const long long most = (lr_tiles(p, LT_ROWS) * turns + 1) / 2, slots = (long long)tgo_multiprocessors() * LowRankOut<BOXES, PAIRED, EIGHTS, TY>::BLOCKS;
    if (most > 0x3fffffff) return TGO_E_BAD_ARG;
    const int width = LowRankParts<TY>::N * ((p.rank + 15) / 16 * 16) * p.columns.slices;
    auto map_of = [](CUtensorMap* map, const void* ptr, long long rows, long long cols, long long stride, int box_rows) {
        return sizeof(TY) == 2 ? tg_map(map, ptr, rows, cols, stride, box_rows) : tg_map_f32(map, ptr, rows, cols, stride, box_rows);
    };
    CUtensorMap map_u, map_b, map_y, map_row, map_out;
    if (!tg_map(&map_u, u, p.T, width, width, LT_ROWS) || !tg_map(&map_b, p.b, (long long)p.adapters * p.N, p.rank, p.rank, LO_COLS) ||
        !map_of(&map_y, p.y, p.T, p.N, p.y_stride, 32) || !map_of(&map_row, p.y, p.T, p.N, p.y_stride, 1) ||
        !map_of(&map_out, p.out, p.T, p.N, p.out_stride, 32))
        return TGO_E_BAD_ARG;
    return tgo_launch_pdl(low_rank_out_kernel<BOXES, PAIRED, EIGHTS, TY>, dim3((unsigned)(most < slots ? most : slots)), dim3(LO_THREADS), bytes, stream,
                          map_u, map_b, map_y, map_row, map_out, p, turns, perm, info, tiles);
}

template <bool EIGHTS, typename TY>
static int low_rank_out_of(const LowRank& p, const bf16* u, const int* perm, const int* info, const int* tiles, cudaStream_t stream) {
    if (LowRankParts<TY>::N * ((p.rank + 15) / 16 * 16) <= 64) return low_rank_out<1, true, EIGHTS, TY>(p, u, perm, info, tiles, stream);
    if (p.rank <= 64) return low_rank_out<1, false, EIGHTS, TY>(p, u, perm, info, tiles, stream);
    if constexpr (!EIGHTS || sizeof(TY) == 2) return low_rank_out<2, false, EIGHTS, TY>(p, u, perm, info, tiles, stream);
    return TGO_E_BAD_ARG;                                    // three parts of two slices: lr_tile_takes refuses them
}

// 32-bit numbers of workspace: the plan, and u's parts in bfloat16.
template <typename TY> static long long lr_tile_work(const LowRank& p) {
    return (p.T + LP_INFO + 3 * lr_tiles(p, LT_ROWS) + 3) / 4 * 4 + (long long)p.T * ((p.rank + 15) / 16 * 16) * p.columns.slices * LowRankParts<TY>::N / 2;
}

template <typename TY> static int low_rank_tiles(const LowRank& p, int* work, cudaStream_t stream) {
    int* const perm = work;
    int* const info = perm + p.T;
    int* const tiles = info + LP_INFO;
    bf16* const u = (bf16*)(work + (p.T + LP_INFO + 3 * lr_tiles(p, LT_ROWS) + 3) / 4 * 4);
    LowRankAhead ahead = {{(const char*)p.x, (const char*)p.y}, {p.x_stride * 2, p.y_stride * (long long)sizeof(TY)},
                          {p.K * 2, p.N * (int)sizeof(TY)}, {}, p.out != p.y};
    long long left = LP_AHEAD;
    for (int m = 0; m < 2; ++m) {
        ahead.many[m] = (int)(left / ahead.bytes[m] < p.T ? left / ahead.bytes[m] : p.T);
        left -= (long long)ahead.many[m] * ahead.bytes[m];
    }
    int rc = tgo_launch_pdl(low_rank_plan_kernel, dim3(1 + 2 * tgo_multiprocessors()), dim3(LP_THREADS), 0, stream, p.ids, p.T, p.adapters,
                            LT_ROWS, perm, info, tiles, ahead);
    if (rc) return rc;
    const LowRankTile g = lr_plan(p);
    const int cols = lt_columns(g);
    if (cols == 32) rc = low_rank_u<32>(p, g, LowRankParts<TY>::N, perm, info, tiles, u, stream);
    else if (cols == 64) rc = low_rank_u<64>(p, g, LowRankParts<TY>::N, perm, info, tiles, u, stream);
    else if (cols == 128) rc = low_rank_u<128>(p, g, LowRankParts<TY>::N, perm, info, tiles, u, stream);
    else if (cols == 256) rc = low_rank_u<256>(p, g, LowRankParts<TY>::N, perm, info, tiles, u, stream);
    else rc = low_rank_u<512>(p, g, LowRankParts<TY>::N, perm, info, tiles, u, stream);
    if (rc) return rc;
    return p.columns.interleaved ? low_rank_out_of<true, TY>(p, u, perm, info, tiles, stream)
                                 : low_rank_out_of<false, TY>(p, u, perm, info, tiles, stream);
}

#define LR_TILE_BYTES 40000000ll
#define LR_TILE_ROWS 1024
// Whether a call goes by tiles of 128 rows: three kernels take 15 us however few the rows are, and each further adapter a
// part tile; the clusters read an adapter again for every eight rows, at about 3 TB/s, and come in rounds of 444 blocks. So
// from 40 MB of such reading or 1024 rows on. MEASURED (us, clusters / tiles; rows in four runs, then of 24 adapters at
// random): width 4096, q, k and v, rank 16, 384 rows 13 / 17 and 23 / 28, 768 28 / 19 and 36 / 33; rank 64, 96 rows 19 / 19 and
// 24 / 35, 256 25 / 19 and 30 / 37, 384 32 / 19 and 53 / 39; gate and up of 12288, rank 32, 128 rows 27 / 21 and 27 / 45, 384
// 38 / 21 and 69 / 54; 2048 x 2048, rank 16, 768 rows 15 / 15 and 20 / 24, 1536 25 / 17 and 31 / 27.
static int lr_forced = 0;                                    // for tests: 1 clusters, 2 tiles; 0: by the rule
TGO_API void tgo_low_rank_force_way(int way) { lr_forced = way; }
static bool lr_many(const LowRank& p) {
    if (lr_forced) return lr_forced == 2;
    return p.T >= LR_TILE_ROWS || (long long)p.T * p.rank * ((long long)p.columns.slices * p.K + p.N) * 2 / LF_ROWS >= LR_TILE_BYTES;
}

template <typename T, typename TY> static int low_rank_any(const LowRank& p, float* u, cudaStream_t stream) {
    const int width = p.columns.slices * p.rank;
    const int rc = tgo_launch_pdl(low_rank_down_kernel<T>, dim3(p.T, (width + 31) / 32), dim3(256), 0, stream, (const T*)p.x,
                                  p.x_stride, (const T*)p.a, p.scale, p.ids, p.adapters, width, p.K, u);
    if (rc) return rc;
    return tgo_launch_pdl(low_rank_up_kernel<T, TY>, dim3(p.T, (p.N + 255) / 256), dim3(256), 0, stream, (const float*)u,
                          (const T*)p.b, p.ids, p.adapters, p.rank, p.columns, p.N, (const TY*)p.y, p.y_stride, (TY*)p.out,
                          p.out_stride);
}

#define LR_E_WORK 1001            // returned, nothing done: the workspace is too small
// 32-bit numbers of workspace that a call needs.
template <typename T, typename TY> static long long lr_work(const LowRank& p) {
    const int width = p.columns.slices * p.rank;
    if constexpr (sizeof(T) == 2)
        if (lr_many(p) && lr_tile_takes<TY>(p)) return lr_tile_work<TY>(p);
    if (lr_few_takes<T>(p)) return !lr_scanned(p) ? p.T + LP_INFO + 3 * lr_tiles(p, LF_ROWS) : 0;
    return (long long)p.T * width;
}

// What a call returns: an error, 0 for one kernel launched, or minus the number of them.
static int lr_done(int rc, int kernels) { return rc || kernels == 1 ? rc : -kernels; }

template <typename T, typename TY> static int low_rank_launch(const LowRank& p, void* work, long long work_ints, cudaStream_t stream) {
    if (work_ints < lr_work<T, TY>(p)) return LR_E_WORK;
    if constexpr (sizeof(T) == 2)
        if (lr_many(p) && lr_tile_takes<TY>(p)) return lr_done(low_rank_tiles<TY>(p, (int*)work, stream), 3);
    if (lr_few_takes<T>(p)) return lr_done(low_rank_few<T, TY>(p, (int*)work, stream), lr_scanned(p) ? 1 : 2);
    return lr_done(low_rank_any<T, TY>(p, (float*)work, stream), 2);
}

static bool lr_fill(LowRank& p, int T, int K, int N, int adapters, int rank, int slices, const int* widths, int interleaved) {
    if (T <= 0 || K <= 0 || N <= 0 || adapters <= 0 || rank <= 0 || slices <= 0 || slices > LR_MAX_SLICES ||
        (N + 255) / 256 > 65535 || (interleaved && (slices != 2 || widths[0] != widths[1] || widths[0] % 8)))
        return false;
    p.T = T; p.K = K; p.N = N; p.adapters = adapters; p.rank = rank;
    p.columns.slices = slices;
    p.columns.interleaved = interleaved;
    long long end = 0;
    for (int i = 0; i < slices; ++i) {
        end += widths[i];
        if (widths[i] <= 0 || end > N) return false;
        p.columns.ends[i] = (int)end;
    }
    return end == N;
}

// The code that a wait of the kernels for many rows left when it ran out, or 0. Synchronises.
TGO_API int tgo_low_rank_error(int* value) { return (int)cudaMemcpyFromSymbol(value, low_rank_error_flag, sizeof(int)); }

// What a block of u's kernel takes of its multiprocessor for slices x rank values a row and clusters of `rows` rows: columns of tensor
// memory; *bytes gets the shared memory.
TGO_API int tgo_low_rank_tile_needs(int width, int rows, int* bytes) {
    const LowRankTile g = lt_tile(width, 4096, rows, 1);
    *bytes = lt_bytes(g);
    return lt_columns(g);
}

// Rows up to which a call of up to LR_SCAN_ADAPTERS adapters needs no workspace, if the kernel for few rows takes it.
TGO_API int tgo_low_rank_scanned_rows() { return LR_SCAN_ROWS; }

// x [T, K] of type dt, y and out [T, N] of type dt_y, rows strided; out may be y. a [adapters, slices, rank, K],
// b [adapters, N, rank] of type dt; widths: each slice's columns. `work` holds `work_ints` 32-bit
// numbers and lies on 16 bytes; LR_E_WORK: too few (for up to 512 rows most calls need none). With `needs` given
// nothing runs, and it gets how many the call needs. Returns an error, 0 for one kernel launched, or minus the number of them.
TGO_API int tgo_low_rank_add(const void* x, long long x_stride, const void* y, long long y_stride, void* out,
                             long long out_stride, const void* a, const void* b, const float* scale, const int* ids,
                             int dt, int dt_y, int T, int K, int N, int adapters, int rank, int slices, const int* widths,
                             int interleaved, void* work, long long work_ints, long long* needs, cudaStream_t stream) {
    if (T <= 0) return 0;
    LowRank p = {x, y, a, b, out, x_stride, y_stride, out_stride, scale, ids};
    if (!lr_fill(p, T, K, N, adapters, rank, slices, widths, interleaved)) return TGO_E_BAD_ARG;
    if (dt == TGO_F32 && dt_y == TGO_F32) {
        if (needs) { *needs = lr_work<float, float>(p); return 0; }
        return low_rank_launch<float, float>(p, work, work_ints, stream);
    }
    if (dt == TGO_BF16 && dt_y == TGO_BF16) {
        if (needs) { *needs = lr_work<bf16, bf16>(p); return 0; }
        return low_rank_launch<bf16, bf16>(p, work, work_ints, stream);
    }
    if (dt == TGO_BF16 && dt_y == TGO_F32) {
        if (needs) { *needs = lr_work<bf16, float>(p); return 0; }
        return low_rank_launch<bf16, float>(p, work, work_ints, stream);
    }
    return TGO_E_BAD_ARG;
}
