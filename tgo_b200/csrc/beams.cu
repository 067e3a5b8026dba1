// Beam search on the device: the best continuations of every request over its beams and the
// vocabulary, and rows of caches and states taken over from the beams they continue.
#include "common.cuh"

// ------------------------------------------------------------------------- beam_select
// For a request of W beams with scores c_w and rows of logits x_w over V tokens:
//   v(w, i) = c_w + x_w[i] - lse(x_w),  lse(x) = m + ln sum_i exp(x_i - m),  m = max x,
// and the K pairs (w, i) with the largest v, descending, equal ones by (w, i) ascending. A token with
// x = -inf is no candidate, nor is any token of a beam whose score or lse is not finite. Places without
// a candidate get (-inf, -1, -1).
//
// Inside a row the order is that of x itself, so one pass over a row gives both what the normaliser
// needs (a running maximum and sum per thread) and the row's K best. Blocks of the first kernel take a
// slice of a row each: sixteen values a thread and turn, the next turn's already under way; a thread
// looks closer at its values only when their largest, which the running maximum needs anyway, reaches
// the slice's K-th best so far. The second kernel has a block a request: it joins the slices' maxima
// and sums and merges their lists, ordered already, K times the best head. v is formed in 64 bits, so
// that close candidates of different beams are ordered by their values and not by a rounding.
#define BS_THREADS 256
#define BS_WARPS (BS_THREADS / 32)
#define BS_MAX_K 64
#define BS_MAX_BEAMS 32
#define BS_LISTS 256              // lists of a request: slices of a row x beams; a thread of the merge each
#define BS_LOOK 192               // candidates in the buffer from which it is cut back to K

// larger float <-> larger unsigned; the value is no NaN
__device__ __forceinline__ uint32_t bs_order(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bs_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// larger key <-> larger value, then lower index; 0 is no candidate (x > -inf has an order above 0x007fffff).
// x + 0 makes a negative zero equal to a positive one.
__device__ __forceinline__ unsigned long long bs_key(float x, int i) {
    return ((unsigned long long)bs_order(x + 0.f) << 32) | (0xffffffffu - (uint32_t)i);
}

// e^x for x <= 0, as a power of two; results below 2^-126 are 0 (they add nothing to a sum that holds a 1).
__device__ __forceinline__ float bs_exp(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504088896341f));
    return r;
}

// The K largest of buf[0..n) to buf[0..K), descending (n may be less than K: then all of them). Every
// thread calls it; keys are distinct.
__device__ void bs_cut(unsigned long long* buf, unsigned long long* sorted, unsigned* hist, int n, int K) {
    const int t = threadIdx.x;
    if (n > BS_THREADS) {
        // the K-th largest by its bits, eight at a time, then the keys from it on to the front
        __shared__ unsigned long long prefix_s;
        __shared__ int left_s, front_s;
        if (t == 0) { prefix_s = 0; left_s = K; front_s = 0; }
        for (int shift = 56; shift >= 0; shift -= 8) {
            hist[t] = 0;
            __syncthreads();
            const unsigned long long prefix = prefix_s;
            for (int i = t; i < n; i += BS_THREADS)
                if (shift == 56 || (buf[i] >> (shift + 8)) == (prefix >> (shift + 8)))
                    atomicAdd(&hist[(unsigned)(buf[i] >> shift) & 255u], 1u);
            __syncthreads();
            if (t == 0) {
                int left = left_s, b = 255;
                for (; b > 0 && (int)hist[b] < left; --b) left -= hist[b];
                prefix_s = prefix | ((unsigned long long)b << shift);
                left_s = left;
            }
            __syncthreads();
        }
        const unsigned long long least = prefix_s;
        for (int i = t; i < n; i += BS_THREADS)
            if (buf[i] >= least) sorted[atomicAdd(&front_s, 1)] = buf[i];
        __syncthreads();
        if (t < K) buf[t] = sorted[t];
        n = K;
        __syncthreads();
    }
    const unsigned long long mine = t < n ? buf[t] : 0;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += buf[j] > mine;
    __syncthreads();
    if (t < n && rank < K) buf[rank] = mine;
    __syncthreads();
}

// VPT vectors of four values a thread and turn.
template <int VPT>
__global__ void __launch_bounds__(BS_THREADS)
beam_part_kernel(const float* __restrict__ logits, long long stride, int V, const float* __restrict__ scores, int K,
                 int parts, int turns, float2* __restrict__ sums, unsigned long long* __restrict__ lists) {
    constexpr int TILE = BS_THREADS * VPT;                  // vectors a turn
    __shared__ unsigned long long buf[4 * TILE + BS_LOOK];
    __shared__ unsigned long long sorted[BS_MAX_K];
    __shared__ unsigned hist[BS_THREADS];
    __shared__ float2 red[BS_WARPS];
    __shared__ int count;
    __shared__ unsigned warp_least[BS_WARPS];
    pdl_wait();
    const int row = blockIdx.y, part = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    unsigned long long* const list = lists + ((size_t)row * parts + part) * K;
    const float score = scores[row];
    if (!(score > -INFINITY && score < INFINITY)) {          // the same for the whole block
        if (t < K) list[t] = 0;
        if (t == 0) sums[(size_t)row * parts + part] = make_float2(-INFINITY, 0.f);
        return;
    }
    const float* const x = logits + (size_t)row * stride;
    // vectors lie on 16-byte boundaries: vector v holds the row's values 4 v - off .. 4 v - off + 3
    const int off = (int)(((uintptr_t)x >> 2) & 3);
    const int vectors = (V + off + 3) / 4;
    const int v0 = part * turns * TILE, v1 = min(v0 + turns * TILE, vectors);
    if (t == 0) count = 0;

    float4 next[VPT];
    auto load = [&](int base) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int v = base + j * BS_THREADS + t, e = 4 * v - off;
            float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (v < v1) {
                if (e >= 0 && e + 3 < V) q = __ldcs((const float4*)(x + e));
                else {
                    if (e >= 0 && e < V) q.x = x[e];
                    if (e + 1 >= 0 && e + 1 < V) q.y = x[e + 1];
                    if (e + 2 >= 0 && e + 2 < V) q.z = x[e + 2];
                    if (e + 3 >= 0 && e + 3 < V) q.w = x[e + 3];
                }
            }
            next[j] = q;
        }
    };
    load(v0);
    float m = -INFINITY, s = 0.f;                            // this thread's running maximum and sum
    unsigned long long least = 0;                            // a later candidate's key is larger than this
    float least_x = -INFINITY;
    for (int base = v0; base < v1; base += TILE) {
        float4 cur[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) cur[j] = next[j];
        if (base + TILE < v1) load(base + TILE);
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < VPT; ++j) top = fmaxf(top, fmaxf(fmaxf(cur[j].x, cur[j].y), fmaxf(cur[j].z, cur[j].w)));
        // where everything so far is -inf, 0 stands for the maximum: the exponentials are 0 and not NaN. The
        // difference is formed before the scaling: rows masked with the type's lowest value stay in range.
        const float now = fmaxf(m, top), at = now > -INFINITY ? now : 0.f;
        s *= m > -INFINITY ? bs_exp(m - at) : 0.f;
        float add = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            add += (bs_exp(cur[j].x - at) + bs_exp(cur[j].y - at)) + (bs_exp(cur[j].z - at) + bs_exp(cur[j].w - at));
        s += add;
        m = now;
        if (base == v0) {
            // before anything is kept: of each warp's threads' maxima the ceil(K / 8)-th, and the least of
            // those over the warps, is reached by K values at least
            const int q = (K + BS_WARPS - 1) / BS_WARPS;
            unsigned mine = bs_order(top + 0.f), got = 0;
            for (int i = 0; i < q; ++i) {
                got = __reduce_max_sync(0xffffffffu, mine);
                if (lane == __ffs(__ballot_sync(0xffffffffu, mine == got)) - 1) mine = 0;
            }
            if (lane == 0) warp_least[warp] = got;
            __syncthreads();
            unsigned o = warp_least[0];
#pragma unroll
            for (int i = 1; i < BS_WARPS; ++i) o = min(o, warp_least[i]);
            const float from = bs_value(o);
            if (from > -INFINITY) {
                least = ((unsigned long long)o << 32) - 1;
                least_x = from;
            }
        }
        bool full = false;
        if (top >= least_x && top > -INFINITY) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int e = 4 * (base + j * BS_THREADS + t) - off;
                const float q[4] = {cur[j].x, cur[j].y, cur[j].z, cur[j].w};
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (q[c] >= least_x && q[c] > -INFINITY) {
                        const unsigned long long key = bs_key(q[c], e + c);
                        if (key > least) {
                            const int place = atomicAdd(&count, 1);
                            buf[place] = key;
                            full = full || place >= BS_LOOK - 1;
                        }
                    }
            }
        }
        if (__syncthreads_or(full)) {
            const int n = count;
            bs_cut(buf, sorted, hist, n, K);
            if (t == 0) count = min(n, K);
            __syncthreads();
            least = buf[K - 1];                              // BS_LOOK > K: there are K of them
            least_x = bs_value((uint32_t)(least >> 32));
            __syncthreads();
        }
    }
    __syncthreads();
    const int n = count;
    bs_cut(buf, sorted, hist, n, K);
    if (t < K) list[t] = t < n ? buf[t] : 0;
    const float wm = warp_max(m);
    const float ws = warp_sum(m > -INFINITY ? s * bs_exp(m - wm) : s);
    if (lane == 0) red[warp] = make_float2(wm, ws);
    __syncthreads();
    if (t == 0) {
        float bm = red[0].x;
        for (int i = 1; i < BS_WARPS; ++i) bm = fmaxf(bm, red[i].x);
        float sum = 0.f;
        for (int i = 0; i < BS_WARPS; ++i) sum += red[i].x > -INFINITY ? red[i].y * bs_exp(red[i].x - bm) : red[i].y;
        sums[(size_t)row * parts + part] = make_float2(bm, sum);
    }
}

// One block a request. (m, s) of a slice: its values' exp(x - m) sum to s; a NaN or +inf among them has
// made s NaN, a slice of -inf alone has m = -inf and s = 0.
__global__ void __launch_bounds__(BS_LISTS)
beam_merge_kernel(const float* __restrict__ scores, int W, int K, int parts, const float2* __restrict__ sums,
                  const unsigned long long* __restrict__ lists, float* __restrict__ picked, int* __restrict__ parents,
                  int* __restrict__ tokens) {
    __shared__ double base_s[BS_MAX_BEAMS];                  // score - ln s, or NaN: the beam gives nothing
    __shared__ float max_s[BS_MAX_BEAMS];
    __shared__ double best_v[BS_LISTS / 32];
    __shared__ int best_w[BS_LISTS / 32], best_i[BS_LISTS / 32], best_t[BS_LISTS / 32];
    pdl_wait();
    const int b = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31, warps = blockDim.x >> 5;
    for (int w = warp; w < W; w += warps) {
        const float2* row = sums + ((size_t)b * W + w) * parts;
        float m = -INFINITY;
        for (int p = lane; p < parts; p += 32) m = fmaxf(m, row[p].x);
        m = warp_max(m);
        double s = 0.0;
        for (int p = lane; p < parts; p += 32)
            s += row[p].x > -INFINITY ? (double)row[p].y * exp((double)row[p].x - (double)m) : (double)row[p].y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const double base = (double)scores[b * W + w] - log(s);
        if (lane == 0) {
            base_s[w] = base > -INFINITY && base < INFINITY ? base : __longlong_as_double(0x7ff8000000000000ll);
            max_s[w] = m;
        }
    }
    __syncthreads();
    const int w = t / parts;
    const bool have = w < W;
    const unsigned long long* list = lists + ((size_t)b * W * parts + t) * K;
    const double base = have ? base_s[w] : 0.0, top = have ? (double)max_s[w] : 0.0;
    int at = 0, tok = 0;
    double v = -INFINITY;
    auto head = [&]() {                                      // -inf: the list is used up
        v = -INFINITY;
        if (have && at < K && base == base) {
            const unsigned long long key = list[at];
            if (key) {
                v = base + ((double)bs_value((uint32_t)(key >> 32)) - top);
                tok = (int)(0xffffffffu - (uint32_t)key);
            }
        }
    };
    head();
    for (int k = 0; k < K; ++k) {
        double bv = v;
        int bw = have ? w : BS_MAX_BEAMS, bi = tok, bt = t;
        auto take = [&](double ov, int ow, int oi, int ot) {
            if (ov > bv || (ov == bv && (ow < bw || (ow == bw && oi < bi)))) { bv = ov; bw = ow; bi = oi; bt = ot; }
        };
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int ow = __shfl_xor_sync(0xffffffffu, bw, o), oi = __shfl_xor_sync(0xffffffffu, bi, o),
                      ot = __shfl_xor_sync(0xffffffffu, bt, o);
            take(ov, ow, oi, ot);
        }
        if (lane == 0) { best_v[warp] = bv; best_w[warp] = bw; best_i[warp] = bi; best_t[warp] = bt; }
        __syncthreads();
        bv = best_v[0]; bw = best_w[0]; bi = best_i[0]; bt = best_t[0];
        for (int i = 1; i < warps; ++i) take(best_v[i], best_w[i], best_i[i], best_t[i]);
        const bool none = !(bv > -INFINITY);
        if (t == 0) {
            const size_t o = (size_t)b * K + k;
            picked[o] = none ? -INFINITY : (float)bv;
            parents[o] = none ? -1 : bw;
            tokens[o] = none ? -1 : bi;
        }
        if (!none && t == bt) { ++at; head(); }
        __syncthreads();
    }
}

static void beam_plan(int rows, int W, int V, int sms, int* vpt, int* turns, int* parts) {
    *vpt = 4;
    const int tiles = (V + 3 + 4 * BS_THREADS * 4 - 1) / (4 * BS_THREADS * 4);
    int p = (4 * sms + rows - 1) / rows;                     // four blocks a multiprocessor
    p = p < tiles ? p : tiles;
    p = p < BS_LISTS / W ? p : BS_LISTS / W;
    *turns = (tiles + p - 1) / p;
    *parts = (tiles + *turns - 1) / *turns;
}

// Slices of a row that tgo_beam_select works with: it needs rows x slices x (8 + 8 K) bytes of workspace.
TGO_API int tgo_beam_select_parts(int requests, int beams, int V) {
    if (requests <= 0 || beams <= 0 || beams > BS_MAX_BEAMS || V <= 0 || V > 0x7fffffff - 8) return 0;
    int vpt, turns, parts;
    beam_plan(requests * beams, beams, V, tgo_multiprocessors(), &vpt, &turns, &parts);
    return parts;
}

// picked, parents, tokens [requests, K]; scores [requests, beams]; logits rows `stride` floats apart, beams of
// a request one after the other. `work` has `parts` slices' room for each row, parts as above.
TGO_API int tgo_beam_select(const float* logits, long long stride, const float* scores, int requests, int beams, int V,
                            int K, float* picked, int* parents, int* tokens, void* work, int parts, cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (beams <= 0 || beams > BS_MAX_BEAMS || K <= 0 || K > BS_MAX_K || V <= 0 || V > 0x7fffffff - 8 ||
        (long long)requests * beams > 65535)
        return TGO_E_BAD_ARG;
    int vpt, turns, mine;
    beam_plan(requests * beams, beams, V, tgo_multiprocessors(), &vpt, &turns, &mine);
    if (mine != parts) return TGO_E_BAD_ARG;
    const int rows = requests * beams;
    float2* sums = (float2*)work;
    unsigned long long* lists = (unsigned long long*)(sums + (size_t)rows * parts);
    const int rc = tgo_launch_pdl(beam_part_kernel<4>, dim3(parts, rows), dim3(BS_THREADS), 0, stream, logits, stride, V,
                                  scores, K, parts, turns, sums, lists);
    if (rc) return rc;
    const int threads = (beams * parts + 31) / 32 * 32;
    return tgo_launch_pdl(beam_merge_kernel, dim3(requests), dim3(threads), 0, stream, scores, beams, K, parts,
                          (const float2*)sums, (const unsigned long long*)lists, picked, parents, tokens);
}

// ------------------------------------------------------------------------ reorder_rows
// In every tensor, for every group of W rows: row index[w] <- old row index[parents[w]], in place. A thread
// owns a column of up to 16 bytes of a group's rows: it reads what the changed rows take and only then
// writes, so no other thread's reads can meet its writes, whatever chain or exchange the parents make. Bound
// by memory: a changed row is written once, a source read once from memory (the second child finds it in
// the cache).
#define RR_MAX_TENSORS 64
#define RR_MAX_BEAMS 32
#define RR_THREADS 256

struct ReorderRows {
    char* base[RR_MAX_TENSORS];
    long long outer_stride[RR_MAX_TENSORS], row_stride[RR_MAX_TENSORS], row_bytes[RR_MAX_TENSORS], rows[RR_MAX_TENSORS];
    int outer[RR_MAX_TENSORS];
};

template <typename VEC, int W>
__global__ void __launch_bounds__(RR_THREADS)
reorder_rows_kernel(const __grid_constant__ ReorderRows d, const int* __restrict__ index, const int* __restrict__ parents,
                    int beams) {
    __shared__ long long to[RR_MAX_BEAMS], from[RR_MAX_BEAMS];       // byte offsets; from < 0: the row stays
    pdl_wait();
    const int k = blockIdx.z, g = blockIdx.y, t = threadIdx.x;
    const long long vectors = d.row_bytes[k] / (long long)sizeof(VEC), chunks = (vectors + RR_THREADS - 1) / RR_THREADS;
    if (blockIdx.x >= chunks * d.outer[k]) return;
    bool moves = false;
    if (t < beams) {
        const int p = parents[(size_t)g * beams + t];
        const long long r = index[(size_t)g * beams + t];
        const long long q = p >= 0 && p < beams ? index[(size_t)g * beams + p] : -1;
        moves = p != t && r >= 0 && r < d.rows[k] && q >= 0 && q < d.rows[k];
        to[t] = r * d.row_stride[k];
        from[t] = moves ? q * d.row_stride[k] : -1;
    }
    if (!__syncthreads_or(moves)) return;
    const int o = (int)(blockIdx.x / chunks);
    const long long v = (blockIdx.x - o * chunks) * RR_THREADS + t;
    if (v >= vectors) return;
    char* const base = d.base[k] + o * d.outer_stride[k] + v * (long long)sizeof(VEC);
    VEC got[W];
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < beams && from[w] >= 0) got[w] = *(const VEC*)(base + from[w]);
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (w < beams && from[w] >= 0) *(VEC*)(base + to[w]) = got[w];
}

template <typename VEC>
static int reorder_launch(const ReorderRows& d, int tensors, int groups, int beams, long long blocks, const int* index,
                          const int* parents, cudaStream_t stream) {
    const dim3 grid((unsigned)blocks, groups, tensors), block(RR_THREADS);
    if (beams <= 4) return tgo_launch_pdl(reorder_rows_kernel<VEC, 4>, grid, block, 0, stream, d, index, parents, beams);
    if (beams <= 8) return tgo_launch_pdl(reorder_rows_kernel<VEC, 8>, grid, block, 0, stream, d, index, parents, beams);
    if (beams <= 16) return tgo_launch_pdl(reorder_rows_kernel<VEC, 16>, grid, block, 0, stream, d, index, parents, beams);
    return tgo_launch_pdl(reorder_rows_kernel<VEC, 32>, grid, block, 0, stream, d, index, parents, beams);
}

// desc: per tensor six numbers: address, outer count, bytes from one outer block to the next, rows, bytes
// from one row to the next, bytes of a row. index, parents [groups, beams].
TGO_API int tgo_reorder_rows(const long long* desc, int tensors, const int* index, const int* parents, int groups,
                             int beams, cudaStream_t stream) {
    if (tensors <= 0 || groups <= 0) return 0;
    if (beams <= 0 || beams > RR_MAX_BEAMS || groups > 65535) return TGO_E_BAD_ARG;
    for (int first = 0; first < tensors; first += RR_MAX_TENSORS) {
        ReorderRows d;
        const int n = tensors - first < RR_MAX_TENSORS ? tensors - first : RR_MAX_TENSORS;
        long long all = 0;
        for (int i = 0; i < n; ++i) {
            const long long* q = desc + 6 * (first + i);
            if (q[1] <= 0 || q[1] > 0x7fffffff || q[3] <= 0 || q[4] < q[5] || q[5] <= 0) return TGO_E_BAD_ARG;
            d.base[i] = (char*)q[0];
            d.outer[i] = (int)q[1];
            d.outer_stride[i] = q[2];
            d.rows[i] = q[3];
            d.row_stride[i] = q[4];
            d.row_bytes[i] = q[5];
            all |= q[0] | q[2] | q[4] | q[5];
        }
        const int width = all & 1 ? 1 : all & 2 ? 2 : all & 4 ? 4 : all & 8 ? 8 : 16;
        long long blocks = 0;
        for (int i = 0; i < n; ++i) {
            const long long c = (d.row_bytes[i] / width + RR_THREADS - 1) / RR_THREADS * d.outer[i];
            blocks = c > blocks ? c : blocks;
        }
        if (blocks > 0x7fffffff) return TGO_E_BAD_ARG;
        int rc;
        if (width == 16) rc = reorder_launch<uint4>(d, n, groups, beams, blocks, index, parents, stream);
        else if (width == 8) rc = reorder_launch<uint2>(d, n, groups, beams, blocks, index, parents, stream);
        else if (width == 4) rc = reorder_launch<uint32_t>(d, n, groups, beams, blocks, index, parents, stream);
        else if (width == 2) rc = reorder_launch<uint16_t>(d, n, groups, beams, blocks, index, parents, stream);
        else return TGO_E_BAD_ARG;
        if (rc) return rc;
    }
    return 0;
}
