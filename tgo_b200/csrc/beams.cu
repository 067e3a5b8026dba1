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
// needs (a maximum and a sum per thread) and the row's K best. A request's blocks are shared out evenly among its beams
// that live, a slice of a row each: sixteen values a thread and turn, the next turn's already under way; a thread looks
// closer at its values only when their largest, which the sum needs anyway, reaches the slice's K-th best so far. Then one
// block a request joins the slices' maxima and sums and ranks what can be among the K best: in a second kernel, or, for
// few rows, in the first block of a cluster. v is formed in 64 bits: candidates of one beam are ordered as their logits are, those of
// different beams but for the error of the sums under the logarithms, which are 32-bit sums of approximate exponentials.
//
// MEASURED (B200, calls in a graph): 512 rows of 151936 and 16 picks 57.4 us, 5.4 TB/s (59.7 where the host makes each call);
// without looking for candidates the same pass takes 50, with a look only every fourth turn, at values read again, 64, from a ring filled by bulk
// copies 66, with warps that meet only when one has found enough 65. 64 rows of it 15.4 us; one live beam of five in 12
// requests 10.3 (13.8 where the others' blocks find nothing to do); 4 rows of 32768 7.6. There the kernels' latencies
// show, about 4 and 3 us, and the first turns' many candidates.
#define BS_THREADS 256
#define BS_VPT 4                  // vectors of four values a thread and turn
#define BS_TILE (BS_THREADS * BS_VPT)       // vectors a turn
#define BS_BLOCKS 4               // of a multiprocessor (64 registers a thread; 48 spill nothing and are slower)
#define BS_WARPS (BS_THREADS / 32)
#define BS_MAX_K 64
#define BS_MAX_BEAMS 32

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

#define BS_LOG2E 1.44269504088896341f
// 2^x; results below 2^-126 are 0 (they add nothing to a sum that holds a 1).
__device__ __forceinline__ float bs_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float bs_exp(float x) { return bs_exp2(x * BS_LOG2E); }

// Two numbers at a time.
__device__ __forceinline__ unsigned long long bs_pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void bs_unpair(unsigned long long p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ unsigned long long bs_mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long bs_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The K largest of kept[0..k) and buf[0..n), descending, to `to` (fewer: all of them). Every thread calls it;
// keys are distinct, buf has room for k more, what is read has been synchronised and what is written has not.
__device__ void bs_cut(const unsigned long long* kept, int k, unsigned long long* buf, int n, unsigned* hist,
                       unsigned long long* to, int K) {
    __shared__ unsigned long long front[BS_MAX_K];
    const int t = threadIdx.x;
    if (k + n > BS_THREADS) {
        // the K-th largest by its bits, eight at a time, then the keys from it on to the front
        __shared__ unsigned long long prefix_s;
        __shared__ int left_s, front_s;
        __shared__ int warp_sums[BS_WARPS];
        static_assert(BS_THREADS == 256, "a thread a bin");
        if (t < k) buf[n + t] = kept[t];
        n += k;
        k = 0;
        if (t == 0) { prefix_s = 0; left_s = K; front_s = 0; }
        for (int shift = 56; shift >= 0; shift -= 8) {
            hist[t] = 0;
            __syncthreads();
            const unsigned long long prefix = prefix_s;
            const int left = left_s;
            for (int i = t; i < n; i += BS_THREADS)
                if (shift == 56 || (buf[i] >> (shift + 8)) == (prefix >> (shift + 8)))
                    atomicAdd(&hist[(unsigned)(buf[i] >> shift) & 255u], 1u);
            __syncthreads();
            // keys in this thread's bin, the bins above it and this one, counted from the top
            const int bin = 255 - t, mine = (int)hist[bin];
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int below = __shfl_up_sync(0xffffffffu, sum, o);
                sum += (t & 31) >= o ? below : 0;
            }
            if ((t & 31) == 31) warp_sums[t >> 5] = sum;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < BS_WARPS; ++w) sum += w < t >> 5 ? warp_sums[w] : 0;
            if (sum >= left && sum - mine < left) {          // one thread's
                prefix_s = prefix | ((unsigned long long)bin << shift);
                left_s = left - (sum - mine);
            }
            __syncthreads();
        }
        const unsigned long long least = prefix_s;
        for (int i = t; i < n; i += BS_THREADS)
            if (buf[i] >= least) front[atomicAdd(&front_s, 1)] = buf[i];
        __syncthreads();
        buf = front;
        n = K;
    }
    if ((t & ~31) >= k + n) return;
    const unsigned long long mine = t < k ? kept[t] : t < k + n ? buf[t - k] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < k; ++j) rank += kept[j] > mine;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += buf[j] > mine;
    if (t < k + n && rank < K) to[rank] = mine;
}

// The block's slice `part` of `parts` even ones of a row x of V values: its K best to `list`, descending (0: none), its maximum and sum to `sum`.
// buf has BS_BUF numbers of shared memory.
#define BS_BUF (4 * BS_TILE + 4 * BS_MAX_K)
__device__ __forceinline__ void bs_scan(const float* __restrict__ x, int V, int K, int part, int parts, unsigned long long* buf,
                                        float2* sum, unsigned long long* list) {
    __shared__ unsigned long long kept[2][BS_MAX_K];
    __shared__ unsigned hist[256];
    __shared__ float2 red[BS_WARPS];
    __shared__ int counts[2];         // candidates in buf; the other one is set to 0 meanwhile
    __shared__ unsigned warp_least[BS_WARPS];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    // vectors lie on 16-byte boundaries: vector v holds the row's values 4 v - off .. 4 v - off + 3
    const int off = (int)(((uintptr_t)x >> 2) & 3);
    const int vectors = (V + off + 3) / 4;
    const int share = (int)((unsigned)(vectors + parts - 1) / (unsigned)parts), v0 = min(part * share, vectors), v1 = min(v0 + share, vectors);
    if (t < 2) counts[t] = 0;

    float4 next[BS_VPT];
    const float* const at_v = x - off;                       // where vector 0 would begin; aligned
    // the vectors before v_head and from v_tail on reach over the row's ends
    const int v_head = off ? 1 : 0, v_tail = min(v1, (V + off) / 4);
    auto load = [&](int base) {
        if (base >= v_head && base + BS_TILE <= v_tail) {
#pragma unroll
            for (int j = 0; j < BS_VPT; ++j) next[j] = __ldcs((const float4*)(at_v + 4 * (size_t)(base + t)) + j * BS_THREADS);
            return;
        }
#pragma unroll
        for (int j = 0; j < BS_VPT; ++j) {
            const int v = base + j * BS_THREADS + t, e = 4 * v - off;
            float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (v >= v_head && v < v_tail) q = __ldcs((const float4*)(at_v + 4 * (size_t)v));
            else if (v < v1) {
                if (e >= 0 && e < V) q.x = x[e];
                if (e + 1 >= 0 && e + 1 < V) q.y = x[e + 1];
                if (e + 2 >= 0 && e + 2 < V) q.z = x[e + 2];
                if (e + 3 >= 0 && e + 3 < V) q.w = x[e + 3];
            }
            next[j] = q;
        }
    };
    load(v0);
    float m = -INFINITY, s = 0.f;                            // this thread's running maximum and sum
    unsigned long long least = 0;                            // a later candidate's key is larger than this
    float least_x = -INFINITY;
    // The buffer is cut back to K whenever it holds this many: the higher the K-th, the fewer threads look closer,
    // but a cut stops the block for about 1000 cycles.
    const int look = max(3 * K, 32);
    int k = 0, epoch = 0;                                    // kept[epoch & 1][0..k), counts[epoch & 1]
    for (int base = v0; base < v1; base += BS_TILE) {
        float4 cur[BS_VPT];
#pragma unroll
        for (int j = 0; j < BS_VPT; ++j) cur[j] = next[j];
        if (base + BS_TILE < v1) load(base + BS_TILE);
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < BS_VPT; ++j) top = fmaxf(top, fmaxf(fmaxf(cur[j].x, cur[j].y), fmaxf(cur[j].z, cur[j].w)));
        const float v[16] = {cur[0].x, cur[0].y, cur[0].z, cur[0].w, cur[1].x, cur[1].y, cur[1].z, cur[1].w,
                             cur[2].x, cur[2].y, cur[2].z, cur[2].w, cur[3].x, cur[3].y, cur[3].z, cur[3].w};
        // The sum is taken against a maximum that is renewed when a value passes it by more than 40: e^40 of
        // them are far from the range's end. Where everything so far is -inf, 0 stands for it: the
        // exponentials are 0 and not NaN.
        if (!(top <= m + 40.f) && top == top) {
            s *= m > -INFINITY ? bs_exp(m - top) : 0.f;
            m = top;
        }
        // The difference comes first, then the factor: its rounding goes by its own size. A difference of two products with
        // log2 e is off by 2^-24 of the maximum's, whatever the difference: by hundreds where tokens are masked with -1e10.
        const float at = m > -INFINITY ? m : 0.f;
        const unsigned long long by = bs_pair(-at, -at), scale = bs_pair(BS_LOG2E, BS_LOG2E);
        unsigned long long sum[2] = {bs_pair(s, 0.f), 0ull};
#pragma unroll
        for (int i = 0; i < 16 / 2; ++i) {
            float a, b;
            bs_unpair(bs_mul2(bs_add2(bs_pair(v[2 * i], v[2 * i + 1]), by), scale), a, b);
            sum[i & 1] = bs_add2(sum[i & 1], bs_pair(bs_exp2(a), bs_exp2(b)));
        }
        float a, b;
        bs_unpair(bs_add2(sum[0], sum[1]), a, b);
        s = a + b;
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
            unsigned hits = 0;
#pragma unroll
            for (int i = 0; i < 4 * BS_VPT; ++i) hits |= v[i] >= least_x ? 1u << i : 0u;
            // a value at a time from each thread that has any: picked from the registers by its number's bits
            while (hits) {
                const int i = __ffs(hits) - 1;
                hits &= hits - 1;
                float h[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) h[c] = i & 8 ? v[c + 8] : v[c];
#pragma unroll
                for (int c = 0; c < 4; ++c) h[c] = i & 4 ? h[c + 4] : h[c];
                h[0] = i & 2 ? h[2] : h[0];
                h[1] = i & 2 ? h[3] : h[1];
                const float x_i = i & 1 ? h[1] : h[0];
                const unsigned long long key = bs_key(x_i, 4 * (base + (i >> 2) * BS_THREADS + t) - off + (i & 3));
                if (key > least && x_i > -INFINITY) {
                    const int place = atomicAdd(&counts[epoch & 1], 1);
                    buf[place] = key;
                    full = full || place >= look - 1;
                }
            }
        }
        if (__syncthreads_or(full)) {
            const int n = counts[epoch & 1];
            if (t == 0) counts[~epoch & 1] = 0;
            bs_cut(kept[epoch & 1], k, buf, n, hist, kept[~epoch & 1], K);
            k = min(k + n, K);
            ++epoch;
            __syncthreads();
            if (k == K) {
                least = kept[epoch & 1][K - 1];
                least_x = bs_value((uint32_t)(least >> 32));
            }
        }
    }
    __syncthreads();
    const int n = counts[epoch & 1];
    bs_cut(kept[epoch & 1], k, buf, n, hist, list, K);
    if (t >= k + n && t < K) list[t] = 0;
    const float wm = warp_max(m);
    const float ws = warp_sum(m > -INFINITY ? s * bs_exp(m - wm) : s);
    if (lane == 0) red[warp] = make_float2(wm, ws);
    __syncthreads();
    if (t == 0) {
        float bm = red[0].x;
        for (int i = 1; i < BS_WARPS; ++i) bm = fmaxf(bm, red[i].x);
        float all = 0.f;
        for (int i = 0; i < BS_WARPS; ++i) all += red[i].x > -INFINITY ? red[i].y * bs_exp(red[i].x - bm) : red[i].y;
        *sum = make_float2(bm, all);
    }
}

// How a request's blocks are shared out: evenly among the beams that live, those whose score is finite, and no finer than
// a turn a block. (A search's first step has one beam of each request.)
struct BeamShare {
    unsigned lives;                                          // a bit a beam
    int live, parts;
    float score;                                             // of the beam of this lane's number (any for a lane past them)
    // a / b for both up to 256: the quotient of a + 1/2 is 1/512 or more from a whole number
    __device__ __forceinline__ static int divide(int a, int b) { return (int)__fdividef((float)a + 0.5f, (float)b); }
    __device__ __forceinline__ BeamShare(float mine, int W, int V, int blocks) : score(mine) {
        const int lane = threadIdx.x & 31, turns = (V + 3 + 4 * BS_TILE - 1) / (4 * BS_TILE);
        lives = __ballot_sync(0xffffffffu, lane < W && score > -INFINITY && score < INFINITY);
        live = __popc(lives);
        parts = live ? min(divide(blocks, live), turns) : 0;
    }
    // The j-th beam that lives.
    __device__ __forceinline__ int beam(int j) const {
        const int lane = threadIdx.x & 31;
        return __ffs(__ballot_sync(0xffffffffu, (lives >> lane & 1) && __popc(lives & ((1u << lane) - 1)) == j)) - 1;
    }
    // Block `block` of the request does its part, if it has one.
    __device__ __forceinline__ void scan(const float* logits, long long stride, size_t row, int V, int K, int block, unsigned long long* buf,
                                         float2* sum, unsigned long long* list) const {
        if (block >= live * parts) return;
        const int j = divide(block, parts);
        const float* const x = logits + (row + beam(j)) * stride;
        bs_scan(x, V, K, block - j * parts, parts, buf, sum, list);
    }
};
__device__ __forceinline__ float bs_score(const float* scores, int W) { return (threadIdx.x & 31) < W ? scores[threadIdx.x & 31] : 0.f; }

__global__ void __launch_bounds__(BS_THREADS, BS_BLOCKS)
beam_part_kernel(const float* __restrict__ logits, long long stride, int V, const float* __restrict__ scores, int W, int K,
                 float2* __restrict__ sums, unsigned long long* __restrict__ lists) {
    __shared__ unsigned long long buf[BS_BUF];
    pdl_wait();
    const int block = blockIdx.x, blocks = gridDim.x;
    const size_t b = blockIdx.y, at = b * blocks + block;
    BeamShare(bs_score(scores + b * W, W), W, V, blocks).scan(logits, stride, b * W, V, K, block, buf, sums + at, lists + at * K);
}

// The block joins a request's slices. (m, s) of a slice: its values' exp(x - m) sum to s; a NaN or +inf among them has
// made s NaN, a slice of -inf alone has m = -inf and s = 0. The slices' lists are sorted: the K-th best of
// their first candidates (as many of each as make 3 K) bounds what can be among the K best, at most K lists
// reach it, and what reaches it is ranked by counting.
#define BM_THREADS 256
#define BM_LISTS 256
#define BM_CANDIDATES 4096        // of a request's lists together

// Larger (first, then second) is better: the order of v's bits, the complement of beam and token.
struct __align__(16) Pick {
    unsigned long long v, place;
};
__device__ __forceinline__ int better(const Pick& a, const Pick& b) { return (int)(a.v > b.v) | ((int)(a.v == b.v) & (int)(a.place > b.place)); }
__device__ __forceinline__ unsigned long long bm_order(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double bm_value(unsigned long long o) {
    return __longlong_as_double((long long)(o >> 63 ? o & 0x7fffffffffffffffull : ~o));
}
// How many of from[0..n) are better than p.
__device__ __forceinline__ int bm_rank(const Pick* from, int n, const Pick& p) {
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += better(from[j], p);
    return rank;
}

// lists [live * parts][K] and sums [live * parts]; `first`: the lists' number of this thread; `room`: as much shared memory as beam_merge_bytes says.
__device__ __forceinline__ void bm_join(const BeamShare& share, int K, const float2* sums,
                                        const unsigned long long* lists, unsigned long long first,
                                        unsigned char* room, float* picked, int* parents, int* tokens) {
    __shared__ double base_s[BS_MAX_BEAMS];                  // score - ln s, or NaN: the beam gives nothing
    __shared__ float max_s[BS_MAX_BEAMS];
    __shared__ int beam_s[BS_MAX_BEAMS];
    __shared__ Pick bound_s;
    __shared__ int count;
    const int W = share.live, parts = share.parts;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, n = W * parts;
    const int q = n ? min((3 * K + n - 1) / n, K) : 0;       // a list's heads
    Pick* const all = (Pick*)room;                           // [n][K]
    Pick* const heads = all + n * K;                         // [n][q]
    Pick* const found = heads + n * q;                       // [n][K]
    if (t == 0) { count = 0; bound_s = Pick{0, 0}; }
    for (int w = warp; w < W; w += BM_THREADS / 32) {
        const float2* row = sums + w * parts;
        const int beam = share.beam(w);
        const float score = __shfl_sync(0xffffffffu, share.score, beam);
        float m = -INFINITY;
        for (int p = lane; p < parts; p += 32) m = fmaxf(m, row[p].x);
        m = warp_max(m);
        float s = 0.f;
        for (int p = lane; p < parts; p += 32) s += row[p].x > -INFINITY ? row[p].y * bs_exp(row[p].x - m) : row[p].y;
        s = warp_sum(s);
        // ln s = e ln 2 + ln(f), s = 2^e f, 1 <= f < 2: the larger part in 64 bits
        const int e = (int)(__float_as_uint(s) >> 23) - 127;
        const float f = __uint_as_float((__float_as_uint(s) & 0x007fffffu) | 0x3f800000u);
        const double base = (double)score - ((double)e * 0.693147180559945309 + (double)log1pf(f - 1.f));
        if (lane == 0) {
            base_s[w] = s > 0.f && s < INFINITY && m < INFINITY ? base : __longlong_as_double(0x7ff8000000000000ll);
            max_s[w] = m;
            beam_s[w] = beam;
        }
    }
    __syncthreads();
    for (int e = t; e < n * K; e += BM_THREADS) {
        const unsigned long long key = e == t ? first : lists[e];
        const int l = e / K, i = e - l * K, w = l / parts;
        const double base = base_s[w];
        Pick p = {0, 0};                                     // nothing
        if (key && base == base) {
            p.v = bm_order(base + ((double)bs_value((uint32_t)(key >> 32)) - (double)max_s[w]));
            p.place = ~(((unsigned long long)beam_s[w] << 32) | (0xffffffffu - (uint32_t)key));
        }
        all[e] = p;
        if (i < q) heads[l * q + i] = p;
    }
    __syncthreads();
    for (int e = t; e < n * q; e += BM_THREADS) {
        const Pick p = heads[e];
        if (p.v && bm_rank(heads, n * q, p) == K - 1) bound_s = p;   // places differ: at most one
    }
    __syncthreads();
    const Pick bound = bound_s;                              // {0, 0}: fewer than K heads, everything reaches it
    for (int e = t; e < n * K; e += BM_THREADS) {
        const Pick p = all[e];
        if (p.v && !better(bound, p)) found[atomicAdd(&count, 1)] = p;
    }
    __syncthreads();
    const int c = count;
    for (int e = t; e < c; e += BM_THREADS) {
        const Pick p = found[e];
        const int rank = bm_rank(found, c, p);
        if (rank < K) {
            picked[rank] = (float)bm_value(p.v);
            parents[rank] = (int)(~p.place >> 32);
            tokens[rank] = (int)(uint32_t)~p.place;
        }
    }
    for (int k = c + t; k < K; k += BM_THREADS) {
        picked[k] = -INFINITY;
        parents[k] = tokens[k] = -1;
    }
}

__global__ void __launch_bounds__(BM_THREADS)
beam_merge_kernel(const float* __restrict__ scores, int V, int W, int K, int blocks, const float2* __restrict__ sums,
                  const unsigned long long* __restrict__ lists, float* __restrict__ picked, int* __restrict__ parents,
                  int* __restrict__ tokens) {
    extern __shared__ __align__(16) unsigned char bm_smem[];
    __shared__ float2 sum_s[BM_LISTS];
    pdl_wait();
    const size_t b = blockIdx.x;
    lists += b * blocks * K;
    const int t = threadIdx.x;
    static_assert(BM_LISTS == BM_THREADS, "a thread a sum");
    const float score = bs_score(scores + b * W, W);         // these three at once
    const unsigned long long first = t < blocks * K ? lists[t] : 0;
    if (t < blocks) sum_s[t] = sums[b * blocks + t];
    const BeamShare share(score, W, V, blocks);
    __syncthreads();
    bm_join(share, K, sum_s, lists, first, bm_smem, picked + b * K, parents + b * K, tokens + b * K);
}

// Bytes of shared memory to join up to so many lists: candidates, heads (at most 3 K - 1 and one a list), and those that
// reach the bound.
__host__ __device__ static constexpr size_t beam_merge_bytes(int lists, int K) {
    return ((size_t)lists * (2 * K + 1) + 3 * K - 1) * sizeof(Pick);
}

// Both at once: a cluster of sixteen blocks a request; the slices' sums and lists go to the first block's shared memory,
// which joins them.
#define BC_BLOCKS 16
#define BC_ROOM (beam_merge_bytes(BC_BLOCKS, BS_MAX_K) > BS_BUF * 8 ? beam_merge_bytes(BC_BLOCKS, BS_MAX_K) : BS_BUF * 8)

template <typename T> __device__ __forceinline__ T* bc_first(T* mine) {      // the first block's
    T* theirs;
    asm("mapa.u64 %0, %1, 0;" : "=l"(theirs) : "l"(mine));
    return theirs;
}

__global__ void __launch_bounds__(BS_THREADS, BS_BLOCKS)
beam_cluster_kernel(const float* __restrict__ logits, long long stride, int V, const float* __restrict__ scores, int W, int K,
                    float* __restrict__ picked, int* __restrict__ parents, int* __restrict__ tokens) {
    __shared__ __align__(16) unsigned char room[BC_ROOM];    // the scan's buffer, then what joining takes
    __shared__ unsigned long long lists[BC_BLOCKS * BS_MAX_K];
    __shared__ float2 sums[BC_BLOCKS];
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    pdl_wait();
    const int block = blockIdx.x % BC_BLOCKS;
    const size_t b = blockIdx.x / BC_BLOCKS;
    const BeamShare share(bs_score(scores + b * W, W), W, V, BC_BLOCKS);
    asm volatile("barrier.cluster.wait;" ::: "memory");      // the first block is there
    share.scan(logits, stride, b * W, V, K, block, (unsigned long long*)room, bc_first(sums + block), bc_first(lists + block * K));
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (block == 0) bm_join(share, K, sums, lists, threadIdx.x < BC_BLOCKS * BS_MAX_K ? lists[threadIdx.x] : 0, room, picked + b * K, parents + b * K, tokens + b * K);
}

// Slices of a row: the count that is cheapest by a small model. The blocks run in rounds of four a multiprocessor; a
// block costs a unit a turn and three to begin and end.
static int beam_parts(int rows, int W, int V, int K, int sms) {
    const int tiles = (V + 3 + 4 * BS_TILE - 1) / (4 * BS_TILE);
    const int most = BM_CANDIDATES / (W * K) < BM_LISTS / W ? BM_CANDIDATES / (W * K) : BM_LISTS / W;
    long long best = -1;
    int turns = tiles;
    for (int p = 1; p <= most && p <= tiles; ++p) {
        const int n = (tiles + p - 1) / p;
        const long long rounds = ((long long)rows * p + BS_BLOCKS * sms - 1) / (BS_BLOCKS * sms), cost = rounds * (n + 3);
        if (best < 0 || cost < best) { best = cost; turns = n; }
    }
    return (tiles + turns - 1) / turns;
}

static bool beam_takes(int requests, int beams, int V, int K) {
    return requests > 0 && beams > 0 && beams <= BS_MAX_BEAMS && K > 0 && K <= BS_MAX_K && V > 0 && V <= 0x7fffffff - 8 &&
           (long long)requests * beams <= 65535;
}

static int beam_cluster(const float* logits, long long stride, const float* scores, int requests, int beams, int V, int K, float* picked,
                        int* parents, int* tokens, int dev, cudaStream_t stream) {
    static bool sized[64] = {};                              // per device
    if (!sized[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(beam_cluster_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        sized[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)requests * BC_BLOCKS);
    cfg.blockDim = dim3(BS_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = BC_BLOCKS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tgo_pdl_enabled() ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, beam_cluster_kernel, logits, stride, V, scores, beams, K, picked, parents, tokens);
}

static int beam_forced = 0;                                  // for tests: 1 two kernels, 2 clusters; 0: by the rule
TGO_API void tgo_beam_force_way(int way) { beam_forced = way; }
// Whether a call goes by clusters: one launch and no workspace, 5.5 us of the host's time where two kernels take 10, but only
// sixteen blocks a request. So where two turns of each are enough and no multiprocessor has more than two blocks. MEASURED
// (us on the device, clusters / two kernels), 32768 tokens: 1 x 1 beams 6.1 / 6.6, 1 x 4 7.7 / 8.1, 16 x 4 9.0 / 9.8, 32 x 4 13.5 /
// 11.5, 16 x 5 (three turns) 10.9 / 10.6, 1 x 8 10.6 / 10.4; 151936 tokens: 1 x 1 (three turns) 8.2 / 7.4, 1 x 4 13.9 / 11.3.
static bool beam_by_clusters(int requests, int beams, int V) {
    if (beams > BC_BLOCKS) return false;
    if (beam_forced) return beam_forced == 2;
    const int parts = BC_BLOCKS / beams, tiles = (V + 4 * BS_TILE - 1) / (4 * BS_TILE);
    return requests * BC_BLOCKS <= 2 * tgo_multiprocessors() && (tiles + parts - 1) / parts <= 2;
}

// 64-bit numbers of workspace that a call needs (a call by clusters none); a refused one 0.
TGO_API int tgo_beam_select_work(int requests, int beams, int V, int K) {
    if (!beam_takes(requests, beams, V, K) || beam_by_clusters(requests, beams, V)) return 0;
    const long long n = (long long)requests * beams * beam_parts(requests * beams, beams, V, K, tgo_multiprocessors()) * (1 + K);
    return n > 0x7fffffff ? 0 : (int)n;
}

// picked, parents, tokens [requests, K]; scores [requests, beams]; logits rows `stride` floats apart, beams of
// a request one after the other. `work`: as above, `work_longs` of them.
TGO_API int tgo_beam_select(const float* logits, long long stride, const float* scores, int requests, int beams, int V,
                            int K, float* picked, int* parents, int* tokens, void* work, int work_longs,
                            cudaStream_t stream) {
    if (requests <= 0) return 0;
    if (!beam_takes(requests, beams, V, K)) return TGO_E_BAD_ARG;
    static bool sized[64] = {};                              // per device
    int dev = 0;
    const cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return (int)err;
    if (dev < 0 || dev >= 64) return TGO_E_BAD_ARG;
    if (beam_by_clusters(requests, beams, V))
        return beam_cluster(logits, stride, scores, requests, beams, V, K, picked, parents, tokens, dev, stream);
    const int blocks = beams * beam_parts(requests * beams, beams, V, K, tgo_multiprocessors());       // of a request
    if (work_longs < (long long)requests * blocks * (1 + K)) return TGO_E_BAD_ARG;
    if (!sized[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   200 * 1024);
        if (e != cudaSuccess) return (int)e;
        sized[dev] = true;
    }
    float2* sums = (float2*)work;
    unsigned long long* lists = (unsigned long long*)(sums + (size_t)requests * blocks);
    const int rc = tgo_launch_pdl(beam_part_kernel, dim3(blocks, requests), dim3(BS_THREADS), 0, stream, logits, stride, V,
                                  scores, beams, K, sums, lists);
    if (rc) return rc;
    return tgo_launch_pdl(beam_merge_kernel, dim3(requests), dim3(BM_THREADS), beam_merge_bytes(blocks, K), stream, scores, V, beams, K,
                          blocks, (const float2*)sums, (const unsigned long long*)lists, picked, parents, tokens);
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

template <typename VEC, int W, bool AHEAD>
__global__ void __launch_bounds__(RR_THREADS)
reorder_rows_kernel(const __grid_constant__ ReorderRows d, const int* __restrict__ index, const int* __restrict__ parents,
                    int beams, int run) {
    __shared__ long long to[RR_MAX_BEAMS], from[RR_MAX_BEAMS];       // byte offsets; from < 0: the row stays
    pdl_wait();
    const int k = blockIdx.z, g = blockIdx.y, t = threadIdx.x;
    const long long vectors = d.row_bytes[k] / (long long)sizeof(VEC);
    // pieces of RR_THREADS vectors of a row of every outer block, one after the other
    const int pieces = (int)((vectors + RR_THREADS - 1) / RR_THREADS), last = min((int)blockIdx.x * run + run, pieces * d.outer[k]);
    int i = blockIdx.x * run;
    if (i >= last) return;
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
    int o = i / pieces, c = i - o * pieces;
    VEC got[AHEAD ? 2 : 1][W];
    char* base;
    bool mine;
    auto load = [&](VEC* into) {
        const long long v = (long long)c * RR_THREADS + t;
        base = d.base[k] + o * d.outer_stride[k] + v * (long long)sizeof(VEC);
        mine = v < vectors;
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (mine && w < beams && from[w] >= 0) into[w] = *(const VEC*)(base + from[w]);
    };
    auto store = [&](const VEC* what, char* at, bool had) {
#pragma unroll
        for (int w = 0; w < W; ++w)
            if (had && w < beams && from[w] >= 0) *(VEC*)(at + to[w]) = what[w];
    };
    load(got[0]);
    if constexpr (!AHEAD) store(got[0], base, mine);         // run is 1
    else {
        // the next piece is read before this one is written
        auto step = [&](VEC* now, VEC* next) {
            char* const at = base;
            const bool had = mine;
            if (++c == pieces) { c = 0; ++o; }
            if (++i < last) load(next);
            store(now, at, had);
        };
        while (true) {
            step(got[0], got[1]);
            if (i >= last) break;
            step(got[1], got[0]);
            if (i >= last) break;
        }
    }
}

// Two pieces a block where that still leaves every multiprocessor two rounds of blocks, and up to 64 bytes of a piece a
// thread: finding the rows costs a block two reads that wait for each other. MEASURED (us, one piece, two, four): 16 groups of 4
// pages of 36 layers, three of each moved, 33.4, 32.4 (5.8 TB/s), 32.9; 8 groups of 4 states of 8 MB, three moved, 107.5, 101.8 (6.6 TB/s), 104.4; 1
// group of 4 pages of 8 layers 2.0, 2.3, 2.9.
template <typename VEC, int W>
static int reorder_of(const ReorderRows& d, int tensors, int groups, int beams, long long blocks, const int* index,
                      const int* parents, cudaStream_t stream) {
    if constexpr (W * sizeof(VEC) <= 64)
        if (blocks * groups * tensors >= 2ll * 2 * 8 * tgo_multiprocessors())
            return tgo_launch_pdl(reorder_rows_kernel<VEC, W, true>, dim3((unsigned)((blocks + 1) / 2), groups, tensors), dim3(RR_THREADS), 0, stream, d,
                                  index, parents, beams, 2);
    return tgo_launch_pdl(reorder_rows_kernel<VEC, W, false>, dim3((unsigned)blocks, groups, tensors), dim3(RR_THREADS), 0, stream, d, index,
                          parents, beams, 1);
}

template <typename VEC>
static int reorder_launch(const ReorderRows& d, int tensors, int groups, int beams, long long blocks, const int* index,
                          const int* parents, cudaStream_t stream) {
    if (beams <= 4) return reorder_of<VEC, 4>(d, tensors, groups, beams, blocks, index, parents, stream);
    if (beams <= 8) return reorder_of<VEC, 8>(d, tensors, groups, beams, blocks, index, parents, stream);
    if (beams <= 16) return reorder_of<VEC, 16>(d, tensors, groups, beams, blocks, index, parents, stream);
    return reorder_of<VEC, 32>(d, tensors, groups, beams, blocks, index, parents, stream);
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
        if (blocks > 0x7fffff00) return TGO_E_BAD_ARG;
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
