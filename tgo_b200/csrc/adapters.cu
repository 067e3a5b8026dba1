// Low-rank adapters of many requests beside a shared projection.
//
// Row t of a batch with adapter i = ids[t]:
//   u[t, s, j] = scale_i sum_k x[t, k] A_i[s, j, k],    out[t, n] = y[t, n] + sum_j u[t, s(n), j] B_i[n, j],
// y being the projection's own result and s(n) the slice of its columns that n lies in (q, k and v of a
// joined matrix; gate and up rows in eights): each slice has an A of its own. A row whose id names no
// adapter keeps y. u is held in 32 bits.
#include "common.cuh"

#define LR_MAX_SLICES 4

struct LowRankColumns {
    int ends[LR_MAX_SLICES];      // the column after each slice's last
    int slices;
    int interleaved;              // eight columns of slice 0, eight of slice 1, and so on
};

__device__ __forceinline__ int lr_slice(const LowRankColumns& c, int n) {
    if (c.interleaved) return (n >> 3) & 1;
    int s = 0;
#pragma unroll
    for (int i = 0; i < LR_MAX_SLICES - 1; ++i) s += (i + 1 < c.slices && n >= c.ends[i]);
    return s;
}

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

template <typename T, typename TY>
static int low_rank_launch(const void* x, long long x_stride, const void* y, long long y_stride, void* out,
                           long long out_stride, const void* a, const void* b, const float* scale, const int* ids, int T_,
                           int K, int N, int adapters, int rank, const LowRankColumns& columns, float* u,
                           cudaStream_t stream) {
    const int width = columns.slices * rank;
    int rc = tgo_launch_pdl(low_rank_down_kernel<T>, dim3(T_, (width + 31) / 32), dim3(256), 0, stream, (const T*)x, x_stride,
                            (const T*)a, scale, ids, adapters, width, K, u);
    if (rc) return rc;
    return tgo_launch_pdl(low_rank_up_kernel<T, TY>, dim3(T_, (N + 255) / 256), dim3(256), 0, stream, (const float*)u,
                          (const T*)b, ids, adapters, rank, columns, N, (const TY*)y, y_stride, (TY*)out, out_stride);
}

// x [T, K] of type dt, y and out [T, N] of type dt_y, rows strided; out may be y. a [adapters, slices, rank, K],
// b [adapters, N, rank] of type dt; ends: the column after each slice's last. work: T x slices x rank floats.
TGO_API int tgo_low_rank_add(const void* x, long long x_stride, const void* y, long long y_stride, void* out,
                             long long out_stride, const void* a, const void* b, const float* scale, const int* ids,
                             int dt, int dt_y, int T, int K, int N, int adapters, int rank, int slices, const int* ends,
                             int interleaved, float* work, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (K <= 0 || N <= 0 || adapters <= 0 || rank <= 0 || slices <= 0 || slices > LR_MAX_SLICES || (N + 255) / 256 > 65535 ||
        (interleaved && (slices != 2 || N % 16)))
        return TGO_E_BAD_ARG;
    LowRankColumns c = {};
    c.slices = slices;
    c.interleaved = interleaved;
    for (int i = 0; i < slices; ++i) c.ends[i] = ends[i];
    if (dt == TGO_F32 && dt_y == TGO_F32)
        return low_rank_launch<float, float>(x, x_stride, y, y_stride, out, out_stride, a, b, scale, ids, T, K, N, adapters,
                                             rank, c, work, stream);
    if (dt == TGO_BF16 && dt_y == TGO_BF16)
        return low_rank_launch<bf16, bf16>(x, x_stride, y, y_stride, out, out_stride, a, b, scale, ids, T, K, N, adapters,
                                           rank, c, work, stream);
    if (dt == TGO_BF16 && dt_y == TGO_F32)
        return low_rank_launch<bf16, float>(x, x_stride, y, y_stride, out, out_stride, a, b, scale, ids, T, K, N, adapters,
                                            rank, c, work, stream);
    return TGO_E_BAD_ARG;
}
