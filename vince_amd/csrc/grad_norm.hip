// The 2-norm over many gradient tensors, clipping to a largest norm, and the SGD step that takes the clipping coefficient from device
// memory (include/vince_hip.h has the formulas).  A table in device memory lists the tensors in pieces of a few thousand elements.
// Squares of fp32 / bf16 values are exact in fp64 and their fp64 sum neither overflows nor underflows, whatever the gradients' scale.
#include "common.h"

namespace {

// Pieces of 2048 .. 16384 elements: small enough that a few hundred thousand elements reach every CU, large enough that the entries are
// nothing beside what they list.
constexpr int GRAD_CHUNK_MIN = 2048, GRAD_CHUNK_MAX = 16384;
// Up to two pieces a wavefront of one workgroup (grad_small_kernel).  us on the device of clipping in that one launch / in two, 16, 32 and
// 64 pieces of 2048 fp32 values: 3.8 / 5.0, 4.9 / 5.1, 7.2 / 5.1.
constexpr int SMALL_CHUNKS = 32;
// Workgroups: 8 MB of loads in flight where only gradients are read, 4 MB where they are written back too, 6 MB in the SGD step's three
// streams.  us at 256 / 512 / 1024 / 2048 of them, 160 M fp32: norm 128 / 109 / 110 / 113 (5.9 TB/s at 512), scaling 226 / 253 / 249 / 248;
// norm and SGD step of 28 M 123 / 113 / 118 / 118.
constexpr int GRAD_NORM_BLOCKS = 512, GRAD_SCALE_BLOCKS = 256, SGD_BLOCKS = 512;
constexpr uint32_t GRAD_BF16 = 1u << 31;

struct GradChunk {
    uint64_t data;
    uint32_t n;        // elements, | GRAD_BF16
    float scale;
};
static_assert(sizeof(GradChunk) == 16, "the table's layout is the header's");

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double red[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// 16 bytes from an address aligned to the element only (the hardware takes any; the type tells the compiler so).  The table's addresses
// are device memory: said to the compiler too, which would otherwise make flat accesses of them.
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_any_t;
typedef __attribute__((address_space(1))) u32x4_any_t global_u32x4_any_t;
__device__ __forceinline__ uint4 load16(const void* p) {
    const u32x4_any_t v = *(const global_u32x4_any_t*)p;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store16(void* p, const uint4& v) {
    const u32x4_any_t w = {v.x, v.y, v.z, v.w};
    *(global_u32x4_any_t*)p = w;
}

// this thread's share of a piece's sum of squares; THREADS of them, `thread` the number of this one
template <int THREADS, typename T> __device__ __forceinline__ double squares_of(const T* __restrict__ g, int n, int thread) {
    constexpr int V = Elem<T>::CH, STEP = THREADS * V, DEEP = 4;
    double s0 = 0.0, s1 = 0.0;
    int i = thread * V;
    for (; i + (DEEP - 1) * STEP + V <= n; i += DEEP * STEP) {       // DEEP loads are in flight before the first is used
        uint4 q[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) q[d] = load16(g + i + d * STEP);
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            float f[V];
            Chunk<T>::unpack(q[d], f);
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                s0 = fma((double)f[e], (double)f[e], s0);
                s1 = fma((double)f[e + 1], (double)f[e + 1], s1);
            }
        }
    }
    for (; i < n; i += STEP) {
        if (i + V <= n) {
            float f[V];
            Chunk<T>::unpack(load16(g + i), f);
#pragma unroll
            for (int e = 0; e < V; ++e) s0 = fma((double)f[e], (double)f[e], s0);
        } else {
            for (int j = i; j < n; ++j) {
                const double v = to_float(g[j]);
                s1 = fma(v, v, s1);
            }
        }
    }
    return s0 + s1;
}

__global__ __launch_bounds__(256) void grad_squares_kernel(const GradChunk* __restrict__ table, int64_t chunks, double* __restrict__ partial) {
    double sum = 0.0;
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const GradChunk k = table[c];
        const int n = (int)(k.n & ~GRAD_BF16);
        const double s = k.n & GRAD_BF16 ? squares_of<256>((const bf16_t*)k.data, n, threadIdx.x) : squares_of<256>((const float*)k.data, n, threadIdx.x);
        sum = fma((double)k.scale * (double)k.scale, s, sum);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// [norm, coefficient] from the workgroups' sums, by every thread of a workgroup of 256: norm = sqrt(sum), coefficient =
// min(1, max_norm / (norm + 1e-6)); an infinite max_norm clips nothing, a NaN norm gives a NaN coefficient
__device__ __forceinline__ float2 clip_of(double sum, float max_norm) {
    const double norm = sqrt(sum), c = (double)max_norm / (norm + 1e-6);
    return make_float2((float)norm, max_norm == INFINITY || c > 1.0 ? 1.f : (float)c);
}
__device__ __forceinline__ float2 clip_of(const double* __restrict__ partial, int n, float max_norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
    return clip_of(block_sum(s), max_norm);
}

__global__ __launch_bounds__(256) void grad_clip_kernel(const double* __restrict__ partial, int n, float max_norm, float* __restrict__ clip) {
    const float2 r = clip_of(partial, n, max_norm);
    if (threadIdx.x == 0) { clip[0] = r.x; clip[1] = r.y; }
}

template <int THREADS, typename T> __device__ __forceinline__ void scale_piece(T* __restrict__ g, int n, float f, int thread) {
    constexpr int V = Elem<T>::CH, STEP = THREADS * V, DEEP = 4;
    int i = thread * V;
    for (; i + (DEEP - 1) * STEP + V <= n; i += DEEP * STEP) {
        uint4 q[DEEP];
#pragma unroll
        for (int d = 0; d < DEEP; ++d) q[d] = load16(g + i + d * STEP);
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            float v[V];
            Chunk<T>::unpack(q[d], v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] *= f;
            store16(g + i + d * STEP, Chunk<T>::pack(v));
        }
    }
    for (; i < n; i += STEP) {
        if (i + V <= n) {
            float v[V];
            Chunk<T>::unpack(load16(g + i), v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] *= f;
            store16(g + i, Chunk<T>::pack(v));
        } else {
            for (int j = i; j < n; ++j) put(g + j, to_float(g[j]) * f);
        }
    }
}

// FINAL: the coefficient comes from the sums of grad_squares_kernel, added up by every workgroup for itself (4 KB at most, in the
// caches) -- one launch fewer than a kernel of its own for it; else from clip[1]
template <bool FINAL>
__global__ __launch_bounds__(256) void grad_scale_kernel(const GradChunk* __restrict__ table, int64_t chunks, float* __restrict__ clip,
                                                         const double* __restrict__ partial, int n_partial, float max_norm) {
    float f;
    if constexpr (FINAL) {
        const float2 r = clip_of(partial, n_partial, max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) { clip[0] = r.x; clip[1] = r.y; }
        f = r.y;
    } else {
        f = clip[1];
    }
    if (f == 1.f) return;                  // every product would be the gradient itself
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const GradChunk k = table[c];
        const int n = (int)(k.n & ~GRAD_BF16);
        if (k.n & GRAD_BF16) scale_piece<256>((bf16_t*)k.data, n, f, threadIdx.x);
        else scale_piece<256>((float*)k.data, n, f, threadIdx.x);
    }
}

// Few pieces (SMALL_CHUNKS): everything in one workgroup, a piece to a wavefront, and in one launch without scratch.
template <bool SCALE>
__global__ __launch_bounds__(1024) void grad_small_kernel(const GradChunk* __restrict__ table, int chunks, float max_norm, float* __restrict__ clip) {
    __shared__ double red[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double sum = 0.0;
    for (int c = wave; c < chunks; c += 16) {
        const GradChunk k = table[c];
        const int n = (int)(k.n & ~GRAD_BF16);
        const double s = k.n & GRAD_BF16 ? squares_of<64>((const bf16_t*)k.data, n, lane) : squares_of<64>((const float*)k.data, n, lane);
        sum = fma((double)k.scale * (double)k.scale, s, sum);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += red[i];
    const float2 r = clip_of(sum, max_norm);
    if (threadIdx.x == 0) { clip[0] = r.x; clip[1] = r.y; }
    if constexpr (SCALE) {
        if (r.y == 1.f) return;
        for (int c = wave; c < chunks; c += 16) {        // (the pieces that this wavefront itself has read)
            const GradChunk k = table[c];
            const int n = (int)(k.n & ~GRAD_BF16);
            if (k.n & GRAD_BF16) scale_piece<64>((bf16_t*)k.data, n, r.y, lane);
            else scale_piece<64>((float*)k.data, n, r.y, lane);
        }
    }
}

// sgd_kernel (misc.hip) with the scale of the gradient taken from device memory: the same operations in the same order.  The momentum
// passes the Infinity Cache by (non-temporal both ways; nothing reads it before the next step), which leaves the gradients there that the
// norm has just read, and the parameters for the average and the weight copies that follow: norm and step of 28 M parameters 124 -> 113 us,
// with the key encoder's average behind them 176 -> 167.
typedef __attribute__((ext_vector_type(4))) float f32x4_nt_t;
__global__ __launch_bounds__(256) void sgd_clip_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ buf, int64_t n,
                                                       float lr, float mom, float wd, float grad_scale, const float* __restrict__ clip) {
    const float gs = grad_scale * clip[1];
    const int64_t n4 = n >> 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
        float4 pv = ((float4*)p)[i];
        const float4 gv = ((const float4*)g)[i];
        f32x4_nt_t bq = __builtin_nontemporal_load((const f32x4_nt_t*)buf + i);
        float4 bv = make_float4(bq[0], bq[1], bq[2], bq[3]);
        float d;
        d = fmaf(wd, pv.x, gv.x * gs); bv.x = fmaf(bv.x, mom, d); pv.x = fmaf(-lr, bv.x, pv.x);
        d = fmaf(wd, pv.y, gv.y * gs); bv.y = fmaf(bv.y, mom, d); pv.y = fmaf(-lr, bv.y, pv.y);
        d = fmaf(wd, pv.z, gv.z * gs); bv.z = fmaf(bv.z, mom, d); pv.z = fmaf(-lr, bv.z, pv.z);
        d = fmaf(wd, pv.w, gv.w * gs); bv.w = fmaf(bv.w, mom, d); pv.w = fmaf(-lr, bv.w, pv.w);
        ((float4*)p)[i] = pv;
        bq = (f32x4_nt_t){bv.x, bv.y, bv.z, bv.w};
        __builtin_nontemporal_store(bq, (f32x4_nt_t*)buf + i);
    }
    if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
        const int64_t i = (n4 << 2) + threadIdx.x;
        const float d = fmaf(wd, p[i], g[i] * gs);
        const float b = fmaf(buf[i], mom, d);
        buf[i] = b;
        p[i] = fmaf(-lr, b, p[i]);
    }
}

int blocks_of(int64_t chunks, int most) { return (int)(chunks < most ? chunks : most); }
int64_t chunk_of(const vince_grad_tensor* tensors, int32_t count) {
    int64_t total = 0, chunk = GRAD_CHUNK_MIN;
    for (int32_t i = 0; i < count; ++i) total += tensors[i].n;
    while (chunk < GRAD_CHUNK_MAX && chunk * 2 * GRAD_NORM_BLOCKS <= total) chunk *= 2;
    return chunk;
}

}  // namespace

extern "C" int64_t vince_grad_table_chunks(const vince_grad_tensor* tensors, int32_t count) {
    VINCE_CHECK_ARG(count >= 0 && (tensors || count == 0), VINCE_E_ARG, "vince_grad_table_chunks: bad arguments");
    int64_t chunks = 0;
    for (int32_t i = 0; i < count; ++i) {
        const vince_grad_tensor& t = tensors[i];
        VINCE_CHECK_ARG(t.dtype == VINCE_F32 || t.dtype == VINCE_BF16, VINCE_E_DTYPE, "vince_grad_table: tensor %d: dtype %d (VINCE_F32 or VINCE_BF16)",
                        i, t.dtype);
        VINCE_CHECK_ARG(t.n >= 0 && (t.data || t.n == 0), VINCE_E_ARG, "vince_grad_table: tensor %d: n=%lld", i, (long long)t.n);
        VINCE_CHECK_ARG(((uintptr_t)t.data & (t.dtype == VINCE_F32 ? 3 : 1)) == 0, VINCE_E_ALIGN, "vince_grad_table: tensor %d is not aligned to its elements", i);
        VINCE_CHECK_ARG(t.scale - t.scale == 0.f, VINCE_E_ARG, "vince_grad_table: tensor %d: scale %g", i, (double)t.scale);
    }
    const int64_t chunk = chunk_of(tensors, count);
    for (int32_t i = 0; i < count; ++i) chunks += tensors[i].n / chunk + (tensors[i].n % chunk != 0);
    return chunks;
}

extern "C" int vince_grad_table_fill(const vince_grad_tensor* tensors, int32_t count, void* table, int64_t chunks) {
    const int64_t want = vince_grad_table_chunks(tensors, count);
    if (want < 0) return (int)want;
    VINCE_CHECK_ARG(chunks == want && (table || chunks == 0), VINCE_E_ARG, "vince_grad_table_fill: %lld entries, not %lld", (long long)chunks, (long long)want);
    GradChunk* c = (GradChunk*)table;
    const int64_t chunk = chunk_of(tensors, count);
    for (int32_t i = 0; i < count; ++i) {
        const vince_grad_tensor& t = tensors[i];
        const uint64_t size = t.dtype == VINCE_F32 ? 4 : 2;
        for (int64_t at = 0; at < t.n; at += chunk, ++c) {
            c->data = (uint64_t)(uintptr_t)t.data + (uint64_t)at * size;
            c->n = (uint32_t)(t.n - at < chunk ? t.n - at : chunk) | (t.dtype == VINCE_BF16 ? GRAD_BF16 : 0u);
            c->scale = t.scale;
        }
    }
    return VINCE_OK;
}

extern "C" size_t vince_grad_norm_scratch_bytes(int64_t chunks) {
    return chunks > SMALL_CHUNKS ? (size_t)blocks_of(chunks, GRAD_NORM_BLOCKS) * sizeof(double) : 0;
}

#define GRAD_NORM_CHECK(name)                                                                                                              \
    VINCE_CHECK_ARG(chunks >= 0 && clip && (chunks == 0 || table) && (chunks <= SMALL_CHUNKS || scratch), VINCE_E_ARG, name ": bad arguments"); \
    VINCE_CHECK_ARG(max_norm >= 0.f, VINCE_E_ARG, name ": max_norm=%g", (double)max_norm);                                                 \
    VINCE_CHECK_ARG(scratch_bytes >= vince_grad_norm_scratch_bytes(chunks), VINCE_E_ARG, name ": scratch of %zu bytes", scratch_bytes)

extern "C" int vince_grad_norm(const void* table, int64_t chunks, float max_norm, float* clip, void* scratch, size_t scratch_bytes, void* stream) {
    GRAD_NORM_CHECK("vince_grad_norm");
    if (chunks <= SMALL_CHUNKS) {
        hipLaunchKernelGGL(grad_small_kernel<false>, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const GradChunk*)table, (int)chunks, max_norm, clip);
        VINCE_CHECK_LAUNCH();
        return VINCE_OK;
    }
    const int blocks = blocks_of(chunks, GRAD_NORM_BLOCKS);
    hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks, (double*)scratch);
    hipLaunchKernelGGL(grad_clip_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)scratch, blocks, max_norm, clip);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" int vince_grad_scale(const void* table, int64_t chunks, const float* clip, void* stream) {
    VINCE_CHECK_ARG(chunks >= 0 && clip && (chunks == 0 || table), VINCE_E_ARG, "vince_grad_scale: bad arguments");
    if (chunks == 0) return VINCE_OK;
    hipLaunchKernelGGL(grad_scale_kernel<false>, dim3(blocks_of(chunks, GRAD_SCALE_BLOCKS)), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks,
                       (float*)clip, (const double*)nullptr, 0, 0.f);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" int vince_grad_clip(const void* table, int64_t chunks, float max_norm, float* clip, void* scratch, size_t scratch_bytes, void* stream) {
    GRAD_NORM_CHECK("vince_grad_clip");
    if (chunks <= SMALL_CHUNKS) {
        hipLaunchKernelGGL(grad_small_kernel<true>, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const GradChunk*)table, (int)chunks, max_norm, clip);
        VINCE_CHECK_LAUNCH();
        return VINCE_OK;
    }
    const int blocks = blocks_of(chunks, GRAD_NORM_BLOCKS);
    hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks, (double*)scratch);
    hipLaunchKernelGGL(grad_scale_kernel<true>, dim3(blocks_of(chunks, GRAD_SCALE_BLOCKS)), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks, clip,
                       (const double*)scratch, blocks, max_norm);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" int vince_sgd_flat_clip(float* param, const float* grad, float* buf, int64_t n, float lr, float momentum, float weight_decay,
                                   float grad_scale, const float* clip, void* stream) {
    VINCE_CHECK_ARG(param && grad && buf && clip && n > 0, VINCE_E_ARG, "vince_sgd_flat_clip: bad arguments");
    VINCE_CHECK_ARG((((uintptr_t)param | (uintptr_t)grad | (uintptr_t)buf) & 15) == 0, VINCE_E_ALIGN,
                    "vince_sgd_flat_clip: pointers must be 16-byte aligned");
    const int64_t blocks = (n / 4 + 256) / 256;
    hipLaunchKernelGGL(sgd_clip_kernel, dim3((unsigned)(blocks < SGD_BLOCKS ? blocks : SGD_BLOCKS)), dim3(256), 0, (hipStream_t)stream, param, grad, buf, n, lr,
                       momentum, weight_decay, grad_scale, clip);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}
