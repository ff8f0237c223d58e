// The 2-norm over many gradient tensors, clipping to a largest norm, and the SGD step that takes the clipping coefficient from device
// memory (include/vince_hip.h has the formulas).  A table in device memory lists the tensors in pieces of at most GRAD_CHUNK elements.
// Squares of fp32 / bf16 values are exact in fp64 and their fp64 sum neither overflows nor underflows, whatever the gradients' scale.
#include "common.h"

namespace {

constexpr int GRAD_CHUNK = 16384;
constexpr int GRAD_BLOCKS = 1024;      // 4 workgroups a CU
constexpr uint32_t GRAD_BF16 = 1u << 31;

struct GradChunk {
    uint64_t data;
    uint32_t n;        // elements, | GRAD_BF16
    float scale;
};
static_assert(sizeof(GradChunk) == 16, "the table's layout is the header's");

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double red[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void grad_squares_kernel(const GradChunk* __restrict__ table, int64_t chunks, double* __restrict__ partial) {
    double sum = 0.0;
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const GradChunk k = table[c];
        const int n = (int)(k.n & ~GRAD_BF16);
        double s = 0.0;
        if (k.n & GRAD_BF16) {
            const bf16_t* g = (const bf16_t*)k.data;
            for (int i = threadIdx.x; i < n; i += 256) { const double v = bf16_to_f32(g[i]); s = fma(v, v, s); }
        } else {
            const float* g = (const float*)k.data;
            for (int i = threadIdx.x; i < n; i += 256) { const double v = g[i]; s = fma(v, v, s); }
        }
        sum = fma((double)k.scale * (double)k.scale, s, sum);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// clip[0] = norm, clip[1] = min(1, max_norm / (norm + 1e-6)); an infinite max_norm clips nothing, a NaN norm gives a NaN coefficient
__global__ __launch_bounds__(256) void grad_clip_kernel(const double* __restrict__ partial, int n, float max_norm, float* __restrict__ clip) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += partial[i];
    s = block_sum(s);
    if (threadIdx.x == 0) {
        const double norm = sqrt(s), c = (double)max_norm / (norm + 1e-6);
        clip[0] = (float)norm;
        clip[1] = max_norm == INFINITY || c > 1.0 ? 1.f : (float)c;
    }
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const GradChunk* __restrict__ table, int64_t chunks, const float* __restrict__ clip) {
    const float f = clip[1];
    if (f == 1.f) return;                  // every product would be the gradient itself
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const GradChunk k = table[c];
        const int n = (int)(k.n & ~GRAD_BF16);
        if (k.n & GRAD_BF16) {
            bf16_t* g = (bf16_t*)k.data;
            for (int i = threadIdx.x; i < n; i += 256) g[i] = f32_to_bf16(bf16_to_f32(g[i]) * f);
        } else {
            float* g = (float*)k.data;
            for (int i = threadIdx.x; i < n; i += 256) g[i] *= f;
        }
    }
}

// sgd_kernel (misc.hip) with the scale of the gradient taken from device memory: the same operations in the same order
__global__ __launch_bounds__(256) void sgd_clip_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ buf, int64_t n,
                                                       float lr, float mom, float wd, float grad_scale, const float* __restrict__ clip) {
    const float gs = grad_scale * clip[1];
    const int64_t n4 = n >> 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
        float4 pv = ((float4*)p)[i];
        const float4 gv = ((const float4*)g)[i];
        float4 bv = ((float4*)buf)[i];
        float d;
        d = fmaf(wd, pv.x, gv.x * gs); bv.x = fmaf(bv.x, mom, d); pv.x = fmaf(-lr, bv.x, pv.x);
        d = fmaf(wd, pv.y, gv.y * gs); bv.y = fmaf(bv.y, mom, d); pv.y = fmaf(-lr, bv.y, pv.y);
        d = fmaf(wd, pv.z, gv.z * gs); bv.z = fmaf(bv.z, mom, d); pv.z = fmaf(-lr, bv.z, pv.z);
        d = fmaf(wd, pv.w, gv.w * gs); bv.w = fmaf(bv.w, mom, d); pv.w = fmaf(-lr, bv.w, pv.w);
        ((float4*)p)[i] = pv;
        ((float4*)buf)[i] = bv;
    }
    if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
        const int64_t i = (n4 << 2) + threadIdx.x;
        const float d = fmaf(wd, p[i], g[i] * gs);
        const float b = fmaf(buf[i], mom, d);
        buf[i] = b;
        p[i] = fmaf(-lr, b, p[i]);
    }
}

int grad_blocks(int64_t chunks) { return (int)(chunks < GRAD_BLOCKS ? chunks : GRAD_BLOCKS); }

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
        chunks += t.n / GRAD_CHUNK + (t.n % GRAD_CHUNK != 0);
    }
    return chunks;
}

extern "C" int vince_grad_table_fill(const vince_grad_tensor* tensors, int32_t count, void* table, int64_t chunks) {
    const int64_t want = vince_grad_table_chunks(tensors, count);
    if (want < 0) return (int)want;
    VINCE_CHECK_ARG(chunks == want && (table || chunks == 0), VINCE_E_ARG, "vince_grad_table_fill: %lld entries, not %lld", (long long)chunks, (long long)want);
    GradChunk* c = (GradChunk*)table;
    for (int32_t i = 0; i < count; ++i) {
        const vince_grad_tensor& t = tensors[i];
        const uint64_t size = t.dtype == VINCE_F32 ? 4 : 2;
        for (int64_t at = 0; at < t.n; at += GRAD_CHUNK, ++c) {
            c->data = (uint64_t)(uintptr_t)t.data + (uint64_t)at * size;
            c->n = (uint32_t)(t.n - at < GRAD_CHUNK ? t.n - at : GRAD_CHUNK) | (t.dtype == VINCE_BF16 ? GRAD_BF16 : 0u);
            c->scale = t.scale;
        }
    }
    return VINCE_OK;
}

extern "C" size_t vince_grad_norm_scratch_bytes(int64_t chunks) { return chunks > 0 ? (size_t)grad_blocks(chunks) * sizeof(double) : 0; }

extern "C" int vince_grad_norm(const void* table, int64_t chunks, float max_norm, float* clip, void* scratch, size_t scratch_bytes, void* stream) {
    VINCE_CHECK_ARG(chunks >= 0 && clip && (chunks == 0 || (table && scratch)), VINCE_E_ARG, "vince_grad_norm: bad arguments");
    VINCE_CHECK_ARG(max_norm >= 0.f, VINCE_E_ARG, "vince_grad_norm: max_norm=%g", (double)max_norm);
    VINCE_CHECK_ARG(scratch_bytes >= vince_grad_norm_scratch_bytes(chunks), VINCE_E_ARG, "vince_grad_norm: scratch of %zu bytes", scratch_bytes);
    const int blocks = grad_blocks(chunks);
    if (blocks > 0)
        hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks, (double*)scratch);
    hipLaunchKernelGGL(grad_clip_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, (const double*)scratch, blocks, max_norm, clip);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" int vince_grad_scale(const void* table, int64_t chunks, const float* clip, void* stream) {
    VINCE_CHECK_ARG(chunks >= 0 && clip && (chunks == 0 || table), VINCE_E_ARG, "vince_grad_scale: bad arguments");
    if (chunks == 0) return VINCE_OK;
    hipLaunchKernelGGL(grad_scale_kernel, dim3(grad_blocks(chunks)), dim3(256), 0, (hipStream_t)stream, (const GradChunk*)table, chunks, clip);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" int vince_grad_clip(const void* table, int64_t chunks, float max_norm, float* clip, void* scratch, size_t scratch_bytes, void* stream) {
    const int rc = vince_grad_norm(table, chunks, max_norm, clip, scratch, scratch_bytes, stream);
    return rc != VINCE_OK ? rc : vince_grad_scale(table, chunks, clip, stream);
}

extern "C" int vince_sgd_flat_clip(float* param, const float* grad, float* buf, int64_t n, float lr, float momentum, float weight_decay,
                                   float grad_scale, const float* clip, void* stream) {
    VINCE_CHECK_ARG(param && grad && buf && clip && n > 0, VINCE_E_ARG, "vince_sgd_flat_clip: bad arguments");
    VINCE_CHECK_ARG((((uintptr_t)param | (uintptr_t)grad | (uintptr_t)buf) & 15) == 0, VINCE_E_ALIGN,
                    "vince_sgd_flat_clip: pointers must be 16-byte aligned");
    const int64_t blocks = (n / 4 + 256) / 256;
    hipLaunchKernelGGL(sgd_clip_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, (hipStream_t)stream, param, grad, buf, n, lr,
                       momentum, weight_decay, grad_scale, clip);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}
