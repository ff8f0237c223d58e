// Layer norm over the last axis of [rows][cols], forward and backward (include/vince_hip.h has the formulas).
// One wavefront a row; the statistics are two-pass (the mean first, then the squares of the centred values), in fp32.
#include "common.h"

namespace {

template <typename T> __device__ __forceinline__ float load1(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return bf16_to_f32(*p);
}
template <typename T> __device__ __forceinline__ void store1(T* p, float v) {
    if constexpr (sizeof(T) == 4) *p = v;
    else *p = f32_to_bf16(v);
}

template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                     T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                     int cols, float eps, int relu) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        const T* xr = x + row * cols;
        T* yr = out + row * cols;
        float s = 0.f;
        for (int64_t i = lane; i < cols; i += 64) s += load1(xr + i);
        const float m = wave_sum(s) / (float)cols;
        float q = 0.f;
        for (int64_t i = lane; i < cols; i += 64) { const float d = load1(xr + i) - m; q = fmaf(d, d, q); }
        const float r = 1.f / sqrtf(wave_sum(q) / (float)cols + eps);
        for (int64_t i = lane; i < cols; i += 64) {
            float y = (load1(xr + i) - m) * r;
            if (w) y = fmaf(y, w[i], b ? b[i] : 0.f);
            if (relu && y < 0.f) y = 0.f;          // (a NaN stays)
            store1(yr + i, y);
        }
        if (lane == 0) { mean[row] = m; rstd[row] = r; }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_dx_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, const T* __restrict__ dout, const T* __restrict__ act,
                                                        T* __restrict__ dx, int64_t rows, int cols) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        const int64_t at = row * cols;
        const float m = mean[row], r = rstd[row];
        float c1 = 0.f, c2 = 0.f;
        for (int64_t i = lane; i < cols; i += 64) {
            float g = load1(dout + at + i);
            if (act && !(load1(act + at + i) > 0.f)) g = 0.f;
            if (w) g *= w[i];
            c1 += g;
            c2 = fmaf(g, (load1(x + at + i) - m) * r, c2);
        }
        c1 = wave_sum(c1) / (float)cols;
        c2 = wave_sum(c2) / (float)cols;
        for (int64_t i = lane; i < cols; i += 64) {
            float g = load1(dout + at + i);
            if (act && !(load1(act + at + i) > 0.f)) g = 0.f;
            if (w) g *= w[i];
            store1(dx + at + i, r * (g - c1 - (load1(x + at + i) - m) * r * c2));
        }
    }
}

// sums over the rows [y * per, (y + 1) * per) of 64 columns: partial [part][2][cols]
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_dw_kernel(const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                        const T* __restrict__ dout, const T* __restrict__ act, float* __restrict__ partial,
                                                        int64_t rows, int cols, int64_t per) {
    __shared__ float red[2][4][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + tx;
    const int64_t r0 = (int64_t)blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float dw = 0.f, db = 0.f;
    if (c < cols)
        for (int64_t row = r0 + ty; row < r1; row += 4) {
            const int64_t i = row * cols + c;
            float g = load1(dout + i);
            if (act && !(load1(act + i) > 0.f)) g = 0.f;
            db += g;
            dw = fmaf(g, (load1(x + i) - mean[row]) * rstd[row], dw);
        }
    red[0][ty][tx] = dw;
    red[1][ty][tx] = db;
    __syncthreads();
    if (ty < 2 && c < cols)
        partial[((int64_t)blockIdx.y * 2 + ty) * cols + c] = red[ty][0][tx] + red[ty][1][tx] + red[ty][2][tx] + red[ty][3][tx];
}

// dweight / dbias = (or +=) the sum of the partials in the order of their rows
__global__ __launch_bounds__(256) void ln_bwd_join_kernel(const float* __restrict__ partial, int parts, int cols, float* __restrict__ dw,
                                                          float* __restrict__ db, int accumulate) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * (int64_t)cols) return;
    float* out = i < cols ? dw + i : db + (i - cols);
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += partial[(int64_t)p * 2 * cols + i];
    *out = accumulate ? *out + s : s;
}

int ln_parts(int64_t rows) { return (int)(rows < 64 ? 1 : rows < 64 * 128 ? rows / 64 : 128); }

}  // namespace

#define LN_CHECK(name)                                                                                                                   \
    VINCE_CHECK_ARG(dtype == VINCE_F32 || dtype == VINCE_BF16, VINCE_E_DTYPE, name ": dtype %d (VINCE_F32 or VINCE_BF16)", dtype);       \
    VINCE_CHECK_ARG(rows >= 0 && cols > 0, VINCE_E_SHAPE, name ": rows=%lld cols=%d", (long long)rows, cols)

extern "C" int vince_layer_norm_fwd(int dtype, const void* x, const float* weight, const float* bias, void* out, float* mean, float* rstd,
                                    int64_t rows, int32_t cols, float eps, int32_t relu, void* stream) {
    LN_CHECK("vince_layer_norm_fwd");
    VINCE_CHECK_ARG(eps >= 0.f, VINCE_E_ARG, "vince_layer_norm_fwd: eps=%g", (double)eps);
    if (rows == 0) return VINCE_OK;
    VINCE_CHECK_ARG(x && out && mean && rstd && (weight || !bias), VINCE_E_ARG, "vince_layer_norm_fwd: null pointer, or a bias without a weight");
    const dim3 grid((unsigned)((rows + 3) / 4 < 65536 ? (rows + 3) / 4 : 65536));
    if (dtype == VINCE_F32)
        hipLaunchKernelGGL(ln_fwd_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)x, weight, bias, (float*)out, mean, rstd,
                           rows, cols, eps, relu);
    else
        hipLaunchKernelGGL(ln_fwd_kernel<bf16_t>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16_t*)x, weight, bias, (bf16_t*)out, mean,
                           rstd, rows, cols, eps, relu);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" size_t vince_layer_norm_bwd_scratch_bytes(int dtype, int64_t rows, int32_t cols) {
    (void)dtype;
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)ln_parts(rows) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int vince_layer_norm_bwd(int dtype, const void* x, const float* weight, const float* mean, const float* rstd, const void* dout,
                                    const void* act, void* dx, float* dweight, float* dbias, int32_t accumulate, int64_t rows, int32_t cols,
                                    void* scratch, size_t scratch_bytes, void* stream) {
    LN_CHECK("vince_layer_norm_bwd");
    VINCE_CHECK_ARG((dweight == nullptr) == (dbias == nullptr), VINCE_E_ARG, "vince_layer_norm_bwd: dweight and dbias come together");
    hipStream_t st = (hipStream_t)stream;
    if (rows > 0) {
        VINCE_CHECK_ARG(x && mean && rstd && dout && dx, VINCE_E_ARG, "vince_layer_norm_bwd: null pointer");
        VINCE_CHECK_ARG(!dweight || (scratch && scratch_bytes >= vince_layer_norm_bwd_scratch_bytes(dtype, rows, cols)), VINCE_E_ARG,
                        "vince_layer_norm_bwd: scratch of %zu bytes", scratch_bytes);
        const dim3 grid((unsigned)((rows + 3) / 4 < 65536 ? (rows + 3) / 4 : 65536));
        const int parts = ln_parts(rows);
        const dim3 grid2((unsigned)((cols + 63) / 64), parts);
        const int64_t per = (rows + parts - 1) / parts;
        if (dtype == VINCE_F32) {
            hipLaunchKernelGGL(ln_bwd_dx_kernel<float>, grid, dim3(256), 0, st, (const float*)x, weight, mean, rstd, (const float*)dout,
                               (const float*)act, (float*)dx, rows, cols);
            if (dweight)
                hipLaunchKernelGGL(ln_bwd_dw_kernel<float>, grid2, dim3(256), 0, st, (const float*)x, mean, rstd, (const float*)dout,
                                   (const float*)act, (float*)scratch, rows, cols, per);
        } else {
            hipLaunchKernelGGL(ln_bwd_dx_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t*)x, weight, mean, rstd, (const bf16_t*)dout,
                               (const bf16_t*)act, (bf16_t*)dx, rows, cols);
            if (dweight)
                hipLaunchKernelGGL(ln_bwd_dw_kernel<bf16_t>, grid2, dim3(256), 0, st, (const bf16_t*)x, mean, rstd, (const bf16_t*)dout,
                                   (const bf16_t*)act, (float*)scratch, rows, cols, per);
        }
        VINCE_CHECK_LAUNCH();
    }
    if (dweight && (rows > 0 || !accumulate)) {
        hipLaunchKernelGGL(ln_bwd_join_kernel, dim3((unsigned)((2 * (int64_t)cols + 255) / 256)), dim3(256), 0, st, (const float*)scratch,
                           rows > 0 ? ln_parts(rows) : 0, cols, dweight, dbias, accumulate);
        VINCE_CHECK_LAUNCH();
    }
    return VINCE_OK;
}
