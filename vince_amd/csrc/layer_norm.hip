// Layer norm over the last axis of [rows][cols], forward and backward (include/vince_hip.h has the formulas).
//
// Bound by HBM: the forward reads and writes every element once, the backward reads two (three with a ReLU) and writes one.  So a row
// stays in registers from its one read to its write: TPR threads hold K 16-byte chunks each, the statistics are two-pass over the
// registers (fp32; the mean first, then the squares of the centred values), and the next row's loads are in flight meanwhile.  Rows of
// up to a wavefront's width take part of a wavefront, or one, with no barrier; longer ones a workgroup with one barrier a row.  Rows
// past what a workgroup's registers hold are read again for every pass (the *_long kernels).
#include "common.h"

namespace {

// ---- 16-byte chunks of a row at any element-aligned address ---------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_any_t;

template <typename T> __device__ __forceinline__ uint4 load16(const T* __restrict__ p) {
    const u32x4_any_t v = *(const u32x4_any_t*)p;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// The chunk at column `col` of a row, zeros behind the row's end.  One load whatever the chunk holds: a chunk that the row's end cuts
// is read as the row's last 16 bytes and shifted down (element by element it would be seven loads, or seven round trips).
template <typename T, bool FULL, typename I> __device__ __forceinline__ uint4 load_chunk(const T* __restrict__ row, I col, I cols) {
    constexpr int V = Elem<T>::CH, BITS = 8 * sizeof(T);
    if constexpr (FULL) return load16<T>(row + col);
    if (cols < V) {                                       // (a row of less than 16 bytes; uniform)
        uint32_t u[4] = {0u, 0u, 0u, 0u};
        if (col == 0)
#pragma unroll
            for (int e = 0; e < V - 1; ++e) {
                const T one = row[e < cols ? e : 0];
                uint32_t bits;
                if constexpr (sizeof(T) == 4) bits = __float_as_uint(one);
                else bits = one;
                if (e < cols) u[e * sizeof(T) / 4] |= bits << (e * BITS % 32);
            }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
    const I last = cols - V, from = col < last ? col : last;
    uint4 q = load16<T>(row + from);
    if (col > last) {
        const int shift = (int)(col - last < V ? col - last : V) * BITS;       // 128: nothing of the chunk is in the row
        unsigned __int128 v = ((unsigned __int128)(((uint64_t)q.w << 32) | q.z) << 64) | (((uint64_t)q.y << 32) | q.x);
        v = shift >= 128 ? 0 : v >> shift;
        q = make_uint4((uint32_t)v, (uint32_t)(v >> 32), (uint32_t)(v >> 64), (uint32_t)(v >> 96));
    }
    return q;
}
// n elements of a chunk to p: whole, or the 4 / 2 / 1 elements that n is made of
template <typename T> __device__ __forceinline__ void store_chunk(T* __restrict__ p, int n, const float* f) {
    typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t u32x2_any_t;
    typedef __attribute__((aligned(2))) uint32_t u32_any_t;
    constexpr int V = Elem<T>::CH;
    const uint4 q = Chunk<T>::pack(f);
    if (n >= V) {
        const u32x4_any_t v = {q.x, q.y, q.z, q.w};
        *(u32x4_any_t*)p = v;
        return;
    }
    uint32_t a = q.x, b = q.y, c = q.z;
    if (n & (V / 2)) {
        const u32x2_any_t v = {a, b};
        *(u32x2_any_t*)p = v;
        p += V / 2;
        a = c;
        b = q.w;
    }
    if constexpr (sizeof(T) == 2) {
        if (n & 2) {
            *(u32_any_t*)p = a;
            p += 2;
            a = b;
        }
    }
    if (n & 1) {
        if constexpr (sizeof(T) == 4) *p = __uint_as_float(a);
        else *p = (bf16_t)a;
    }
}
// the same columns of an fp32 vector (NULL: `none` everywhere)
template <int V, bool FULL, typename I> __device__ __forceinline__ void load_vector(const float* __restrict__ p, I col, I cols, float none, float* f) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = none;
        return;
    }
#pragma unroll
    for (int e = 0; e < V; e += 4) Chunk<float>::unpack(load_chunk<float, FULL>(p, (I)(col + e), cols), f + e);
}

// ---- sums over groups of lanes, every lane with the same bits ---------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int N> __device__ __forceinline__ float lanes_sum(float v) {   // N = 2 .. 64 neighbouring lanes
    if constexpr (N >= 2) v += dpp<0xB1>(v);       // quad_perm [1,0,3,2]
    if constexpr (N >= 4) v += dpp<0x4E>(v);       // quad_perm [2,3,0,1]
    if constexpr (N >= 8) v += dpp<0x141>(v);      // row_half_mirror
    if constexpr (N >= 16) v += dpp<0x140>(v);     // row_mirror
    if constexpr (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (N >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

constexpr int block_threads(int tpr) { return tpr > 256 ? tpr : 256; }
// Whether a thread keeps its columns' weight (and bias) in registers from row to row.  At 1024 threads, with 128 registers each, there is
// no room: they are read again for every row, from the caches.
constexpr bool holds_weights(int tpr) { return tpr < 1024; }

// Where this thread's K chunks of a row are.  FULL: cols == TPR * K * V, every chunk whole.  Else the first K / 2 are (ln_split takes K > 1
// for rows of more than TPR * K / 2 chunks), the others may be cut by the row's end or lie behind it.
template <typename T, int TPR, int K, bool FULL> struct Cols {
    static constexpr int V = Elem<T>::CH;
    int lane, cols;
    __device__ __forceinline__ Cols(int cols_) : lane((int)threadIdx.x % TPR), cols(cols_) {}
    __device__ __forceinline__ int col(int k) const { return (k * TPR + lane) * V; }
    static constexpr bool whole(int k) { return FULL || k < K / 2; }
    __device__ __forceinline__ int valid(int k) const {   // elements of chunk k that are in the row
        if (whole(k)) return V;
        const int n = cols - col(k);
        return n < 0 ? 0 : n > V ? V : n;
    }
    __device__ __forceinline__ void load(const T* __restrict__ row, uint4 (&q)[K]) const {
#pragma unroll
        for (int k = 0; k < K; ++k) q[k] = whole(k) ? load_chunk<T, true>(row, col(k), cols) : load_chunk<T, false>(row, col(k), cols);
    }
    __device__ __forceinline__ void load(const float* __restrict__ p, float none, int k, float (&f)[V]) const {   // of a vector of the row's length
        if (whole(k)) load_vector<V, true>(p, col(k), cols, none, f);
        else load_vector<V, false>(p, col(k), cols, none, f);
    }
};

template <typename T, int TPR, int K, bool FULL>
__global__ __launch_bounds__(block_threads(TPR)) void ln_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                    const float* __restrict__ b, T* __restrict__ out, float* __restrict__ mean,
                                                                    float* __restrict__ rstd, int64_t rows, int cols, float eps, int relu) {
    constexpr int V = Elem<T>::CH, R = block_threads(TPR) / TPR, WAVES = TPR / 64;
    const Cols<T, TPR, K, FULL> at(cols);
    const float inv = 1.f / (float)cols;
    __shared__ float2 part[2][WAVES > 1 ? WAVES : 1];    // mean and squares of each wavefront's columns, two rows' worth
    float count = 0.f;                                    // elements of a row that this wavefront's (or group's) lanes hold
#pragma unroll
    for (int k = 0; k < K; ++k) count += (float)at.valid(k);
    count = lanes_sum<(TPR < 64 ? TPR : 64)>(count);
    if (FULL) count = (float)((TPR < 64 ? TPR : 64) * K * V);
    __shared__ float counts[WAVES > 1 ? WAVES : 1];
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = count;
        __syncthreads();
    }
    constexpr bool HOLD = holds_weights(TPR);
    float wf[HOLD ? K : 1][V], bf[HOLD ? K : 1][V];
    if constexpr (HOLD) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at.load(w, 1.f, k, wf[k]);
            at.load(b, 0.f, k, bf[k]);
        }
    }
    const int64_t stride = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / TPR;
    uint4 q[K];
    if (row < rows) at.load(x + row * cols, q);
    for (int turn = 0; row < rows; row += stride, turn ^= 1) {      // (a workgroup of one row leaves the loop as one: R == 1 with barriers)
        int64_t again = 0;
        if constexpr (!HOLD) asm volatile("" : "+s"(again));      // (an offset it cannot see through: else the compiler reads w, b once, and spills them)
        float f[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) Chunk<T>::unpack(q[k], f[k]);
        if (row + stride < rows) at.load(x + (row + stride) * cols, q);
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[k][e];
        // means by division, not by a rounded reciprocal: a row of one value has exactly that mean, and its output is the bias
        float m = lanes_sum<(TPR < 64 ? TPR : 64)>(s) / fmaxf(count, 1.f);
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = at.whole(k) || e < at.valid(k) ? f[k][e] - m : 0.f;
                ss = fmaf(d, d, ss);
            }
        ss = lanes_sum<(TPR < 64 ? TPR : 64)>(ss);
        if constexpr (WAVES > 1) {       // the row's from the wavefronts': their squares about their own means, moved to the common one
            if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = make_float2(m, ss);
            __syncthreads();             // (the other turn's slot is written only behind the next row's barrier: one barrier a row)
            float2 p[WAVES];
            m = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                p[i] = part[turn][i];
                m = fmaf(p[i].x, FULL ? (float)(64 * K * V) : counts[i], m);
            }
            m /= (float)cols;
            ss = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) {
                const float d = p[i].x - m;
                ss += fmaf(d * d, FULL ? (float)(64 * K * V) : counts[i], p[i].y);
            }
        }
        const float r = 1.f / sqrtf(fmaf(ss, inv, eps));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int kw = HOLD ? k : 0;
            if constexpr (!HOLD) {
                at.load(w ? w + again : w, 1.f, k, wf[0]);
                at.load(b ? b + again : b, 0.f, k, bf[0]);
            }
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                y[e] = fmaf((f[k][e] - m) * r, wf[kw][e], bf[kw][e]);
                if (relu && y[e] < 0.f) y[e] = 0.f;          // (a NaN stays)
            }
            const int n = at.valid(k);
            if (at.whole(k) || n > 0) store_chunk<T>(out + row * cols + at.col(k), n, y);
        }
        if (at.lane == 0) { mean[row] = m; rstd[row] = r; }
    }
}

// ---- backward: dx, and this workgroup's sums for dweight and dbias ------------------------------------------------------------------
// A thread has the same columns in every row it works on: its parts of dweight and dbias stay in registers until the last row.  Then the
// R row groups of a workgroup are added up in LDS and one partial row [2][cols] a workgroup goes to scratch (or, with DIRECT, the only
// workgroup writes the result).
template <typename T, int TPR, int K, bool FULL, bool ACT>
__global__ __launch_bounds__(block_threads(TPR)) void ln_bwd_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    const T* __restrict__ dout, const T* __restrict__ act, T* __restrict__ dx,
                                                                    float* __restrict__ dw_out, float* __restrict__ db_out, int accumulate,
                                                                    float* __restrict__ partial, int64_t rows, int cols) {
    constexpr int V = Elem<T>::CH, THREADS = block_threads(TPR), R = THREADS / TPR, WAVES = TPR / 64;
    const Cols<T, TPR, K, FULL> at(cols);
    const float inv = 1.f / (float)cols;
    __shared__ float2 part[2][WAVES > 1 ? WAVES : 1];
    constexpr bool HOLD = holds_weights(TPR);
    float wf[HOLD ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (HOLD) at.load(w, 1.f, k, wf[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.f;
    }
    const int64_t stride = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / TPR;
    uint4 qx[K], qd[K], qa[ACT ? K : 1];
    float m_next = 0.f, r_next = 0.f;
    auto fetch = [&](int64_t i) {
        at.load(x + i * cols, qx);
        at.load(dout + i * cols, qd);
        if constexpr (ACT) at.load(act + i * cols, qa);
        m_next = mean[i];
        r_next = rstd[i];
    };
    if (row < rows) fetch(row);
    for (int turn = 0; row < rows; row += stride, turn ^= 1) {
        int64_t again = 0;
        if constexpr (!HOLD) asm volatile("" : "+s"(again));      // (see ln_fwd_kernel)
        float xh[K][V], g[K][V];
        const float m = m_next, r = r_next;
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Chunk<T>::unpack(qx[k], xh[k]);
            Chunk<T>::unpack(qd[k], g[k]);
            if constexpr (ACT) {
                float a[V];
                Chunk<T>::unpack(qa[k], a);
#pragma unroll
                for (int e = 0; e < V; ++e) g[k][e] = a[e] > 0.f ? g[k][e] : 0.f;
            }
        }
        if (row + stride < rows) fetch(row + stride);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int kw = HOLD ? k : 0;
            if constexpr (!HOLD) at.load(w ? w + again : w, 1.f, k, wf[0]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[k][e] = at.whole(k) || e < at.valid(k) ? (xh[k][e] - m) * r : 0.f;
                db[k][e] += g[k][e];
                dw[k][e] = fmaf(g[k][e], xh[k][e], dw[k][e]);
                g[k][e] *= wf[kw][e];
                c1 += g[k][e];
                c2 = fmaf(g[k][e], xh[k][e], c2);
            }
        }
        c1 = lanes_sum<(TPR < 64 ? TPR : 64)>(c1);
        c2 = lanes_sum<(TPR < 64 ? TPR : 64)>(c2);
        if constexpr (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = make_float2(c1, c2);
            __syncthreads();
            c1 = c2 = 0.f;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) { c1 += part[turn][i].x; c2 += part[turn][i].y; }
        }
        c1 *= inv;
        c2 *= inv;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = r * (g[k][e] - c1 - xh[k][e] * c2);
            const int n = at.valid(k);
            if (at.whole(k) || n > 0) store_chunk<T>(dx + row * cols + at.col(k), n, y);
        }
    }
    if (!dw_out) return;
    // one row group a workgroup: the registers are the workgroup's sums; several: added up in LDS in the order of the groups
    __shared__ float red[R > 1 ? THREADS * K * V : 1];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float(&v)[K][V] = half == 0 ? dw : db;
        if constexpr (R > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) red[(threadIdx.x / TPR * K + k) * (TPR * V) + at.lane * V + e] = v[k][e];
            __syncthreads();
        }
        float* final_out = half == 0 ? dw_out : db_out;
        float* to = partial ? partial + ((int64_t)blockIdx.x * 2 + half) * cols : final_out;
        const bool add = !partial && accumulate;
        if constexpr (R > 1) {
            for (int c = threadIdx.x; c < cols; c += THREADS) {       // (cols <= TPR * K * V)
                float s = 0.f;
#pragma unroll 8
                for (int i = 0; i < R; ++i) s += red[i * (K * TPR * V) + c];
                to[c] = add ? to[c] + s : s;
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at.whole(k) || e < at.valid(k)) {
                        const int c = at.col(k) + e;
                        to[c] = add ? to[c] + v[k][e] : v[k][e];
                    }
        }
    }
}

// dweight / dbias = (or +=) the sum of `parts` partial rows [2][cols]: 32 columns x 32 rows at a time, the rows' sums in a fixed order
__global__ __launch_bounds__(1024) void ln_bwd_join_kernel(const float* __restrict__ partial, int parts, int64_t cols2, int cols,
                                                           float* __restrict__ dw, float* __restrict__ db, int accumulate) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (c < cols2) {
        const float* p = partial + c;
        int i = ty;
        for (; i + 96 < parts; i += 128) {
            const float a0 = p[(int64_t)i * cols2], a1 = p[(int64_t)(i + 32) * cols2], a2 = p[(int64_t)(i + 64) * cols2],
                        a3 = p[(int64_t)(i + 96) * cols2];
            s0 += a0; s1 += a1; s2 += a2; s3 += a3;
        }
        for (; i < parts; i += 32) s0 += p[(int64_t)i * cols2];
    }
    red[ty][tx] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (ty == 0 && c < cols2) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][tx];
        float* out = c < cols ? dw + c : db + (c - cols);
        *out = accumulate ? *out + s : s;
    }
}

// ---- rows longer than a workgroup's registers -----------------------------------------------------------------------------------------
template <int WAVES> __device__ __forceinline__ float block_sum(float v, float* red) {
    v = lanes_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) s += red[i];
    return s;
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                           T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                           int cols, float eps, int relu) {
    constexpr int V = Elem<T>::CH;
    __shared__ float red[16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * cols;
        float s = 0.f, f[V];
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            Chunk<T>::unpack(load_chunk<T, false>(xr, c, (int64_t)cols), f);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[e];
        }
        const float m = block_sum<16>(s, red) / (float)cols;
        s = 0.f;
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const int n = cols - c < V ? (int)(cols - c) : V;
            Chunk<T>::unpack(load_chunk<T, false>(xr, c, (int64_t)cols), f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = e < n ? f[e] - m : 0.f;
                s = fmaf(d, d, s);
            }
        }
        const float r = 1.f / sqrtf(block_sum<16>(s, red) / (float)cols + eps);
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const int n = cols - c < V ? (int)(cols - c) : V;
            float wf[V], bf[V];
            Chunk<T>::unpack(load_chunk<T, false>(xr, c, (int64_t)cols), f);
            load_vector<V, false>(w, c, (int64_t)cols, 1.f, wf);
            load_vector<V, false>(b, c, (int64_t)cols, 0.f, bf);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[e] = fmaf((f[e] - m) * r, wf[e], bf[e]);
                if (relu && f[e] < 0.f) f[e] = 0.f;
            }
            store_chunk<T>(out + row * cols + c, n, f);
        }
        if (threadIdx.x == 0) { mean[row] = m; rstd[row] = r; }
    }
}

// d (masked) and xhat of one chunk
template <typename T>
__device__ __forceinline__ void grad_chunk(const T* __restrict__ x, const T* __restrict__ dout, const T* __restrict__ act, int64_t row, int64_t c,
                                           int cols, float m, float r, float* d, float* xh) {
    constexpr int V = Elem<T>::CH;
    Chunk<T>::unpack(load_chunk<T, false>(x + row * cols, c, (int64_t)cols), xh);
    Chunk<T>::unpack(load_chunk<T, false>(dout + row * cols, c, (int64_t)cols), d);
    if (act) {
        float a[V];
        Chunk<T>::unpack(load_chunk<T, false>(act + row * cols, c, (int64_t)cols), a);
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = a[e] > 0.f ? d[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) xh[e] = c + e < cols ? (xh[e] - m) * r : 0.f;
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_dx_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, const T* __restrict__ dout,
                                                              const T* __restrict__ act, T* __restrict__ dx, int64_t rows, int cols) {
    constexpr int V = Elem<T>::CH;
    __shared__ float red[16];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float m = mean[row], r = rstd[row];
        float c1 = 0.f, c2 = 0.f, d[V], xh[V], wf[V];
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const int n = cols - c < V ? (int)(cols - c) : V;
            grad_chunk<T>(x, dout, act, row, c, cols, m, r, d, xh);
            load_vector<V, false>(w, c, (int64_t)cols, 1.f, wf);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float g = d[e] * wf[e];
                c1 += g;
                c2 = fmaf(g, xh[e], c2);
            }
        }
        c1 = block_sum<16>(c1, red) / (float)cols;
        c2 = block_sum<16>(c2, red) / (float)cols;
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const int n = cols - c < V ? (int)(cols - c) : V;
            grad_chunk<T>(x, dout, act, row, c, cols, m, r, d, xh);
            load_vector<V, false>(w, c, (int64_t)cols, 1.f, wf);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = r * (d[e] * wf[e] - c1 - xh[e] * c2);
            store_chunk<T>(dx + row * cols + c, n, d);
        }
    }
}

// partial sums over the rows blockIdx.y, blockIdx.y + gridDim.y, ... of one chunk of columns a thread
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_long_dw_kernel(const T* __restrict__ x, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             const T* __restrict__ dout, const T* __restrict__ act, float* __restrict__ partial,
                                                             int64_t rows, int cols) {
    constexpr int V = Elem<T>::CH;
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= cols) return;
    const int n = cols - c < V ? (int)(cols - c) : V;
    float dw[V], db[V], d[V], xh[V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        grad_chunk<T>(x, dout, act, row, c, cols, mean[row], rstd[row], d, xh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            db[e] += d[e];
            dw[e] = fmaf(d[e], xh[e], dw[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < n) {
            partial[((int64_t)blockIdx.y * 2) * cols + c + e] = dw[e];
            partial[((int64_t)blockIdx.y * 2 + 1) * cols + c + e] = db[e];
        }
}

// ---- which split -----------------------------------------------------------------------------------------------------------------------
// Threads a row and chunks a thread, from the row's number of 16-byte chunks.  Up to 64 chunks: one a lane, the smallest power of two of
// lanes (several rows share a wavefront).  Then a wavefront with up to KMAX a lane, then a workgroup of 256 .. 1024.  KMAX: what the
// registers hold with four wavefronts a SIMD -- 4 forward; backward, which keeps a weight and two sums a column, 16 values (4 fp32
// chunks, 2 bf16).
struct Split { int tpr, k; };
Split ln_split(int64_t chunks, int kmax) {
    if (chunks <= 64) {
        int tpr = 2;
        while (tpr < chunks) tpr *= 2;
        return {tpr, 1};
    }
    for (int tpr = 64; tpr <= 1024; tpr = tpr == 64 ? 256 : tpr * 2)
        for (int k = 1; k <= kmax; k *= 2)
            if ((int64_t)tpr * k >= chunks) return {tpr, k};
    return {0, 0};
}
int ln_chunks(int dtype, int cols) { const int v = dtype == VINCE_F32 ? 4 : 8; return (cols + v - 1) / v; }
constexpr int LN_FWD_K = 4;
constexpr int ln_bwd_k(int dtype) { return dtype == VINCE_F32 ? 4 : 2; }

// Workgroups of the backward: at most two a CU -- each writes a partial row of 8 bytes a column that is read again -- and at least four
// rows for each row group, so that the partial rows stay a small part of what is read anyway.
int ln_bwd_blocks(int64_t rows, const Split& s) {
    const int64_t per = s.tpr == 0 ? 4 : 4 * (block_threads(s.tpr) / s.tpr);
    const int64_t n = (rows + per - 1) / per;
    return (int)(n < 1 ? 1 : n > 512 ? 512 : n);
}

template <typename T, int TPR, int K>
void launch_fwd(const void* x, const float* w, const float* b, void* out, float* mean, float* rstd, int64_t rows, int cols, float eps, int relu,
                hipStream_t st) {
    constexpr int THREADS = block_threads(TPR), R = THREADS / TPR;
    const int64_t want = (rows + R - 1) / R, most = 256 * 2048 / THREADS;
    const dim3 grid((unsigned)(want < most ? want : most));
    if (cols == TPR * K * Elem<T>::CH)
        hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, K, true>), grid, dim3(THREADS), 0, st, (const T*)x, w, b, (T*)out, mean, rstd, rows, cols, eps, relu);
    else
        hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, K, false>), grid, dim3(THREADS), 0, st, (const T*)x, w, b, (T*)out, mean, rstd, rows, cols, eps, relu);
}

template <typename T>
void run_fwd(int dtype, const void* x, const float* w, const float* b, void* out, float* mean, float* rstd, int64_t rows, int cols, float eps,
             int relu, hipStream_t st) {
    const Split s = ln_split(ln_chunks(dtype, cols), LN_FWD_K);
#define LN_CASE(TPR, K) \
    if (s.tpr == TPR && s.k == K) return launch_fwd<T, TPR, K>(x, w, b, out, mean, rstd, rows, cols, eps, relu, st)
    LN_CASE(2, 1); LN_CASE(4, 1); LN_CASE(8, 1); LN_CASE(16, 1); LN_CASE(32, 1); LN_CASE(64, 1); LN_CASE(64, 2); LN_CASE(64, 4);
    LN_CASE(256, 2); LN_CASE(256, 4); LN_CASE(512, 4); LN_CASE(1024, 4);
#undef LN_CASE
    hipLaunchKernelGGL(ln_fwd_long_kernel<T>, dim3((unsigned)(rows < 1024 ? rows : 1024)), dim3(1024), 0, st, (const T*)x, w, b, (T*)out, mean, rstd,
                       rows, cols, eps, relu);
}

struct BwdArgs {
    const void *x, *dout, *act;
    const float *w, *mean, *rstd;
    void* dx;
    float *dw, *db, *partial;
    int accumulate;
    int64_t rows;
    int cols, blocks;
};

template <typename T, int TPR, int K> void launch_bwd(const BwdArgs& a, hipStream_t st) {
    const bool full = a.cols == TPR * K * Elem<T>::CH;
#define LN_LAUNCH(FULL, ACT)                                                                                                              \
    if (full == FULL && (a.act != nullptr) == ACT)                                                                                        \
        hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, K, FULL, ACT>), dim3(a.blocks), dim3(block_threads(TPR)), 0, st, (const T*)a.x, a.w, a.mean, \
                           a.rstd, (const T*)a.dout, (const T*)a.act, (T*)a.dx, a.dw, a.db, a.accumulate, a.partial, a.rows, a.cols)
    LN_LAUNCH(true, false);
    LN_LAUNCH(true, true);
    LN_LAUNCH(false, false);
    LN_LAUNCH(false, true);
#undef LN_LAUNCH
}

template <typename T> void run_bwd(const Split& s, const BwdArgs& a, hipStream_t st) {
#define LN_CASE(TPR, K) \
    if (s.tpr == TPR && s.k == K) return launch_bwd<T, TPR, K>(a, st)
    LN_CASE(2, 1); LN_CASE(4, 1); LN_CASE(8, 1); LN_CASE(16, 1); LN_CASE(32, 1); LN_CASE(64, 1); LN_CASE(64, 2); LN_CASE(256, 2);
    if constexpr (sizeof(T) == 4) {
        LN_CASE(64, 4); LN_CASE(256, 4); LN_CASE(512, 4); LN_CASE(1024, 4);
    } else {
        LN_CASE(256, 1); LN_CASE(512, 2); LN_CASE(1024, 2);
    }
#undef LN_CASE
    hipLaunchKernelGGL(ln_bwd_long_dx_kernel<T>, dim3((unsigned)(a.rows < 1024 ? a.rows : 1024)), dim3(1024), 0, st, (const T*)a.x, a.w, a.mean,
                       a.rstd, (const T*)a.dout, (const T*)a.act, (T*)a.dx, a.rows, a.cols);
    if (a.dw)
        hipLaunchKernelGGL(ln_bwd_long_dw_kernel<T>, dim3((unsigned)((a.cols + 256 * Elem<T>::CH - 1) / (256 * Elem<T>::CH)), (unsigned)a.blocks),
                           dim3(256), 0, st, (const T*)a.x, a.mean, a.rstd, (const T*)a.dout, (const T*)a.act, a.partial, a.rows, a.cols);
}

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
    if (dtype == VINCE_F32) run_fwd<float>(dtype, x, weight, bias, out, mean, rstd, rows, cols, eps, relu, (hipStream_t)stream);
    else run_fwd<bf16_t>(dtype, x, weight, bias, out, mean, rstd, rows, cols, eps, relu, (hipStream_t)stream);
    VINCE_CHECK_LAUNCH();
    return VINCE_OK;
}

extern "C" size_t vince_layer_norm_bwd_scratch_bytes(int dtype, int64_t rows, int32_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    const Split s = ln_split(ln_chunks(dtype, cols), ln_bwd_k(dtype));
    const int blocks = ln_bwd_blocks(rows, s);
    return blocks == 1 && s.tpr ? 0 : (size_t)blocks * 2 * (size_t)cols * sizeof(float);
}

extern "C" int vince_layer_norm_bwd(int dtype, const void* x, const float* weight, const float* mean, const float* rstd, const void* dout,
                                    const void* act, void* dx, float* dweight, float* dbias, int32_t accumulate, int64_t rows, int32_t cols,
                                    void* scratch, size_t scratch_bytes, void* stream) {
    LN_CHECK("vince_layer_norm_bwd");
    VINCE_CHECK_ARG((dweight == nullptr) == (dbias == nullptr), VINCE_E_ARG, "vince_layer_norm_bwd: dweight and dbias come together");
    hipStream_t st = (hipStream_t)stream;
    const Split s = ln_split(ln_chunks(dtype, cols), ln_bwd_k(dtype));
    const int blocks = ln_bwd_blocks(rows, s);
    const bool direct = rows > 0 && blocks == 1 && s.tpr;       // one workgroup: it writes dweight and dbias itself
    if (rows > 0) {
        VINCE_CHECK_ARG(x && mean && rstd && dout && dx, VINCE_E_ARG, "vince_layer_norm_bwd: null pointer");
        const size_t need = dweight ? vince_layer_norm_bwd_scratch_bytes(dtype, rows, cols) : 0;
        VINCE_CHECK_ARG(need == 0 || (scratch && scratch_bytes >= need), VINCE_E_ARG, "vince_layer_norm_bwd: scratch of %zu bytes", scratch_bytes);
        const BwdArgs a = {x, dout, act, weight, mean, rstd, dx, dweight, dbias, direct ? nullptr : (float*)scratch, accumulate, rows, cols, blocks};
        if (dtype == VINCE_F32) run_bwd<float>(s, a, st);
        else run_bwd<bf16_t>(s, a, st);
        VINCE_CHECK_LAUNCH();
    }
    if (dweight && !direct && (rows > 0 || !accumulate)) {
        hipLaunchKernelGGL(ln_bwd_join_kernel, dim3((unsigned)((2 * (int64_t)cols + 31) / 32)), dim3(1024), 0, st, (const float*)scratch,
                           rows > 0 ? blocks : 0, 2 * (int64_t)cols, cols, dweight, dbias, accumulate);
        VINCE_CHECK_LAUNCH();
    }
    return VINCE_OK;
}
