// Layer norm over the last axis of [rows][cols], forward and backward (include/vince_hip.h has the formulas).
//
// Bound by HBM: the forward reads and writes every element once, the backward reads two (three with a ReLU) and writes one.  So a row
// stays in registers from its one read to its write: TPR threads hold K 16-byte chunks each, the statistics are two-pass over the
// registers (fp32; the mean first, then the squares of the centred values), and the next row's loads are in flight meanwhile.  Rows of
// up to a wavefront's width take part of a wavefront, or one, with no barrier; longer ones a workgroup with one barrier a row.  Rows
// past what a workgroup's registers hold are read again for every pass (the *_long kernels).
#include "common.h"

// Where a row's end cuts a 16-byte chunk, two threads compute the columns that its chunk shares with the one before it, and both write
// them: the same bits, so every multiply-add is written out (fmaf) and the compiler makes none by itself.
#pragma clang fp contract(off)

namespace {

// ---- 16-byte chunks at any element-aligned address (the hardware takes any; the type tells the compiler so) --------------------------
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t u32x4_any_t;
template <typename T> __device__ __forceinline__ uint4 load16(const T* __restrict__ p) {
    const u32x4_any_t v = *(const u32x4_any_t*)p;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
template <typename T> __device__ __forceinline__ void store16(T* __restrict__ p, const float* f) {
    const uint4 q = Chunk<T>::pack(f);
    const u32x4_any_t v = {q.x, q.y, q.z, q.w};
    *(u32x4_any_t*)p = v;
}
// the first n elements of a chunk, one by one (rows of less than 16 bytes)
template <typename T> __device__ __forceinline__ uint4 load_few(const T* __restrict__ p, int n) {
    uint32_t u[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < Elem<T>::CH - 1; ++e) {
        const T one = p[e < n ? e : 0];
        uint32_t bits;
        if constexpr (sizeof(T) == 4) bits = __float_as_uint(one);
        else bits = one;
        if (e < n) u[e * sizeof(T) / 4] |= bits << (8 * sizeof(T) * e % 32);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}
template <typename T> __device__ __forceinline__ void store_few(T* __restrict__ p, int n, const float* f) {
#pragma unroll
    for (int e = 0; e < Elem<T>::CH - 1; ++e)
        if (e < n) {
            if constexpr (sizeof(T) == 4) p[e] = f[e];
            else p[e] = f32_to_bf16(f[e]);
        }
}

// The chunk of columns col .. col + V - 1 of a row of `cols`; col may be below 0, the chunk may reach past the row's end or lie outside.
// One that the row does not fill is taken as the 16 bytes of the row that are nearest: one load and one store whatever it holds, nothing
// to shift; the elements outside its own columns are its neighbour's, and stay out of the sums (own()).  SHORT: the row may have less than
// 16 bytes (then col >= 0).
template <typename T, typename I, bool SHORT> struct Piece {
    static constexpr int V = Elem<T>::CH;
    I from;
    int first, n, cols;          // its own elements are first .. first + n - 1
    __device__ __forceinline__ Piece(I col, I cols_) {
        const bool small = SHORT && cols_ < V;
        cols = small ? (int)cols_ : V;
        const I last = small ? 0 : cols_ - V;
        from = col < 0 ? 0 : col < last ? col : last;
        first = (int)(col < from ? 0 : col - from < V ? col - from : V);
        n = small ? (col == 0 ? (int)cols_ : 0) : col < 0 ? (int)(col + V) : V - first;
    }
    __device__ __forceinline__ bool own(int e) const { return (unsigned)(e - first) < (unsigned)n; }
    __device__ __forceinline__ uint4 load(const T* __restrict__ row) const {
        if (SHORT && cols < V) return load_few<T>(row, cols);
        return load16<T>(row + from);
    }
    __device__ __forceinline__ void load_vector(const float* __restrict__ p, float none, float* f) const {
        if (!p || (SHORT && cols < V)) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = SHORT && p && e < cols ? p[e] : none;
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 4) Chunk<float>::unpack(load16<float>(p + from + e), f + e);
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ row, const float* f) const {
        if (n == 0) return;
        if (SHORT && cols < V) store_few<T>(row, cols, f);
        else store16<T>(row + from, f);
    }
};

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

// the sum over the wavefront's lanes l, l + 8, l + 16, ... in each of them
template <int N> __device__ __forceinline__ float strided_sum(float v) {
    static_assert(N == 8, "lanes 8 apart");
    v += dpp<0x128>(v);                            // row_ror:8
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// TPR, threads a row: up to 64 exactly, in workgroups of 256; more than 64, the most of a row's own workgroup, which has as many
// wavefronts (blockDim.x / 64, 16 at most) as the row needs.
constexpr int block_threads(int tpr) { return tpr > 64 ? tpr : 256; }
constexpr int wave_lanes(int tpr) { return tpr < 64 ? tpr : 64; }
// the sum of a workgroup's per-wavefront values, one in each of 16 neighbouring lanes (0 behind the last wavefront)
__device__ __forceinline__ float waves_sum(float v) { return lanes_sum<16>(v); }
// Whether a thread keeps its columns' weight (and bias) in registers from row to row.  Up to 1024 threads, with 128 registers each, there
// is no room: they are read again for every row, from the caches (held, 16384 x 8192 fp32 takes 205 / 313 us forward / backward instead of
// 200 / 292, 16384 x 16384 392 / 676 instead of 400 / 586).
constexpr bool holds_weights(int tpr) { return tpr < 1024; }

// s / n from inv = 1 / n, with one step of correction: exact where the quotient is a float, so that a row of one value has that mean and
// the bias as its output; a third of the instructions of a division, which every wavefront would make for every row
__device__ __forceinline__ float divide(float s, float n, float inv) {
    const float q = s * inv, better = fmaf(fmaf(-q, n, s), inv, q);
    return better == better ? better : q;          // (an infinite sum: the correction is NaN)
}

// How the rows lie.  FULL: cols == TPR * K * V, every chunk whole.  PLAIN: the chunks start with the row, the first K / 2 are whole
// (ln_split takes K > 1 for rows of more than TPR * K / 2 chunks).  SHIFTED: bfloat16 rows of an odd length start at every other address;
// a 16-byte access that is not even aligned to 4 bytes occupies the vector cache three times as long (PMC: 47 M accesses for 13 M in the
// backward of 65536 x 2047 against 2048; 31 M shifted), so the chunks start at the 16-byte boundaries of memory, the first before the row.
// A thread's rows are a multiple of 8 apart (the grid's size is, where it has more than one): the boundaries are the same in each.  us
// PLAIN / SHIFTED: 65536 x 2049 forward 129 / 116, backward 219 / 191; 32768 x 4095 127 / 120 and 212 / 168; 65536 x 2047 98 / 118 and 210 /
// 192, 16384 x 8191 136 / 104 and 192 / 203 -- below a power of two the row has a chunk more than one wavefront (2047 forward) or the
// workgroups with room for their weights (8191 backward) hold.
enum Mode { FULL, PLAIN, SHIFTED };

// This thread's K chunks of a row.
template <typename T, int TPR, int K, Mode MODE> struct Cols {
    static constexpr int V = Elem<T>::CH;
    int start, cols;             // start: the first chunk's column
    __device__ __forceinline__ static int threads() { return TPR > 64 ? (int)blockDim.x : TPR; }
    __device__ __forceinline__ Cols(int cols_, const T* first_row) : start((TPR > 64 ? (int)threadIdx.x : (int)threadIdx.x % TPR) * V), cols(cols_) {
        if constexpr (MODE == SHIFTED) start -= (int)((uintptr_t)first_row / sizeof(T) % V);
    }
    static constexpr bool whole(int k) { return MODE == FULL || (MODE == PLAIN && k < K / 2); }
    __device__ __forceinline__ static bool leads() { return TPR > 64 ? threadIdx.x == 0 : threadIdx.x % TPR == 0; }
    __device__ __forceinline__ int col(int k) const { return k * threads() * V + start; }
    typedef Piece<T, int, TPR == 2> piece_t;             // (only rows of one or two chunks can have less than 16 bytes)
    __device__ __forceinline__ piece_t piece(int k) const { return piece_t(col(k), cols); }
    __device__ __forceinline__ bool own(int k, int e) const { return whole(k) || piece(k).own(e); }
    __device__ __forceinline__ int own(int k) const { return whole(k) ? V : piece(k).n; }
    __device__ __forceinline__ int first_col(int k) const { return whole(k) ? col(k) : piece(k).from; }
    __device__ __forceinline__ void load(const T* __restrict__ row, uint4 (&q)[K]) const {
#pragma unroll
        for (int k = 0; k < K; ++k) q[k] = whole(k) ? load16<T>(row + col(k)) : piece(k).load(row);
    }
    __device__ __forceinline__ void load(const float* __restrict__ p, float none, int k, float (&f)[V]) const {   // of a vector of the row's length
        if (whole(k) && p) {
#pragma unroll
            for (int e = 0; e < V; e += 4) Chunk<float>::unpack(load16<float>(p + col(k) + e), f + e);
        } else if (whole(k)) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = none;
        } else {
            piece(k).load_vector(p, none, f);
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ row, int k, const float (&f)[V]) const {
        if (whole(k)) store16<T>(row + col(k), f);
        else piece(k).store(row, f);
    }
};

template <typename T, int TPR, int K, Mode MODE>
__global__ __launch_bounds__(block_threads(TPR)) void ln_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                    const float* __restrict__ b, T* __restrict__ out, float* __restrict__ mean,
                                                                    float* __restrict__ rstd, int64_t rows, int cols, float eps, int relu) {
    constexpr int V = Elem<T>::CH, R = TPR > 64 ? 1 : 256 / TPR, LANES = wave_lanes(TPR);
    constexpr bool WAVES = TPR > 64;                     // a row is several wavefronts'
    constexpr bool HOLD = holds_weights(TPR);
    const int64_t stride = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + (WAVES ? 0 : threadIdx.x / TPR);
    const Cols<T, TPR, K, MODE> at(cols, x + row * cols);
    const float inv = 1.f / (float)cols;
    __shared__ float2 part[2][WAVES ? 16 : 1];           // mean and squares of each wavefront's columns, two rows' worth
    __shared__ float counts[WAVES ? 16 : 1];
    if constexpr (WAVES) {
        if (threadIdx.x < 16) {
            part[0][threadIdx.x] = part[1][threadIdx.x] = make_float2(0.f, 0.f);
            counts[threadIdx.x] = 0.f;
        }
        __syncthreads();
    }
    float count = (float)(LANES * K * V);                 // elements of a row that this wavefront's (or group's) lanes own
    if constexpr (MODE != FULL) {
        count = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) count += (float)at.own(k);
        count = lanes_sum<LANES>(count);
    }
    float wave_count = 0.f;                               // lane i of 16: wavefront i's
    if constexpr (WAVES) {
        if ((threadIdx.x & 63) == 0) counts[threadIdx.x >> 6] = count;
        __syncthreads();
        wave_count = counts[threadIdx.x & 15];
    }
    const float inv_count = count > 0.f ? 1.f / count : 0.f;
    float wf[HOLD ? K : 1][V], bf[HOLD ? K : 1][V];
    if constexpr (HOLD) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            at.load(w, 1.f, k, wf[k]);
            at.load(b, 0.f, k, bf[k]);
        }
    }
    uint4 q[K];
    if (row < rows) at.load(x + row * cols, q);
    for (int turn = 0; row < rows; row += stride, turn ^= 1) {      // (a workgroup with barriers has one row at a time: it leaves as one)
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
            for (int e = 0; e < V; ++e) s += at.own(k, e) ? f[k][e] : 0.f;
        float m = divide(lanes_sum<LANES>(s), count, inv_count);
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = at.own(k, e) ? f[k][e] - m : 0.f;
                ss = fmaf(d, d, ss);
            }
        ss = lanes_sum<LANES>(ss);
        if constexpr (WAVES) {           // the row's from the wavefronts': their squares about their own means, moved to the common one
            if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = make_float2(m, ss);
            __syncthreads();             // (the other turn's slot is written only behind the next row's barrier: one barrier a row)
            const float2 p = part[turn][threadIdx.x & 15];
            m = divide(waves_sum(p.x * wave_count), (float)cols, inv);
            const float d = p.x - m;
            ss = waves_sum(wave_count > 0.f ? fmaf(d * d, wave_count, p.y) : 0.f);
        }
        const float r = rsqrtf(fmaf(ss, inv, eps));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int kw = HOLD ? k : 0;
            if constexpr (!HOLD) {
                at.load(w ? w + again : w, 1.f, k, wf[0]);
                at.load(b ? b + again : b, 0.f, k, bf[0]);
            }
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = fmaf((f[k][e] - m) * r, wf[kw][e], bf[kw][e]);
            if (relu) {
                asm volatile("");                            // (a branch: two instructions an element for those who want none)
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = y[e] < 0.f ? 0.f : y[e];          // (a NaN stays)
            }
            at.store(out + row * cols, k, y);
        }
        if (at.leads()) { mean[row] = m; rstd[row] = r; }
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------------
// A row's chunks of x, dout and act in registers.
template <typename T, int K, bool ACT> struct RowData {
    static constexpr int V = Elem<T>::CH;
    uint4 x[K], d[K], a[ACT ? K : 1];
    float mean, rstd;
    template <typename C>
    __device__ __forceinline__ void load(const C& at, const T* __restrict__ xs, const T* __restrict__ dout, const T* __restrict__ act,
                                         const float* __restrict__ ms, const float* __restrict__ rs, int64_t row, int cols) {
        at.load(xs + row * cols, x);
        at.load(dout + row * cols, d);
        if constexpr (ACT) at.load(act + row * cols, a);
        mean = ms[row];
        rstd = rs[row];
    }
    __device__ __forceinline__ void unpack(float (&xv)[K][V], float (&g)[K][V]) const {      // x, and dout behind the ReLU
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Chunk<T>::unpack(x[k], xv[k]);
            Chunk<T>::unpack(d[k], g[k]);
            if constexpr (ACT) {
                float av[V];
                Chunk<T>::unpack(a[k], av);
#pragma unroll
                for (int e = 0; e < V; ++e) g[k][e] = av[e] > 0.f ? g[k][e] : 0.f;
            }
        }
    }
};

// the row's averages of g and g xhat from this thread's sums
template <int TPR>
__device__ __forceinline__ void row_averages(float& c1, float& c2, float2* part, float inv) {
    c1 = lanes_sum<wave_lanes(TPR)>(c1);
    c2 = lanes_sum<wave_lanes(TPR)>(c2);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = make_float2(c1, c2);
        __syncthreads();
        const float2 p = part[threadIdx.x & 15];
        c1 = waves_sum(p.x);
        c2 = waves_sum(p.y);
    }
    c1 *= inv;
    c2 *= inv;
}

// dx, and this workgroup's sums for dweight and dbias.  A thread has the same columns in every row it works on: its parts of dweight and
// dbias stay in registers until the last row.  Then the R row groups of a workgroup are added up in LDS and one partial row [2][cols] a
// workgroup goes to scratch (partial == NULL: no weight, no sums).
template <typename T, int TPR, int K, Mode MODE, bool ACT>
__global__ __launch_bounds__(block_threads(TPR)) void ln_bwd_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                    const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                    const T* __restrict__ dout, const T* __restrict__ act, T* __restrict__ dx,
                                                                    float* __restrict__ partial, int64_t rows, int cols) {
    constexpr int V = Elem<T>::CH, R = TPR > 64 ? 1 : 256 / TPR;
    constexpr bool WAVES = TPR > 64, HOLD = holds_weights(TPR);
    const int64_t stride = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + (WAVES ? 0 : threadIdx.x / TPR);
    const Cols<T, TPR, K, MODE> at(cols, x + row * cols);
    const float inv = 1.f / (float)cols;
    __shared__ float2 part[2][WAVES ? 16 : 1];
    if constexpr (WAVES) {
        if (threadIdx.x < 16) part[0][threadIdx.x] = part[1][threadIdx.x] = make_float2(0.f, 0.f);
        __syncthreads();
    }
    float wf[HOLD ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if constexpr (HOLD) at.load(w, 1.f, k, wf[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k][e] = db[k][e] = 0.f;
    }
    RowData<T, K, ACT> in;
    if (row < rows) in.load(at, x, dout, act, mean, rstd, row, cols);
    for (int turn = 0; row < rows; row += stride, turn ^= 1) {
        int64_t again = 0;
        if constexpr (!HOLD) asm volatile("" : "+s"(again));      // (see ln_fwd_kernel)
        float xh[K][V], g[K][V];
        in.unpack(xh, g);
        const float m = in.mean, r = in.rstd;
        if (row + stride < rows) in.load(at, x, dout, act, mean, rstd, row + stride, cols);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int kw = HOLD ? k : 0;
            if constexpr (!HOLD) at.load(w ? w + again : w, 1.f, k, wf[0]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[k][e] = (xh[k][e] - m) * r;
                const float d = at.own(k, e) ? g[k][e] : 0.f;
                db[k][e] += d;
                dw[k][e] = fmaf(d, xh[k][e], dw[k][e]);
                g[k][e] *= wf[kw][e];
                const float go = at.own(k, e) ? g[k][e] : 0.f;
                c1 += go;
                c2 = fmaf(go, xh[k][e], c2);
            }
        }
        row_averages<TPR>(c1, c2, part[turn], inv);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = r * fmaf(-xh[k][e], c2, g[k][e] - c1);
            at.store(dx + row * cols, k, y);
        }
    }
    if (!partial) return;
    // one row group a workgroup: the registers are the workgroup's sums; several: added up in LDS in the order of the groups
    __shared__ float red[R > 1 ? R * TPR * K * V : 1];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float(&v)[K][V] = half == 0 ? dw : db;
        float* to = partial + ((int64_t)blockIdx.x * 2 + half) * cols;
        if constexpr (R > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at.own(k, e)) red[threadIdx.x / TPR * (TPR * K * V) + at.first_col(k) + e] = v[k][e];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += 256) {
                float s = 0.f;
#pragma unroll 8
                for (int i = 0; i < R; ++i) s += red[i * (TPR * K * V) + c];
                to[c] = s;
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (at.own(k, e)) to[at.first_col(k) + e] = v[k][e];
        }
    }
}

// Few rows: one launch.  dweight and dbias need the given mean and rstd only, not what dx needs from a whole row, so workgroups of their
// own sum 8 chunks of columns each over all rows, beside those that compute dx; x and dout are read twice (the second time from a
// cache), nothing goes through scratch.
template <typename T, int TPR, int K, bool ACT>
__global__ __launch_bounds__(block_threads(TPR)) void ln_bwd_few_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                        const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                        const T* __restrict__ dout, const T* __restrict__ act,
                                                                        T* __restrict__ dx, float* __restrict__ dw_out,
                                                                        float* __restrict__ db_out, int accumulate, int rows, int cols,
                                                                        int dx_blocks) {
    constexpr int V = Elem<T>::CH, R = TPR > 64 ? 1 : 256 / TPR;
    constexpr bool WAVES = TPR > 64;
    const int waves = (int)blockDim.x / 64;
    if ((int)blockIdx.x < dx_blocks) {
        const Cols<T, TPR, K, PLAIN> at(cols, x);
        __shared__ float2 part[WAVES ? 16 : 1];
        if constexpr (WAVES) {
            if (threadIdx.x < 16) part[threadIdx.x] = make_float2(0.f, 0.f);
            __syncthreads();
        }
        const int row = (int)blockIdx.x * R + (WAVES ? 0 : (int)threadIdx.x / TPR);
        if (row >= rows) return;                            // (with barriers a workgroup has one row, and there are no more of them)
        RowData<T, K, ACT> in;
        in.load(at, x, dout, act, mean, rstd, row, cols);
        float xh[K][V], g[K][V], c1 = 0.f, c2 = 0.f;
        in.unpack(xh, g);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float wf[V];
            at.load(w, 1.f, k, wf);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[k][e] = (xh[k][e] - in.mean) * in.rstd;
                g[k][e] *= wf[e];
                const float go = at.own(k, e) ? g[k][e] : 0.f;
                c1 += go;
                c2 = fmaf(go, xh[k][e], c2);
            }
        }
        row_averages<TPR>(c1, c2, part, 1.f / (float)cols);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = in.rstd * fmaf(-xh[k][e], c2, g[k][e] - c1);
            at.store(dx + (int64_t)row * cols, k, y);
        }
        return;
    }
    constexpr int LANES = 8;
    const int step = (int)blockDim.x / LANES;
    __shared__ float red[2][block_threads(TPR) / 64][LANES * V];
    const int lane = (int)threadIdx.x % LANES;
    const Piece<T, int, TPR == 2> piece((((int)blockIdx.x - dx_blocks) * LANES + lane) * V, cols);
    float dw[V], db[V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 4
    for (int row = (int)threadIdx.x / LANES; row < rows; row += step) {
        const int64_t i = (int64_t)row * cols;
        float xv[V], d[V];
        Chunk<T>::unpack(piece.load(x + i), xv);
        Chunk<T>::unpack(piece.load(dout + i), d);
        if constexpr (ACT) {
            float a[V];
            Chunk<T>::unpack(piece.load(act + i), a);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = a[e] > 0.f ? d[e] : 0.f;
        }
        const float m = mean[row], r = rstd[row];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            db[e] += d[e];
            dw[e] = fmaf(d[e], (xv[e] - m) * r, dw[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float sw = strided_sum<LANES>(dw[e]), sb = strided_sum<LANES>(db[e]);
        if ((threadIdx.x & 63) < LANES) {
            red[0][threadIdx.x >> 6][lane * V + e] = sw;
            red[1][threadIdx.x >> 6][lane * V + e] = sb;
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < LANES) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float sw = 0.f, sb = 0.f;
            for (int i = 0; i < waves; ++i) { sw += red[0][i][lane * V + e]; sb += red[1][i][lane * V + e]; }
            if (piece.own(e)) {
                const int c = piece.from + e;
                dw_out[c] = accumulate ? dw_out[c] + sw : sw;
                db_out[c] = accumulate ? db_out[c] + sb : sb;
            }
        }
    }
}

// dweight / dbias = (or +=) the sum of `parts` partial rows [2][cols]: 32 columns x 32 rows at a time, the rows' sums in a fixed order.
// Up to JOIN_BLOCKS workgroups of 32 columns, each of which has one turn below 2^25 columns: HIP launches less than 2^32 threads along an
// axis, which a workgroup for every 32 of the longest rows' columns would pass from 2^26 columns on.
constexpr int JOIN_BLOCKS = 1 << 21;
__global__ __launch_bounds__(1024) void ln_bwd_join_kernel(const float* __restrict__ partial, int parts, int64_t cols2, int cols,
                                                           float* __restrict__ dw, float* __restrict__ db, int accumulate) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols2; c0 += (int64_t)gridDim.x * 32) {      // (the same turns for a whole workgroup)
        const int64_t c = c0 + tx;
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
        __syncthreads();                   // (before the next turn writes red)
    }
}

// ---- rows longer than a workgroup's registers -----------------------------------------------------------------------------------------
// A thread's sums over such a row are fp32 within a chunk and fp64 from chunk to chunk: a chain of fp32 additions as long as the row takes
// would be off by more the longer it is (the mean of 2^25 times 0.3 by 3e-4 of it).  us against fp32 throughout: forward 2000 x 40000 fp32 218
// / 216, bf16 106 / 104, 4 x 40000 13.6 / 12.9 and 10.8 / 10.3; backward 1 % at most.
template <int V> __device__ __forceinline__ double chunk_sum(const float* f) {          // pairwise: exact for equal values
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = f[e];
#pragma unroll
    for (int n = V / 2; n > 0; n /= 2)
#pragma unroll
        for (int e = 0; e < n; ++e) s[e] += s[e + n];
    return (double)s[0];
}
template <int V> __device__ __forceinline__ double chunk_dot(const float* f, const float* g) {
    float s[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) s[e] = fmaf(f[e], g[e], f[e + V / 2] * g[e + V / 2]);
    return chunk_sum<V / 2>(s);
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, true),
                            __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ double lanes_sum_of_16(double v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}
__device__ __forceinline__ double sum_of_1024(double v, double* red) {
    v = lanes_sum_of_16(v);
    auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)__double2loint(v), (uint32_t)__double2loint(v), false, false);
    auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)__double2hiint(v), (uint32_t)__double2hiint(v), false, false);
    v = __hiloint2double((int)hi[0], (int)lo[0]) + __hiloint2double((int)hi[1], (int)lo[1]);
    lo = __builtin_amdgcn_permlane32_swap((uint32_t)__double2loint(v), (uint32_t)__double2loint(v), false, false);
    hi = __builtin_amdgcn_permlane32_swap((uint32_t)__double2hiint(v), (uint32_t)__double2hiint(v), false, false);
    v = __hiloint2double((int)hi[0], (int)lo[0]) + __hiloint2double((int)hi[1], (int)lo[1]);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return lanes_sum_of_16(red[threadIdx.x & 15]);
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_fwd_long_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                           T* __restrict__ out, float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                           int cols, float eps, int relu) {
    constexpr int V = Elem<T>::CH;
    __shared__ double red[16];
    const double inv = 1.0 / cols;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * cols;
        double s = 0.0;
        float f[V];
#pragma unroll 4
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const Piece<T, int64_t, false> piece(c, cols);
            Chunk<T>::unpack(piece.load(xr), f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = piece.own(e) ? f[e] : 0.f;
            s += chunk_sum<V>(f);
        }
        const float m = (float)(sum_of_1024(s, red) * inv);
        s = 0.0;
#pragma unroll 4
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const Piece<T, int64_t, false> piece(c, cols);
            Chunk<T>::unpack(piece.load(xr), f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = piece.own(e) ? f[e] - m : 0.f;
            s += chunk_dot<V>(f, f);
        }
        const float r = (float)(1.0 / sqrt(fma(sum_of_1024(s, red), inv, (double)eps)));
#pragma unroll 2
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const Piece<T, int64_t, false> piece(c, cols);
            float wf[V], bf[V];
            Chunk<T>::unpack(piece.load(xr), f);
            piece.load_vector(w, 1.f, wf);
            piece.load_vector(b, 0.f, bf);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[e] = fmaf((f[e] - m) * r, wf[e], bf[e]);
                if (relu && f[e] < 0.f) f[e] = 0.f;
            }
            piece.store(out + row * cols, f);
        }
        if (threadIdx.x == 0) { mean[row] = m; rstd[row] = r; }
    }
}

// d (dout behind the ReLU) and xhat of one chunk
template <typename T>
__device__ __forceinline__ void grad_piece(const Piece<T, int64_t, false>& piece, const T* __restrict__ x, const T* __restrict__ dout,
                                           const T* __restrict__ act, int64_t at, float m, float r, float* d, float* xh) {
    constexpr int V = Elem<T>::CH;
    Chunk<T>::unpack(piece.load(x + at), xh);
    Chunk<T>::unpack(piece.load(dout + at), d);
    if (act) {
        float a[V];
        Chunk<T>::unpack(piece.load(act + at), a);
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = a[e] > 0.f ? d[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) xh[e] = (xh[e] - m) * r;
}

template <typename T>
__global__ __launch_bounds__(1024) void ln_bwd_long_dx_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, const T* __restrict__ dout,
                                                              const T* __restrict__ act, T* __restrict__ dx, int64_t rows, int cols) {
    constexpr int V = Elem<T>::CH;
    __shared__ double red[16];
    const double inv = 1.0 / cols;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float m = mean[row], r = rstd[row];
        double s1 = 0.0, s2 = 0.0;
        float d[V], xh[V], wf[V];
#pragma unroll 2
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const Piece<T, int64_t, false> piece(c, cols);
            grad_piece<T>(piece, x, dout, act, row * cols, m, r, d, xh);
            piece.load_vector(w, 1.f, wf);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = piece.own(e) ? d[e] * wf[e] : 0.f;
            s1 += chunk_sum<V>(d);
            s2 += chunk_dot<V>(d, xh);
        }
        const float c1 = (float)(sum_of_1024(s1, red) * inv), c2 = (float)(sum_of_1024(s2, red) * inv);
#pragma unroll 2
        for (int64_t c = threadIdx.x * V; c < cols; c += 1024 * V) {
            const Piece<T, int64_t, false> piece(c, cols);
            grad_piece<T>(piece, x, dout, act, row * cols, m, r, d, xh);
            piece.load_vector(w, 1.f, wf);
#pragma unroll
            for (int e = 0; e < V; ++e) d[e] = r * fmaf(-xh[e], c2, d[e] * wf[e] - c1);
            piece.store(dx + row * cols, d);
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
    const Piece<T, int64_t, false> piece(c, cols);
    float dw[V], db[V], d[V], xh[V];
#pragma unroll
    for (int e = 0; e < V; ++e) dw[e] = db[e] = 0.f;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        grad_piece<T>(piece, x, dout, act, row * cols, mean[row], rstd[row], d, xh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            db[e] += d[e];
            dw[e] = fmaf(d[e], xh[e], dw[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (piece.own(e)) {
            partial[((int64_t)blockIdx.y * 2) * cols + piece.from + e] = dw[e];
            partial[((int64_t)blockIdx.y * 2 + 1) * cols + piece.from + e] = db[e];
        }
}

// ---- which split -----------------------------------------------------------------------------------------------------------------------
// Threads a row and chunks a thread, from the row's number of 16-byte chunks.  Up to 64 chunks: one a lane, the smallest power of two of
// lanes (several rows share a wavefront).  Then a wavefront with up to KMAX a lane, then a workgroup of the wavefronts it takes, up to 16.
// KMAX: what the registers hold with four wavefronts a SIMD -- 4 forward; backward, which keeps a weight and two sums a column, 16 values
// (4 fp32 chunks, 2 bf16).  From 7 wavefronts on fp32 stops at 2: 16384 x 8192 takes 200 / 293 us forward / backward as 1024 threads of 2
// chunks, 208 / 311 as 512 of 4, 20000 x 7000 takes 212 / 335 and 219 / 328; with 5 and 6 it is the other way, 20000 x 5000 157 / 242 and
// 143 / 224, 20000 x 6000 189 / 275 and 182 / 274.
struct Split { int tpr, k, threads; int64_t chunks; bool shifted = false; };      // tpr, k: the kernel's; threads: a workgroup's
Split ln_split(int dtype, int64_t chunks, int kmax) {
    if (chunks <= 64) {
        int tpr = 2;
        while (tpr < chunks) tpr *= 2;
        return {tpr, 1, 256, chunks};
    }
    for (int tpr = 64; tpr <= 1024; tpr = tpr == 64 ? 256 : tpr * 2)
        for (int k = 1; k <= (dtype == VINCE_F32 && tpr == 512 && chunks > 1536 ? 2 : kmax); k *= 2)
            if ((int64_t)tpr * k >= chunks) return {tpr, k, tpr == 64 ? 256 : (int)((chunks + 64 * k - 1) / (64 * k)) * 64, chunks};
    return {0, 0, 0, chunks};
}
int64_t ln_chunks(int dtype, int64_t cols) { const int v = dtype == VINCE_F32 ? 4 : 8; return (cols + v - 1) / v; }
int ln_bwd_k(int dtype) { return dtype == VINCE_F32 ? 4 : 2; }
Split ln_plain_split(int dtype, int cols, int kmax) { return ln_split(dtype, ln_chunks(dtype, cols), kmax); }
Split ln_row_split(int dtype, int cols, int kmax) {
    if (dtype == VINCE_BF16 && (cols & 1) && cols >= 16) {      // (shorter rows have hardly a whole chunk to align)
        Split s = ln_split(dtype, ln_chunks(dtype, cols + (int64_t)7), kmax);
        s.shifted = true;
        if (s.tpr) return s;
    }
    return ln_plain_split(dtype, cols, kmax);
}
Split ln_fwd_split(int dtype, int cols) { return ln_row_split(dtype, cols, 4); }
Split ln_bwd_split(int dtype, int cols) { return ln_row_split(dtype, cols, ln_bwd_k(dtype)); }
Split ln_few_split(int dtype, int cols) { return ln_plain_split(dtype, cols, ln_bwd_k(dtype)); }

// Workgroups: as many as have 4 MB of rows in their registers -- 2^18 chunks, of one tensor forward, of two backward -- and one a CU at
// least; each goes through its share of the rows.  More rows at a time are slower, fewer too (forward, 65536 x 2048 bf16, us at 256 / 512
// / 1024 / 2048 workgroups of 4 chunks a thread: 94 / 100 / 101 / 99; 10^6 x 128, of 1: 194 / 116 / 91 / 103; backward, 32768 x 4096, of 2:
// 142 / 152 / 176 at 256 / 512 / 1024, where every workgroup also leaves a partial row of 8 bytes a column to be read again).  The same
// number for every CU: 60000 x 1000 bf16 takes 39 us with 512, 44 with 520.  (Any multiple of 8 would do for Mode.)
int64_t ln_blocks(const Split& s, int64_t in_flight) {
    const int64_t n = s.tpr ? in_flight / ((s.tpr > 64 ? 1 : 256 / s.tpr) * s.chunks) : 1024;
    return n < 384 ? 256 : (n + 128) / 256 * 256;
}
int64_t ln_fwd_blocks(int64_t rows, const Split& s) {
    const int64_t r = s.tpr && s.tpr <= 64 ? 256 / s.tpr : 1, want = (rows + r - 1) / r, most = ln_blocks(s, 1 << 18);
    return want < most ? want : most;
}
// (at least four rows for each row group, so that the partial rows stay a small part of what is read; of the longest rows, which can be
// gigabytes, no more partial rows than rows)
int ln_bwd_blocks(int64_t rows, const Split& s) {
    const int64_t per = s.tpr && s.tpr <= 64 ? 4 * (256 / s.tpr) : 4, most = s.tpr ? ln_blocks(s, 1 << 17) : 256;
    const int64_t n = ((rows + per - 1) / per + 7) / 8 * 8;
    return (int)(!s.tpr && n > rows ? rows : n > most ? most : n);
}
// Few rows (ln_bwd_few_kernel): one launch for two and no scratch, against reading x and dout twice and column sums that one workgroup makes
// over all rows.  us on the device, two launches / one: 256 x 2048 fp32 7.4 / 4.5, 512 x 8192 bf16 14.9 / 11.0, 512 x 8192 fp32 16.5 / 17.1, 512 x
// 16384 fp32 26.7 / 28.6; 1024 x 512 fp32 7.0 / 7.4, 1024 x 2048 bf16 10.2 / 12.5.  A call with its host time, the second launch and the
// scratch's allocation among it: 16.4 / 11.8 for each of them but 512 x 8192 fp32, 16.5 / 16.6, and 512 x 16384, 26.3 / 28.1.
bool ln_bwd_few(int dtype, int64_t rows, int cols) {
    return ln_few_split(dtype, cols).tpr && (rows <= 512 || (rows <= 1024 && rows * ln_chunks(dtype, cols) <= 1 << 18));
}

template <typename T, int TPR, int K>
void launch_fwd(bool shifted, const dim3& grid, const dim3& block, const void* x, const float* w, const float* b, void* out, float* mean, float* rstd, int64_t rows, int cols,
                float eps, int relu, hipStream_t st) {
#define LN_LAUNCH(MODE) \
    hipLaunchKernelGGL((ln_fwd_kernel<T, TPR, K, MODE>), grid, block, 0, st, (const T*)x, w, b, (T*)out, mean, rstd, rows, cols, eps, relu)
    if (cols == (TPR > 64 ? (int)block.x : TPR) * K * Elem<T>::CH) {
        LN_LAUNCH(FULL);
        return;
    }
    if constexpr (sizeof(T) == 2) {
        if (shifted) {
            LN_LAUNCH(SHIFTED);
            return;
        }
    }
    LN_LAUNCH(PLAIN);
#undef LN_LAUNCH
}

template <typename T>
void run_fwd(int dtype, const void* x, const float* w, const float* b, void* out, float* mean, float* rstd, int64_t rows, int cols, float eps,
             int relu, hipStream_t st) {
    const Split s = ln_fwd_split(dtype, cols);
    const dim3 grid((unsigned)ln_fwd_blocks(rows, s)), block((unsigned)s.threads);
#define LN_CASE(TPR, K) \
    if (s.tpr == TPR && s.k == K) return launch_fwd<T, TPR, K>(s.shifted, grid, block, x, w, b, out, mean, rstd, rows, cols, eps, relu, st)
    LN_CASE(2, 1); LN_CASE(4, 1); LN_CASE(8, 1); LN_CASE(16, 1); LN_CASE(32, 1); LN_CASE(64, 1); LN_CASE(64, 2); LN_CASE(64, 4);
    LN_CASE(256, 2); LN_CASE(256, 4); LN_CASE(512, 4); LN_CASE(1024, 4);
    if constexpr (sizeof(T) == 4) { LN_CASE(1024, 2); }
#undef LN_CASE
    hipLaunchKernelGGL(ln_fwd_long_kernel<T>, grid, dim3(1024), 0, st, (const T*)x, w, b, (T*)out, mean, rstd,
                       rows, cols, eps, relu);
}

struct BwdArgs {
    const void *x, *dout, *act;
    const float *w, *mean, *rstd;
    void* dx;
    float *dw, *db, *partial;      // partial == NULL with dw: few rows, one launch
    int accumulate;
    int64_t rows;
    int cols, blocks, threads;     // blocks, threads: the launch's
    bool shifted;
};

template <typename T, int TPR, int K> void launch_bwd(const BwdArgs& a, hipStream_t st) {
    constexpr int R = TPR > 64 ? 1 : 256 / TPR, V = Elem<T>::CH;
    if (a.dw && !a.partial) {
        const int dx_blocks = (int)((a.rows + R - 1) / R), dw_blocks = (a.cols + 8 * V - 1) / (8 * V);
#define LN_LAUNCH(ACT)                                                                                                                        \
    hipLaunchKernelGGL((ln_bwd_few_kernel<T, TPR, K, ACT>), dim3(dx_blocks + dw_blocks), dim3(a.threads), 0, st, (const T*)a.x, a.w, a.mean, a.rstd, \
                       (const T*)a.dout, (const T*)a.act, (T*)a.dx, a.dw, a.db, a.accumulate, (int)a.rows, a.cols, dx_blocks)
        if (a.act) LN_LAUNCH(true);
        else LN_LAUNCH(false);
#undef LN_LAUNCH
        return;
    }
#define LN_LAUNCH(MODE, ACT)                                                                                                               \
    hipLaunchKernelGGL((ln_bwd_kernel<T, TPR, K, MODE, ACT>), dim3(a.blocks), dim3(a.threads), 0, st, (const T*)a.x, a.w, a.mean, a.rstd,  \
                       (const T*)a.dout, (const T*)a.act, (T*)a.dx, a.partial, a.rows, a.cols)
    if (a.cols == (TPR > 64 ? a.threads : TPR) * K * V) {
        if (a.act) LN_LAUNCH(FULL, true);
        else LN_LAUNCH(FULL, false);
        return;
    }
    if constexpr (sizeof(T) == 2) {
        if (a.shifted) {
            if (a.act) LN_LAUNCH(SHIFTED, true);
            else LN_LAUNCH(SHIFTED, false);
            return;
        }
    }
    if (a.act) LN_LAUNCH(PLAIN, true);
    else LN_LAUNCH(PLAIN, false);
#undef LN_LAUNCH
}

template <typename T> void run_bwd(const Split& s, const BwdArgs& a, hipStream_t st) {
#define LN_CASE(TPR, K) \
    if (s.tpr == TPR && s.k == K) return launch_bwd<T, TPR, K>(a, st)
    LN_CASE(2, 1); LN_CASE(4, 1); LN_CASE(8, 1); LN_CASE(16, 1); LN_CASE(32, 1); LN_CASE(64, 1); LN_CASE(64, 2); LN_CASE(256, 2);
    if constexpr (sizeof(T) == 4) {
        LN_CASE(64, 4); LN_CASE(256, 4); LN_CASE(512, 4); LN_CASE(1024, 2); LN_CASE(1024, 4);
    } else {
        LN_CASE(256, 1); LN_CASE(512, 2); LN_CASE(1024, 2);
    }
#undef LN_CASE
    hipLaunchKernelGGL(ln_bwd_long_dx_kernel<T>, dim3((unsigned)(a.rows < 1024 ? a.rows : 1024)), dim3(1024), 0, st, (const T*)a.x, a.w, a.mean,
                       a.rstd, (const T*)a.dout, (const T*)a.act, (T*)a.dx, a.rows, a.cols);
    if (a.dw)
        hipLaunchKernelGGL(ln_bwd_long_dw_kernel<T>, dim3((unsigned)((a.cols + (int64_t)(256 * Elem<T>::CH - 1)) / (256 * Elem<T>::CH)), (unsigned)a.blocks),
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
    return ln_bwd_few(dtype, rows, cols) ? 0 : (size_t)ln_bwd_blocks(rows, ln_bwd_split(dtype, cols)) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int vince_layer_norm_bwd(int dtype, const void* x, const float* weight, const float* mean, const float* rstd, const void* dout,
                                    const void* act, void* dx, float* dweight, float* dbias, int32_t accumulate, int64_t rows, int32_t cols,
                                    void* scratch, size_t scratch_bytes, void* stream) {
    LN_CHECK("vince_layer_norm_bwd");
    VINCE_CHECK_ARG((dweight == nullptr) == (dbias == nullptr), VINCE_E_ARG, "vince_layer_norm_bwd: dweight and dbias come together");
    hipStream_t st = (hipStream_t)stream;
    const bool few = rows > 0 && dweight && ln_bwd_few(dtype, rows, cols);
    const Split s = few ? ln_few_split(dtype, cols) : ln_bwd_split(dtype, cols);
    const int blocks = ln_bwd_blocks(rows, s);
    if (rows > 0) {
        VINCE_CHECK_ARG(x && mean && rstd && dout && dx, VINCE_E_ARG, "vince_layer_norm_bwd: null pointer");
        const size_t need = dweight ? vince_layer_norm_bwd_scratch_bytes(dtype, rows, cols) : 0;
        VINCE_CHECK_ARG(need == 0 || (scratch && scratch_bytes >= need), VINCE_E_ARG, "vince_layer_norm_bwd: scratch of %zu bytes", scratch_bytes);
        const uintptr_t dw = (uintptr_t)dweight, db = (uintptr_t)dbias, bytes = (uintptr_t)cols * sizeof(float);
        VINCE_CHECK_ARG(!dweight || dw + bytes <= db || db + bytes <= dw, VINCE_E_ARG, "vince_layer_norm_bwd: dweight and dbias share memory");
        const BwdArgs a = {x, dout, act, weight, mean, rstd, dx, dweight, dbias, few || !dweight ? nullptr : (float*)scratch, accumulate, rows, cols, blocks, s.threads, s.shifted};
        if (dtype == VINCE_F32) run_bwd<float>(s, a, st);
        else run_bwd<bf16_t>(s, a, st);
        VINCE_CHECK_LAUNCH();
    }
    if (dweight && !few && (rows > 0 || !accumulate)) {
        const int64_t groups = (2 * (int64_t)cols + 31) / 32;
        hipLaunchKernelGGL(ln_bwd_join_kernel, dim3((unsigned)(groups < JOIN_BLOCKS ? groups : JOIN_BLOCKS)), dim3(1024), 0, st, (const float*)scratch,
                           rows > 0 ? blocks : 0, 2 * (int64_t)cols, cols, dweight, dbias, accumulate);
        VINCE_CHECK_LAUNCH();
    }
    return VINCE_OK;
}
