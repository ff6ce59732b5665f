// Rows of 8-bit floating-point numbers (e4m3: no infinity, 448 the largest, NaN) with one 32-bit scale a row: what the product of
// 8-bit rows and weights (gemm_e4m3.cu) reads.  For a row h:
//
//     a = max(max_j |h_j|, 2^-100) / 448,   q_j = e4m3(h_j / a), rounded to the nearest, ties to even,
//
// so h_j is a q_j but for the rounding, half a step of 2^-3 at most.  (The lower bound keeps 1 / a finite: a row of zeros has the scale
// 2^-100 / 448 and zeros.  A row with a NaN or an infinity has a NaN or infinite scale, and NaN or zeros for q: its products are NaN.)
// Where h comes from:
//   * the RMS norm of the residual stream with the pending contribution added first: t = x + delta (written back), h = t / sqrt(mean(t^2)
//     + eps) * gain.  With m = max |t g| and r = 1 / sqrt(...) the row's largest is r m, so one pass over the row yields both the sum of
//     the squares and m, and the block meets once: a = max(r m, 2^-100) / 448, q = t (r / a) g;
//   * a matrix's rows as they are;
//   * silu(gate) * up of a [gate | up] product.
// All arithmetic is 32-bit; the squares are added in a fixed order that depends on the row's width alone.
//
// Bound by memory: a row stays in registers between the two passes over it, so it is read once.
// Reference counterpart: rmsnorm_kernel and fused_silu_mul (src/runtime/kernels/cuda_kernels.cu:360-378, :993-1002) write 32-bit rows;
// the reference has no 8-bit rows.
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

typedef __nv_bfloat16 bf16;
constexpr float LARGEST = 448.0f;
constexpr float LEAST = 7.8886090522101181e-31f;        // 2^-100

// N values (8, 2 or 1) of a row as 32-bit ones
template <int N> __device__ __forceinline__ void load(const float* p, float (&v)[N]) {
    if constexpr (N == 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else if constexpr (N == 2) {
        const float2 a = *reinterpret_cast<const float2*>(p);
        v[0] = a.x; v[1] = a.y;
    } else {
        v[0] = p[0];
    }
}
template <int N> __device__ __forceinline__ void load(const bf16* p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = __bfloat162float(p[0]);
    } else {
        unsigned raw[N / 2];
        if constexpr (N == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
        else raw[0] = *reinterpret_cast<const unsigned*>(p);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            v[2 * i] = __uint_as_float(raw[i] << 16);
            v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
        }
    }
}
template <int N> __device__ __forceinline__ void store(float* p, const float (&v)[N]) {
    if constexpr (N == 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else if constexpr (N == 2) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
        p[0] = v[0];
    }
}
// two values to e4m3, the first in the low byte (values are at most 448 but for rounding; NaN stays NaN, infinity cannot come here)
__device__ __forceinline__ unsigned short e4m3_pair(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int N> __device__ __forceinline__ void store_e4m3(unsigned char* p, const float (&v)[N]) {
    if constexpr (N == 8) {
        uint2 w;
        w.x = e4m3_pair(v[0], v[1]) | (unsigned)e4m3_pair(v[2], v[3]) << 16;
        w.y = e4m3_pair(v[4], v[5]) | (unsigned)e4m3_pair(v[6], v[7]) << 16;
        *reinterpret_cast<uint2*>(p) = w;
    } else if constexpr (N == 2) {
        *reinterpret_cast<unsigned short*>(p) = e4m3_pair(v[0], v[1]);
    } else {
        p[0] = (unsigned char)e4m3_pair(v[0], 0.0f);
    }
}

// ---- where a row comes from.  fetch() brings N values at column j, and what else the column needs into `extra`; finish() makes the
// values that are quantised of them.
template <typename T> struct FromRows {
    static constexpr bool NORM = false;
    const T* x; long long ldx;
    template <int N> __device__ __forceinline__ void fetch(int row, int j, float (&v)[N], float (&)[N]) const { load<N>(x + row * ldx + j, v); }
    template <int N> __device__ __forceinline__ void finish(int, int, float (&)[N], float (&)[N]) const {}
};
template <typename T> struct FromGate {
    static constexpr bool NORM = false;
    const T* x; long long ldx; int inter;
    template <int N> __device__ __forceinline__ void fetch(int row, int j, float (&v)[N], float (&up)[N]) const {
        load<N>(x + row * ldx + j, v);
        load<N>(x + row * ldx + inter + j, up);
    }
    template <int N> __device__ __forceinline__ void finish(int, int, float (&v)[N], float (&up)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = sizeof(T) == 2 ? silu_mul_bf16(v[i], up[i]) : v[i] / (1.0f + expf(-v[i])) * up[i];
    }
};
// D: type of the contribution, or void where none is pending
template <typename D, typename G> struct FromNorm {
    static constexpr bool NORM = true;
    const float* x; const D* delta; const G* gain; float* total; int size; float eps;
    template <int N> __device__ __forceinline__ void fetch(int row, int j, float (&v)[N], float (&d)[N]) const {
        load<N>(x + (long long)row * size + j, v);
        if constexpr (!std::is_void_v<D>) load<N>(delta + (long long)row * size + j, d);
    }
    template <int N> __device__ __forceinline__ void finish(int row, int j, float (&v)[N], float (&d)[N]) const {
        if constexpr (!std::is_void_v<D>) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += d[i];
            store<N>(total + (long long)row * size + j, v);
        }
    }
};

// The largest of several |v| as bits: for numbers without a sign they are in the order of the values, infinity above all, NaN above that.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A row's scale and the factor that takes its values to e4m3: `top` the largest |h| before it is multiplied by r.
__device__ __forceinline__ float row_scale(unsigned top, float r) {
    const float m = __uint_as_float(top) * r;
    return (m >= LEAST ? m : (m < LEAST ? LEAST : m)) / LARGEST;       // (NaN stays)
}

// Sum and largest over the threads of a row: the lanes of a warp, or a block's.
template <bool BLOCK>
__device__ __forceinline__ void meet(float& ss, unsigned& top, float* sums, unsigned* tops) {
    ss = warp_sum(ss);
    top = __reduce_max_sync(0xffffffffu, top);
    if (!BLOCK) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) { sums[warp] = ss; tops[warp] = top; }
    __syncthreads();
    ss = warp_sum(lane < warps ? sums[lane] : 0.0f);
    top = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
}

// BLOCK: a block a row; else a warp a row.  V: pieces of N values a thread holds.
template <class Src, int N, int V, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? (V == 1 ? 1024 : 640) : 128) quantise_kernel(const Src src, unsigned char* __restrict__ q, long long ldq, float* __restrict__ scales, int rows, int size) {
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    const int row = BLOCK ? (int)blockIdx.x : (int)(blockIdx.x * 4 + (threadIdx.x >> 5));
    if (!BLOCK && row >= rows) return;
    const int t = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31), step = BLOCK ? (int)blockDim.x : 32;
    pdl_wait();
    float v[V][N], extra[V][N], gain[V][N];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int j = (t + k * step) * N;
        if (j >= size) continue;
        src.template fetch<N>(row, j, v[k], extra[k]);
        if constexpr (Src::NORM) load<N>(src.gain + j, gain[k]);
    }
    float ss = 0.0f;
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int j = (t + k * step) * N;
        if (j >= size) continue;
        src.template finish<N>(row, j, v[k], extra[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (Src::NORM) ss = fmaf(v[k][i], v[k][i], ss);
            top = max(top, magnitude(Src::NORM ? v[k][i] * gain[k][i] : v[k][i]));
        }
    }
    meet<BLOCK>(ss, top, sums, tops);
    float r = 1.0f;
    if constexpr (Src::NORM) r = 1.0f / sqrtf(ss / (float)size + src.eps);
    const float a = row_scale(top, r), f = r / a;
    if (t == 0) scales[row] = a;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int j = (t + k * step) * N;
        if (j >= size) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) v[k][i] = Src::NORM ? (v[k][i] * f) * gain[k][i] : v[k][i] * f;
        store_e4m3<N>(q + row * ldq + j, v[k]);
    }
}

// Any width and alignment: the row is read a second time.  (A norm's second pass reads the sums that the first one wrote: the same
// thread's.)
template <class Src>
__global__ void __launch_bounds__(512) quantise_long_kernel(const Src src, unsigned char* __restrict__ q, long long ldq, float* __restrict__ scales, int rows, int size) {
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int row = (int)blockIdx.x;
    float ss = 0.0f, v[1], extra[1], g[1];
    unsigned top = 0;
    for (int j = (int)threadIdx.x; j < size; j += (int)blockDim.x) {
        src.template fetch<1>(row, j, v, extra);
        src.template finish<1>(row, j, v, extra);
        if constexpr (Src::NORM) {
            load<1>(src.gain + j, g);
            ss = fmaf(v[0], v[0], ss);
            v[0] *= g[0];
        }
        top = max(top, magnitude(v[0]));
    }
    meet<true>(ss, top, sums, tops);
    float r = 1.0f;
    if constexpr (Src::NORM) r = 1.0f / sqrtf(ss / (float)size + src.eps);
    const float a = row_scale(top, r), f = r / a;
    if (threadIdx.x == 0) scales[row] = a;
    for (int j = (int)threadIdx.x; j < size; j += (int)blockDim.x) {
        if constexpr (Src::NORM) {
            load<1>((src.delta ? src.total : src.x) + (long long)row * size + j, v);
            load<1>(src.gain + j, g);
            v[0] = (v[0] * f) * g[0];
        } else {
            src.template fetch<1>(row, j, v, extra);
            src.template finish<1>(row, j, v, extra);
            v[0] *= f;
        }
        store_e4m3<1>(q + row * ldq + j, v);
    }
}

template <class Src, int N, int V>
void launch_block(const Src& src, unsigned char* q, long long ldq, float* scales, int rows, int size, cudaStream_t s) {
    const int threads = ((size / N + V - 1) / V + 31) / 32 * 32;
    llme_launch(quantise_kernel<Src, N, V, true>, dim3(rows), dim3(threads), 0, s, src, q, ldq, scales, rows, size);
}

// `vec`: the largest of 8, 2 and 1 values whose pieces begin on their own size in every operand
template <class Src>
int launch(const Src& src, unsigned char* q, long long ldq, float* scales, int rows, int size, int vec, cudaStream_t s) {
    const int pieces = size / vec;
    if (vec == 8 && pieces <= 32) llme_launch(quantise_kernel<Src, 8, 1, false>, dim3((rows + 3) / 4), dim3(128), 0, s, src, q, ldq, scales, rows, size);
    else if (vec == 8 && pieces <= 1024) launch_block<Src, 8, 1>(src, q, ldq, scales, rows, size, s);
    else if (vec == 8 && pieces <= 4 * 640) launch_block<Src, 8, 4>(src, q, ldq, scales, rows, size, s);
    else if (vec >= 2 && size / 2 <= 8 * 640) launch_block<Src, 2, 8>(src, q, ldq, scales, rows, size, s);
    else llme_launch(quantise_long_kernel<Src>, dim3(rows), dim3(size >= 2048 ? 512 : 128), 0, s, src, q, ldq, scales, rows, size);
    LLME_LAUNCH_STATUS();
}

// The widest pieces (8, 2 or 1 values) that every operand takes: an address and the distance of its rows in values of `bytes` each.
struct Operand { const void* at; long long stride; int bytes; };
int pieces_of(int size, std::initializer_list<Operand> operands) {
    for (const int n : {8, 2}) {
        bool fits = size % n == 0;
        for (const Operand& o : operands) {
            const int piece = n * o.bytes < 16 ? n * o.bytes : 16;          // bytes of a load
            fits = fits && (uintptr_t)o.at % piece == 0 && o.stride * o.bytes % piece == 0;
        }
        if (fits) return n;
    }
    return 1;
}
int bytes_of(int dtype) { return dtype == LLME_F32 ? 4 : 2; }

template <typename D>
int norm(const float* x, const void* delta, const void* gain, int gain_dtype, float* total, unsigned char* q, float* scales, int rows, int size, float eps, int vec, cudaStream_t s) {
    if (gain_dtype == LLME_F32) return launch(FromNorm<D, float>{x, (const D*)delta, (const float*)gain, total, size, eps}, q, size, scales, rows, size, vec, s);
    if (gain_dtype == LLME_BF16) return launch(FromNorm<D, bf16>{x, (const D*)delta, (const bf16*)gain, total, size, eps}, q, size, scales, rows, size, vec, s);
    LLME_REFUSE("rmsnorm_e4m3: unsupported gain dtype %d", gain_dtype);
}

}  // namespace

// x [rows, size] 32-bit; delta nullable, then total = x + delta (total may be x); q [rows, size] e4m3, scales [rows].
LLME_API int llme_rmsnorm_e4m3(const float* x, const void* delta, int delta_dtype, const void* gain, int gain_dtype, float* total,
                               void* q, float* scales, int rows, int size, float eps, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !gain || !q || !scales || size <= 0) LLME_REFUSE("rmsnorm_e4m3: null pointer or non-positive size");
    if (delta && !total) LLME_REFUSE("rmsnorm_e4m3: a contribution needs a place for the sum");
    if (!(eps > 0.0f)) LLME_REFUSE("rmsnorm_e4m3: eps must be positive");
    const int vec = pieces_of(size, {{x, size, 4}, {delta, size, bytes_of(delta_dtype)}, {gain, size, bytes_of(gain_dtype)}, {total, size, 4}, {q, size, 1}});
    unsigned char* out = (unsigned char*)q;
    if (!delta) return norm<void>(x, nullptr, gain, gain_dtype, nullptr, out, scales, rows, size, eps, vec, stream);
    if (delta_dtype == LLME_F32) return norm<float>(x, delta, gain, gain_dtype, total, out, scales, rows, size, eps, vec, stream);
    if (delta_dtype == LLME_BF16) return norm<bf16>(x, delta, gain, gain_dtype, total, out, scales, rows, size, eps, vec, stream);
    LLME_REFUSE("rmsnorm_e4m3: unsupported delta dtype %d", delta_dtype);
}

// x [rows, size] with row stride ldx (elements); q [rows, size] e4m3 with row stride ldq.
LLME_API int llme_rows_e4m3(const void* x, int dtype, long long ldx, void* q, long long ldq, float* scales, int rows, int size, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !q || !scales || size <= 0) LLME_REFUSE("rows_e4m3: null pointer or non-positive size");
    if (ldx < size || ldq < size) LLME_REFUSE("rows_e4m3: a row stride is shorter than the row");
    const int vec = pieces_of(size, {{x, ldx, bytes_of(dtype)}, {q, ldq, 1}});
    if (dtype == LLME_F32) return launch(FromRows<float>{(const float*)x, ldx}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    if (dtype == LLME_BF16) return launch(FromRows<bf16>{(const bf16*)x, ldx}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    LLME_REFUSE("rows_e4m3: unsupported dtype %d", dtype);
}

// x [rows, 2 * size] = [gate | up] with row stride ldx; q [rows, size] = silu(gate) * up.
LLME_API int llme_swiglu_e4m3(const void* x, int dtype, long long ldx, void* q, long long ldq, float* scales, int rows, int size, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !q || !scales || size <= 0) LLME_REFUSE("swiglu_e4m3: null pointer or non-positive size");
    if (ldx < 2LL * size || ldq < size) LLME_REFUSE("swiglu_e4m3: a row stride is shorter than the row");
    const int vec = pieces_of(size, {{x, ldx, bytes_of(dtype)}, {q, ldq, 1}});
    if (dtype == LLME_F32) return launch(FromGate<float>{(const float*)x, ldx, size}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    if (dtype == LLME_BF16) return launch(FromGate<bf16>{(const bf16*)x, ldx, size}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    LLME_REFUSE("swiglu_e4m3: unsupported dtype %d", dtype);
}
