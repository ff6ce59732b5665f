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
// All arithmetic is 32-bit; the squares are added in a fixed order that depends on the row's width and on how the operands are aligned, not on the
// other rows.
//
// Bound by memory: a row stays in registers between the two passes over it, so it is read once.  Norm of 1,999 x 5,120 with a bfloat16 delta
// 18.6 us (6.0 TB/s), 4,096 x 4,096 bfloat16 rows 10.2 us (4.9 TB/s: in so short a time a launch's start and end weigh more), the gate of 2,048 x 17,408
// 31.4 us (5.7 TB/s); a handful of rows 1.2 to 2.5 us, a launch.
// Reference counterpart: rmsnorm_kernel and fused_silu_mul (src/runtime/kernels/cuda_kernels.cu:360-378, :993-1002) write 32-bit rows;
// the reference has no 8-bit rows.
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "operands.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

typedef __nv_bfloat16 bf16;
constexpr float LARGEST = 448.0f;
constexpr float LEAST = 7.8886090522101181e-31f;        // 2^-100

// N values (8, 2 or 1) of a row as they lie in memory: they stay so until they are needed, bfloat16 ones in half the registers.
template <typename T, int N> struct Piece;
template <int N> struct Piece<float, N> {
    float v[N];
    __device__ __forceinline__ void load(const float* p) {
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
    __device__ __forceinline__ float at(int i) const { return v[i]; }
};
template <int N> struct Piece<bf16, N> {
    unsigned raw[(N + 1) / 2];
    __device__ __forceinline__ void load(const bf16* p) {
        if constexpr (N == 8) *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(p);
        else if constexpr (N == 2) raw[0] = *reinterpret_cast<const unsigned*>(p);
        else raw[0] = *reinterpret_cast<const unsigned short*>(p);
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16); }
};
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

inline int least(int a, int b) { return a < b ? a : b; }

// ---- where a row comes from.  fetch() brings what N values at column j are made of, values() makes them.
template <typename T> struct FromRows {
    static constexpr bool NORM = false, EXACT = true;
    static int many(int pieces) { return least(sizeof(T) == 2 ? 4 : 2, pieces / 128); }      // pieces a thread holds where rows are many
    const T* x; long long ldx;
    template <int N> using Raw = Piece<T, N>;
    template <int N> __device__ __forceinline__ void fetch(int row, int j, Raw<N>& r) const { r.load(x + row * ldx + j); }
    template <int N> __device__ __forceinline__ void values(int, int, const Raw<N>& r, float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = r.at(i);
    }
};
// silu(g) for a g that has been through bfloat16, from the hardware's exponential and reciprocal: 2^-22 and 2^-23 of the value (and the rounding of
// the exponent), far below the 2^-4 of what it goes into.  As (g / 4) / (1 / 4 + exp(-g) / 4): the reciprocal of 1 + exp(-g) is below 2^-126 for g
// under -87.3, and would count as zero, a quarter's is a number wherever exp(-g) is one in 32 bits (below -88.7 it is not, and silu is 0).  Arithmetic
// bounds the gate's kernel: with the corrected reciprocal and the exponential for subnormal results 2,048 x 17,408 took 39.0 us.
__device__ __forceinline__ float silu_fast(float g) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -1.4426950408889634f, -2.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0.25f + e));
    return (0.25f * g) * r;
}
template <typename T> struct FromGate {
    static constexpr bool NORM = false, EXACT = false;
    static int many(int pieces) { return sizeof(T) == 4 ? 1 : (pieces <= 3 * 512 ? least(3, pieces / 128) : 6); }
    const T* x; long long ldx; int inter;
    template <int N> struct Raw { Piece<T, N> gate, up; };
    template <int N> __device__ __forceinline__ void fetch(int row, int j, Raw<N>& r) const {
        r.gate.load(x + row * ldx + j);
        r.up.load(x + row * ldx + inter + j);
    }
    template <int N> __device__ __forceinline__ void values(int, int, const Raw<N>& r, float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float g = r.gate.at(i);
            v[i] = (sizeof(T) == 2 ? silu_fast(g) : g / (1.0f + expf(-g))) * r.up.at(i);
        }
    }
};
// D: type of the contribution, or void where none is pending
template <typename D, typename G> struct FromNorm {
    static constexpr bool NORM = true, EXACT = false;
    static int many(int) { return 1; }             // (a row's squares are added in an order that must not depend on how many rows there are)
    const float* x; const D* delta; const G* gain; float* total; int size; float eps;
    template <int N> using Gain = Piece<G, N>;
    template <int N> struct Raw {
        Piece<float, N> x;
        Piece<std::conditional_t<std::is_void_v<D>, bf16, D>, N> d;
    };
    template <int N> __device__ __forceinline__ void fetch(int row, int j, Raw<N>& r) const {
        r.x.load(x + (long long)row * size + j);
        if constexpr (!std::is_void_v<D>) r.d.load(delta + (long long)row * size + j);
    }
    template <int N> __device__ __forceinline__ void values(int row, int j, const Raw<N>& r, float (&v)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = r.x.at(i);
        if constexpr (!std::is_void_v<D>) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += r.d.at(i);
            store<N>(total + (long long)row * size + j, v);
        }
    }
};

// The larger of `top` and |v|, NaN if either is one; for numbers without a sign the order of the values is that of their bits, infinity above
// all, NaN above that.
__device__ __forceinline__ float larger(float top, float v) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v)));
    return top;
}

// v / a from 1 / a and one correction: the quotient's error is known exactly, v - q a.  (Values of a few bits over a scale of theirs meet the
// middle between two e4m3 numbers often, and v times 1 / a would fall to either side of it.)
__device__ __forceinline__ float quotient(float v, float a, float f) {
    const float q = v * f;
    return fmaf(fmaf(-q, a, v), f, q);
}

// A row's scale and the factor that takes its values to e4m3: `top` the largest |h| before it is multiplied by r.
__device__ __forceinline__ float row_scale(float top, float r) {
    const float m = top * r;
    return (m >= LEAST ? m : (m < LEAST ? LEAST : m)) / LARGEST;       // (NaN stays)
}

// Whether the factor r / a that takes a norm's values to e4m3 is above the largest 32-bit number: in rows near zero under an eps below 2.8e-12, where
// r is above 6.0e5 and a may be as small as 2^-100 / 448.  The values then take the two parts one after the other: r makes of them the root of the
// row's width at most, and 1 / a is at most 448 2^100.  (Both parts for every row: 1,999 x 5,120 18.9 us, with this question 18.6.)
__device__ __forceinline__ bool in_two_parts(float f) { return f > 3.402823466e38f; }

// Sum and largest over the threads of a row: the lanes of a warp, or a block's.
template <bool BLOCK>
__device__ __forceinline__ void meet(float& ss, float& top, float* sums, unsigned* tops) {
    ss = warp_sum(ss);
    unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    top = __uint_as_float(bits);
    if (!BLOCK) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) { sums[warp] = ss; tops[warp] = bits; }
    __syncthreads();
    ss = warp_sum(lane < warps ? sums[lane] : 0.0f);
    bits = __reduce_max_sync(0xffffffffu, lane < warps ? tops[lane] : 0u);
    top = __uint_as_float(bits);
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
    typename Src::template Raw<N> raw[V];
#pragma unroll
    for (int k = 0; k < V; ++k)
        if ((t + k * step) * N < size) src.template fetch<N>(row, (t + k * step) * N, raw[k]);
    float v[V][N], ss = 0.0f, top = 0.0f;
    if constexpr (Src::NORM) {
        typename Src::template Gain<N> gain[V];
#pragma unroll
        for (int k = 0; k < V; ++k)
            if ((t + k * step) * N < size) gain[k].load(src.gain + (t + k * step) * N);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int j = (t + k * step) * N;
            if (j >= size) continue;
            src.template values<N>(row, j, raw[k], v[k]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                ss = fmaf(v[k][i], v[k][i], ss);
                top = larger(top, v[k][i] * gain[k].at(i));
            }
        }
        meet<BLOCK>(ss, top, sums, tops);
        const float r = 1.0f / sqrtf(ss / (float)size + src.eps), a = row_scale(top, r);
        float f = r / a;
        if (t == 0) scales[row] = a;
        if (in_two_parts(f)) {
            f = 1.0f / a;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i) v[k][i] *= r;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int j = (t + k * step) * N;
            if (j >= size) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] = (v[k][i] * f) * gain[k].at(i);
            store_e4m3<N>(q + row * ldq + j, v[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int j = (t + k * step) * N;
            if (j >= size) continue;
            src.template values<N>(row, j, raw[k], v[k]);
#pragma unroll
            for (int i = 0; i < N; ++i) top = larger(top, v[k][i]);
        }
        meet<BLOCK>(ss, top, sums, tops);
        const float a = row_scale(top, 1.0f), f = 1.0f / a;
        if (t == 0) scales[row] = a;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const int j = (t + k * step) * N;
            if (j >= size) continue;
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] = Src::EXACT ? quotient(v[k][i], a, f) : v[k][i] * f;
            store_e4m3<N>(q + row * ldq + j, v[k]);
        }
    }
}

// Any width and alignment, N values at a time (2 or 1): the row is read a second time.  (A norm's second pass reads the sums that the first one
// wrote: the same thread's.)
template <class Src, int N>
__global__ void __launch_bounds__(512) quantise_long_kernel(const Src src, unsigned char* __restrict__ q, long long ldq, float* __restrict__ scales, int rows, int size) {
    __shared__ float sums[32];
    __shared__ unsigned tops[32];
    pdl_launch_dependents();
    pdl_wait();
    const int row = (int)blockIdx.x;
    float ss = 0.0f, top = 0.0f, v[N];
    for (int j = N * (int)threadIdx.x; j < size; j += N * (int)blockDim.x) {
        typename Src::template Raw<N> raw;
        src.template fetch<N>(row, j, raw);
        src.template values<N>(row, j, raw, v);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (Src::NORM) {
                ss = fmaf(v[i], v[i], ss);
                v[i] *= to_f32(src.gain[j + i]);
            }
            top = larger(top, v[i]);
        }
    }
    meet<true>(ss, top, sums, tops);
    float r = 1.0f;
    if constexpr (Src::NORM) r = 1.0f / sqrtf(ss / (float)size + src.eps);
    const float a = row_scale(top, r);
    float f = r / a, first = 1.0f;
    if (Src::NORM && in_two_parts(f)) { f = 1.0f / a; first = r; }
    if (threadIdx.x == 0) scales[row] = a;
    for (int j = N * (int)threadIdx.x; j < size; j += N * (int)blockDim.x) {
        if constexpr (Src::NORM) {
            Piece<float, N> t;
            t.load((src.delta ? src.total : src.x) + (long long)row * size + j);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = (t.at(i) * first * f) * to_f32(src.gain[j + i]);
        } else {
            typename Src::template Raw<N> raw;
            src.template fetch<N>(row, j, raw);
            src.template values<N>(row, j, raw, v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = Src::EXACT ? quotient(v[i], a, f) : v[i] * f;
        }
        store_e4m3<N>(q + row * ldq + j, v);
    }
}

template <class Src, int N, int V>
void launch_block(const Src& src, unsigned char* q, long long ldq, float* scales, int rows, int size, cudaStream_t s) {
    const int threads = ((size / N + V - 1) / V + 31) / 32 * 32;
    llme_launch(quantise_kernel<Src, N, V, true>, dim3(rows), dim3(threads), 0, s, src, q, ldq, scales, rows, size);
}

int sm_count() {
    static const int n = [] {
        int dev = 0, v = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
        return v;
    }();
    return n;
}

// `vec`: the widest pieces that every operand takes.
// Few rows: as many threads a row as it has pieces of eight values, for the shortest way through.  Rows for several rounds of the SMs: several
// pieces a thread, so that more rows are on an SM at once and one's loads run while another's threads meet, as far as the registers of two and
// more blocks an SM go (1 / 2 / 3 / 4 / 6 pieces a thread: 4,096 rows of 4,096 bfloat16 values 13.4 / 11.1 / 10.7 / 10.2 / 10.5 us; the gate of
// 2,048 x 5,504 14.7 / 11.2 / 11.1 / 12.9 / 12.1, of 12,288 - / 22.8 / 22.8 / 26.9 / 22.4, of 17,408 - / - / - / 51.5 / 31.4, of 8,192 in 32 bits
// 24.9 / 27.1 / 30.3 / 33.6 / 41.6; the norm, 1,999 x 5,120, 18.7 / 18.7 / 19.2 / 20.4 / 23.0), but no fewer than 128 threads.  (A walk of as
// many blocks as fit, the next row's loads under way in shared memory, was slower throughout: 15.2 to 11.6 us for the first, 42.3 for 17,408.)
template <class Src>
int launch(const Src& src, unsigned char* q, long long ldq, float* scales, int rows, int size, int vec, cudaStream_t s) {
    const int pieces = size / vec;
    int v = rows >= 2 * sm_count() ? Src::many(pieces) : 1;
    while (v > 1 ? pieces > v * 640 : pieces > 1024) ++v;
    if (vec == 8 && pieces <= 32) llme_launch(quantise_kernel<Src, 8, 1, false>, dim3((rows + 3) / 4), dim3(128), 0, s, src, q, ldq, scales, rows, size);
    else if (vec == 8 && v <= 1) launch_block<Src, 8, 1>(src, q, ldq, scales, rows, size, s);
    else if (vec == 8 && v <= 2) launch_block<Src, 8, 2>(src, q, ldq, scales, rows, size, s);
    else if (vec == 8 && v <= 3) launch_block<Src, 8, 3>(src, q, ldq, scales, rows, size, s);
    else if (vec == 8 && v <= 4) launch_block<Src, 8, 4>(src, q, ldq, scales, rows, size, s);
    else if (vec == 8 && v <= 6) launch_block<Src, 8, 6>(src, q, ldq, scales, rows, size, s);
    else if (vec >= 2 && size / 2 <= 8 * 640) launch_block<Src, 2, 8>(src, q, ldq, scales, rows, size, s);
    else if (vec >= 2) llme_launch(quantise_long_kernel<Src, 2>, dim3(rows), dim3(512), 0, s, src, q, ldq, scales, rows, size);
    else llme_launch(quantise_long_kernel<Src, 1>, dim3(rows), dim3(size >= 2048 ? 512 : 128), 0, s, src, q, ldq, scales, rows, size);
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
    if (rows > MOST || size > MOST) LLME_REFUSE("rmsnorm_e4m3: %d rows of %d values, at most %d of either", rows, size, MOST);
    if (delta && !total) LLME_REFUSE("rmsnorm_e4m3: a contribution needs a place for the sum");
    if (!(eps > 0.0f)) LLME_REFUSE("rmsnorm_e4m3: eps must be positive");
    const Span at_x = span(x, rows, size, size, 4), at_delta = span(delta, rows, size, size, bytes_of(delta_dtype)), at_gain = span(gain, 1, size, size, bytes_of(gain_dtype));
    const Span at_total = span(delta ? total : nullptr, rows, size, size, 4), at_q = span(q, rows, size, size, 1), at_scales = span(scales, 1, rows, rows, 4);
    if (meets(at_q, {at_x, at_delta, at_gain, at_total, at_scales}) || meets(at_scales, {at_x, at_delta, at_gain, at_total}) ||
        meets(at_total, {at_delta, at_gain}) || (total != x && meets(at_total, {at_x})))
        LLME_REFUSE("rmsnorm_e4m3: an output lies over another operand");
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
    if (rows > MOST || size > MOST) LLME_REFUSE("rows_e4m3: %d rows of %d values, at most %d of either", rows, size, MOST);
    if (ldx < size || ldq < size) LLME_REFUSE("rows_e4m3: a row stride is shorter than the row");
    const Span at_x = span(x, rows, size, ldx, bytes_of(dtype)), at_q = span(q, rows, size, ldq, 1), at_scales = span(scales, 1, rows, rows, 4);
    if (meets(at_q, {at_x, at_scales}) || meets(at_scales, {at_x})) LLME_REFUSE("rows_e4m3: an output lies over another operand");
    const int vec = pieces_of(size, {{x, ldx, bytes_of(dtype)}, {q, ldq, 1}});
    if (dtype == LLME_F32) return launch(FromRows<float>{(const float*)x, ldx}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    if (dtype == LLME_BF16) return launch(FromRows<bf16>{(const bf16*)x, ldx}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    LLME_REFUSE("rows_e4m3: unsupported dtype %d", dtype);
}

// x [rows, 2 * size] = [gate | up] with row stride ldx; q [rows, size] = silu(gate) * up.
LLME_API int llme_swiglu_e4m3(const void* x, int dtype, long long ldx, void* q, long long ldq, float* scales, int rows, int size, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !q || !scales || size <= 0) LLME_REFUSE("swiglu_e4m3: null pointer or non-positive size");
    if (rows > MOST || size > MOST) LLME_REFUSE("swiglu_e4m3: %d rows of %d values, at most %d of either", rows, size, MOST);
    if (ldx < 2LL * size || ldq < size) LLME_REFUSE("swiglu_e4m3: a row stride is shorter than the row");
    const Span at_x = span(x, rows, 2LL * size, ldx, bytes_of(dtype)), at_q = span(q, rows, size, ldq, 1), at_scales = span(scales, 1, rows, rows, 4);
    if (meets(at_q, {at_x, at_scales}) || meets(at_scales, {at_x})) LLME_REFUSE("swiglu_e4m3: an output lies over another operand");
    const int vec = pieces_of(size, {{x, ldx, bytes_of(dtype)}, {q, ldq, 1}});
    if (dtype == LLME_F32) return launch(FromGate<float>{(const float*)x, ldx, size}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    if (dtype == LLME_BF16) return launch(FromGate<bf16>{(const bf16*)x, ldx, size}, (unsigned char*)q, ldq, scales, rows, size, vec, stream);
    LLME_REFUSE("swiglu_e4m3: unsupported dtype %d", dtype);
}
