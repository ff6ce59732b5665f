// out[M,N] = xs[m] ws[n] (x[M,K] * W[N,K]^T) with x and W in 8-bit floating point (e4m3) and one 32-bit scale for every row of x and
// of W: the product of a layer whose weights and activations are 8-bit.  Sums are 32-bit, the scales multiply the finished sum.
//
// A handful of tokens: bound by reading W once.  16 rows of W are the M side of a mma.sync.m16n8k32 tile and the tokens its N side.
// The order in which the k values of a dot product are added is free: within every 64 values the four lanes of a quad take 16
// consecutive ones each, for W and x alike, so that a lane's operands for two steps are one 16-byte load of a row of W (two rows a
// lane) and one of a row of x, straight into the registers the instruction reads.  A block owns 16 rows of W, its warps take the
// 128-value chunks of K in turn, and their partial sums are added in a fixed order.
//
// The reference's products are cublasSgemm (src/runtime/kernels/cuda_kernels.cu:892-908); it has none of 8-bit floats.
#include <cuda.h>

#include "common.cuh"
#include "operands.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

#include "umma.cuh"
#include "gemm_wide.cuh"

constexpr int KC = 128;           // values (bytes) per chunk: two blocks of 64

struct Args {
    const unsigned char* x; long long ldx; const float* xs;
    const unsigned char* w; long long ldw; const float* ws;
    void* out; long long ldo;
    int M, N, K;
};

#include "gemm_e4m3_pair.cuh"

__device__ __forceinline__ void mma_e4m3(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// weights are read once: do not keep them in L1
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// MT: 8-token tiles.  UNROLL: chunks of K whose loads a warp issues together.
template <int MT, typename O, int UNROLL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) skinny_kernel(Args a) {
    __shared__ float red[WARPS][MT * 8][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r = lane >> 2;
    const int n0 = blockIdx.x * 16;
    const unsigned char* w0 = a.w + (size_t)min(n0 + r, a.N - 1) * a.ldw + quad * 16;        // (a row past the end is read, never stored)
    const unsigned char* w1 = a.w + (size_t)min(n0 + r + 8, a.N - 1) * a.ldw + quad * 16;
    const unsigned char* xr[MT];
    bool xok[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        xok[m] = m * 8 + r < a.M;
        xr[m] = a.x + (size_t)(xok[m] ? m * 8 + r : 0) * a.ldx + quad * 16;
    }
    float acc[MT][4] = {};
    const int chunks = (a.K + KC - 1) / KC;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    pdl_wait();
    pdl_launch_dependents();
    for (int c = warp; c < chunks; c += UNROLL * WARPS) {
        uint4 wa[UNROLL][2], wb[UNROLL][2], xv[UNROLL][MT][2];
#pragma unroll
        for (int q = 0; q < UNROLL; ++q)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int k = (c + q * WARPS) * KC + b * 64;
                const bool ok = k + quad * 16 < a.K;              // K is a multiple of 16: a piece is inside or outside
                wa[q][b] = ok ? load_stream(w0 + k) : zero;
                wb[q][b] = ok ? load_stream(w1 + k) : zero;
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[q][m][b] = ok && xok[m] ? *reinterpret_cast<const uint4*>(xr[m] + k) : zero;
            }
#pragma unroll
        for (int q = 0; q < UNROLL; ++q)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    mma_e4m3(acc[m], wa[q][b].x, wb[q][b].x, wa[q][b].y, wb[q][b].y, xv[q][m][b].x, xv[q][m][b].y);
                    mma_e4m3(acc[m], wa[q][b].z, wb[q][b].z, wa[q][b].w, wb[q][b].w, xv[q][m][b].z, xv[q][m][b].w);
                }
    }
    // the warps' partial sums, added in a fixed order
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][m * 8 + quad * 2 + (i & 1)][r + (i >> 1) * 8] = acc[m][i];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 8 * 16; i += WARPS * 32) {
        const int tok = (i >> 4), row = n0 + (i & 15);
        if (tok >= a.M || row >= a.N) continue;
        float v = red[0][i >> 4][i & 15];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) v += red[w][i >> 4][i & 15];
        reinterpret_cast<O*>(a.out)[(size_t)tok * a.ldo + row] = from_f32<O>(v * a.xs[tok] * a.ws[row]);
    }
}

// More tokens than the weight-streaming kernel takes at once: 256 x 256 tiles on pairs of SMs, or narrower tiles with K cut over a cluster,
// whichever a model of its time says is faster.  A step of 128 values takes a pair 580 cycles, starting and the last tile some 11,000
// (64 x 4096 x 4096 / 12288: 16.2 / 34.2 us).
template <typename O>
int launch_wide(const Args& a, cudaStream_t s) {
    constexpr int out_f32 = sizeof(O) == 4;
    wide::Args g{};
    g.out = a.out; g.ldo = a.ldo; g.out_f32 = out_f32;
    g.M = a.M; g.N = a.N; g.K = a.K;
    g.xs = a.xs; g.ws = a.ws;
    g.vec_out = (uintptr_t)a.out % (out_f32 ? 16 : 8) == 0 && a.ldo % 4 == 0;
    double cycles;
    if (int rc = wide::shape<false, 4, false>(g, &cycles)) return rc;
    const long long pairs = sm_count() / 2, tiles = (long long)((a.M + 255) / 256) * ((a.N + 255) / 256);
    if ((double)((tiles + pairs - 1) / pairs) * ((a.K + 127) / 128) * 580.0 + 11000.0 < cycles) return pair::launch<O>(a, s);
    alignas(64) CUtensorMap mw, mx;
    if (int rc = make_map(&mw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.N, a.K, a.ldw, BM, wide::STEP)) return rc;
    if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.M, a.K, a.ldx, g.nt, wide::STEP)) return rc;
    return wide::launch<false, 4, false>(mw, mx, g, s);
}

template <typename O>
int launch(const Args& a, cudaStream_t s) {
    if (a.M > 16) return launch_wide<O>(a, s);
    const int groups = (a.N + 15) / 16;
    if (a.M <= 8) llme_launch(skinny_kernel<1, O, 4, 8>, dim3(groups), dim3(256), 0, s, a);
    else llme_launch(skinny_kernel<2, O, 2, 8>, dim3(groups), dim3(256), 0, s, a);
    LLME_LAUNCH_STATUS();
}

}  // namespace

// x [M,K] and w [N,K] e4m3 with row strides ldx, ldw (bytes), xs [M] and ws [N] their scales; out [M,N] float (out_dtype 0) or bfloat16
// (1), row stride ldo.  K and the strides are multiples of 16, the operands begin on 16 bytes.
LLME_API int llme_gemm_e4m3(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, void* out,
                            int out_dtype, long long ldo, int M, int N, int K, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !xs || !w || !ws || !out) LLME_REFUSE("gemm_e4m3: null pointer");
    if (K <= 0 || K % 16 || ldx % 16 || ldw % 16 || ldx < K || ldw < K) LLME_REFUSE("gemm_e4m3: K=%d ldx=%lld ldw=%lld is not supported (multiples of 16, rows that do not overlap)", K, ldx, ldw);
    if (((uintptr_t)x | (uintptr_t)w) % 16) LLME_REFUSE("gemm_e4m3: operands must be 16-byte aligned");
    if (ldo < N) LLME_REFUSE("gemm_e4m3: output row stride shorter than the row");
    if (meets(span(out, M, N, ldo, out_dtype == LLME_F32 ? 4 : 2), {span(x, M, K, ldx, 1), span(w, N, K, ldw, 1), span(xs, 1, M, M, 4), span(ws, 1, N, N, 4)}))
        LLME_REFUSE("gemm_e4m3: the output lies over an operand");
    const Args a{(const unsigned char*)x, ldx, xs, (const unsigned char*)w, ldw, ws, out, ldo, M, N, K};
    if (out_dtype == LLME_F32) return launch<float>(a, stream);
    if (out_dtype == LLME_BF16) return launch<bf16>(a, stream);
    LLME_REFUSE("gemm_e4m3: unsupported output dtype %d", out_dtype);
}

// 0 if no bounded wait has given up since the last call (synchronises the device).
LLME_API int llme_gemm_e4m3_status() { LLME_TAKE_STATUS(g_status); }
