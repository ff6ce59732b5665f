// out[M,N] = xs[m] ws[n] (x[M,K] * W[N,K]^T) with x and W in 8-bit floating point (e4m3) and one 32-bit scale for every row of x and
// of W: the product of a layer whose weights and activations are 8-bit.  Sums are 32-bit, the scales multiply the finished sum.
//
// Up to 16 tokens: bound by reading W once.  16 rows of W are the M side of a mma.sync.m16n8k32 tile and the tokens its N side.  The
// order in which the k values of a dot product are added is free: within every 64 values the four lanes of a quad take 16 consecutive ones
// each, for W and x alike, so that a lane's operands for two steps are 16 bytes of a row of W (two rows a lane), on their way through a ring
// in shared memory (weight_stream.cuh), and one 16-byte load of a row of x.  8 x 6144 x 4096 6.8 us (3.7 TB/s), 8 x 24576 x 4096 19.5 (5.2 TB/s).
// More: tcgen05, the weights on the lanes of tensor memory (gemm_wide.cuh: 77 x 4096 x 12288 14.6 us, 3.6 TB/s) or 256 x 256 tiles on pairs of
// SMs (gemm_e4m3_pair.cuh: 2048 x 24576 x 4096 148 us, 2.8 PFLOP/s, at the 1.5 GHz that the power limit leaves; 178 after a second of it).
//
// The reference's products are cublasSgemm (src/runtime/kernels/cuda_kernels.cu:892-908); it has none of 8-bit floats.
#include <cuda.h>
#include <type_traits>

#include "common.cuh"
#include "operands.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

#include "umma.cuh"
#include "gemm_wide.cuh"
#include "weight_stream.cuh"

constexpr int KC = stream::PIECE; // values (bytes) of a row in a step: two blocks of 64

int g_form = 0;                   // llme_gemm_e4m3_form()

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
// MT: 8-token tiles.  SHARE: warps that share a row group; AN_SM: warps an SM is to hold.
template <int MT, typename O, int SHARE, int AN_SM>
__global__ void __launch_bounds__(SHARE * 32, AN_SM / SHARE) skinny_kernel(Args a) {
    extern __shared__ __align__(128) unsigned char rings[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r = lane >> 2, n0 = blockIdx.x * 16;
    const unsigned char* w0 = a.w + (size_t)min(n0 + r, a.N - 1) * a.ldw + quad * 16;        // (a row past the end is read, never stored)
    const unsigned char* w1 = a.w + (size_t)min(n0 + r + 8, a.N - 1) * a.ldw + quad * 16;
    // (lanes without a token read the first one: a token's sums are its own, and theirs are not stored)
    const unsigned char* xp[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xp[m] = a.x + (size_t)(m * 8 + r < a.M ? m * 8 + r : 0) * a.ldx + quad * 16 + warp * KC;
    float acc[MT][4] = {};
    const int pieces = (a.K + KC - 1) / KC;
    const stream::Ring ring(rings);
    // (The kernel before may write what is taken for weights here: ahead of it goes only a request to have the first ones in L2.)
    if (quad == 0)
        for (int i = 0, t = warp; i < stream::DEPTH - 1 && t < pieces; ++i, t += SHARE) { stream::prefetch_l2(w0 + (size_t)t * KC); stream::prefetch_l2(w1 + (size_t)t * KC); }
    pdl_wait();
    pdl_launch_dependents();
    int ahead = warp;                                       // the piece that is brought next
    w0 += (size_t)warp * KC;
    w1 += (size_t)warp * KC;
    auto bring = [&](int slot) {
        // K is a multiple of 16: a lane's 16 bytes are inside or outside
        if (ahead < pieces) ring.bring(slot, w0, w1, ahead * KC + quad * 16 < a.K, ahead * KC + 64 + quad * 16 < a.K);
        stream::Ring::close();
        ahead += SHARE;
        w0 += SHARE * KC;
        w1 += SHARE * KC;
    };
#pragma unroll
    for (int i = 0; i < stream::DEPTH - 1; ++i) bring(i);
    int slot = 0;
    for (int t = warp; t < pieces; t += SHARE) {
        bring(slot == 0 ? stream::DEPTH - 1 : slot - 1);
        uint4 xv[MT][2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int m = 0; m < MT; ++m)
                xv[m][b] = t * KC + b * 64 + quad * 16 < a.K ? *reinterpret_cast<const uint4*>(xp[m] + b * 64) : make_uint4(0u, 0u, 0u, 0u);
        stream::Ring::wait();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            uint4 c0 = ring.read(slot, b, 0), c1 = ring.read(slot, b, 1);
            // (behind K nothing was brought: what lies there may be no number)
            if (t * KC + b * 64 + quad * 16 >= a.K) c0 = c1 = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mma_e4m3(acc[m], c0.x, c1.x, c0.y, c1.y, xv[m][b].x, xv[m][b].y);
                mma_e4m3(acc[m], c0.z, c1.z, c0.w, c1.w, xv[m][b].z, xv[m][b].w);
            }
        }
        slot = slot + 1 == stream::DEPTH ? 0 : slot + 1;
#pragma unroll
        for (int m = 0; m < MT; ++m) xp[m] += SHARE * KC;
    }
    // the sums of the warps that share a row group, added in their order
    float (*red)[16] = reinterpret_cast<float (*)[16]>(rings);                     // [warp * 8 MT + token][row]: over the rings, which are empty now
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp * MT * 8 + m * 8 + quad * 2 + (i & 1)][r + (i >> 1) * 8] = acc[m][i];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 8 * 16; i += SHARE * 32) {
        const int tok = i >> 4, row = n0 + (i & 15);
        if (tok >= a.M || row >= a.N) continue;
        float v = red[tok][i & 15];
#pragma unroll
        for (int w = 1; w < SHARE; ++w) v += red[w * MT * 8 + tok][i & 15];
        reinterpret_cast<O*>(a.out)[(size_t)tok * a.ldo + row] = from_f32<O>(v * a.xs[tok] * a.ws[row]);
    }
}

template <int MT, typename O, int SHARE, int AN_SM>
int launch_skinny(const Args& a, cudaStream_t s) {
    constexpr size_t smem = SHARE * stream::RING;
    static_assert(MT * 8 * 16 * 4 <= stream::RING, "the sums lie over the rings");
    auto kernel = skinny_kernel<MT, O, SHARE, AN_SM>;
    static LlmeGrants grants;
    if (cudaError_t e = llme_grant_smem(grants, kernel, smem)) LLME_REFUSE("gemm_e4m3: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llme_launch(kernel, dim3((a.N + 15) / 16), dim3(SHARE * 32), smem, s, a);
    LLME_LAUNCH_STATUS();
}
template <int MT, typename O>
int launch_skinny(const Args& a, cudaStream_t s) {
    return stream::with(stream::sharing((a.N + 15) / 16, (a.K + KC - 1) / KC, sm_count()), [&](auto warps, auto an_sm) {
        return launch_skinny<MT, O, decltype(warps)::value, decltype(an_sm)::value>(a, s);
    });
}

// More tokens than the weight-streaming kernel takes at once: 256 x 256 tiles on pairs of SMs, or narrower tiles with K cut over a cluster,
// whichever a model of its time says is faster (its cycles: wide::shape()).  A step of 128 values takes a pair 580 cycles, all tiles but the last 4,300 at least, which
// the way out of the one before takes, and starting and the last one's way out some 9,800 (384 x 4096 x 512 / 4096: 5.4 / 14.2 us, 2048 x 24576 x
// 128 29.2).
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
    const double tile = (a.K + 127) / 128 * 580.0;
    const double paired = (double)((tiles + pairs - 1) / pairs - 1) * (tile < 4300.0 ? 4300.0 : tile) + tile + 9800.0;
    if (g_form == 2 || (g_form == 0 && paired < cycles)) return pair::launch<O>(a, s);
    alignas(64) CUtensorMap mw, mx;
    if (int rc = make_map(&mw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.N, a.K, a.ldw, BM, wide::STEP)) return rc;
    if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.M, a.K, a.ldx, g.nt, wide::STEP)) return rc;
    return wide::launch<false, 4, false>(mw, mx, g, s);
}

template <typename O>
int launch(const Args& a, cudaStream_t s) {
    if (a.M > 16) return launch_wide<O>(a, s);
    return a.M <= 8 ? launch_skinny<1, O>(a, s) : launch_skinny<2, O>(a, s);
}

}  // namespace

// x [M,K] and w [N,K] e4m3 with row strides ldx, ldw (bytes), xs [M] and ws [N] their scales; out [M,N] float (out_dtype 0) or bfloat16
// (1), row stride ldo.  K and the strides are multiples of 16, the operands begin on 16 bytes.
LLME_API int llme_gemm_e4m3(const void* x, long long ldx, const float* xs, const void* w, long long ldw, const float* ws, void* out,
                            int out_dtype, long long ldo, int M, int N, int K, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !xs || !w || !ws || !out) LLME_REFUSE("gemm_e4m3: null pointer");
    if (M > MOST || N > MOST || K > MOST) LLME_REFUSE("gemm_e4m3: %d x %d x %d, at most %d of each", M, N, K, MOST);
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

// More than 16 tokens: 0 (the default): whichever kernel should be faster; 1: narrow tiles, K cut over clusters; 2: pairs of SMs.  For tests
// and measurements.
LLME_API int llme_gemm_e4m3_form(int how) {
    if (how >= 0 && how <= 2) g_form = how;
    return g_form;
}

// 0 if no bounded wait has given up since the last call (synchronises the device).
LLME_API int llme_gemm_e4m3_status() { LLME_TAKE_STATUS(g_status); }
