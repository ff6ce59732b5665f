// out[M,N] = x[M,K] * w^T with w[n,k] = s[n,g] (c[n,k] - z[n,g]), g = k / G: bfloat16 rows times weights of 4 bits (c in 0..15) with a
// bfloat16 scale and a zero point (8 where none are given) for every G = 32, 64 or 128 neighbouring values of a weight row.
//
// How the codes lie: a row in blocks of 128 values (the last one filled up with zeros), 64 bytes each.  Word 4 q + j of a block's
// sixteen 32-bit words holds values 32 j + 8 q .. + 7, the even ones in the low half, the odd ones in the high half, four bits each, in
// order.  So lane q of a quad finds in ONE 16-byte load eight values of each of the block's four runs of 32: the 16 values of a matrix
// instruction always lie in one group, whichever G.  And (word >> 4 p) & 0x000f000f are the codes of two neighbouring values in the two
// halves of a register: with 0x4300 in front of each they are the bfloat16 numbers 128 + c, from which 128 + z is subtracted exactly.
//
// A handful of tokens: bound by reading the codes.  As in the bfloat16 product (gemm_skinny.cu) 16 weight rows are the M side of a
// mma.sync.m16n8k16 tile and the tokens its N side.  The codes c - z enter the instruction as they are; a group's sums are multiplied by
// its scale, in 32-bit, when the group ends: no weight is rounded.
//
// The reference's weight-only product has 8-bit blocks (src/runtime/kernels/cuda_kernels.cu:296-358); it has none of 4 bits.
#include <cuda.h>

#include "common.cuh"
#include "operands.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

#include "umma.cuh"
#include "gemm_wide.cuh"

constexpr int BLOCK_K = 128, BLOCK_BYTES = 64;

struct Args {
    const bf16* x; long long ldx;
    const unsigned char* w; long long ldw;                  // bytes from row to row
    const bf16* scales; const unsigned char* zeros; long long lds;      // values from row to row of both
    bf16* out; long long ldo;
    int M, N, K;
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// weights are read once: do not keep them in L1
__device__ __forceinline__ uint4 load_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// codes 2p and 2p + 1 of a word as bfloat16 numbers minus z (`bias` holds 128 + z twice)
__device__ __forceinline__ unsigned two_codes(unsigned word, int p, __nv_bfloat162 bias) {
    const unsigned c = ((word >> (4 * p)) & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), bias);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ __nv_bfloat162 bias_of(unsigned zero) {
    const unsigned b = 0x43004300u | zero | zero << 16;
    return *reinterpret_cast<const __nv_bfloat162*>(&b);
}

// MT: 8-token tiles.  RUNS: runs of 32 values in a group (1, 2 or 4).  UNROLL: blocks of 128 values whose loads a warp issues together.
template <int MT, int RUNS, bool ZEROS, int UNROLL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) skinny_kernel(Args a) {
    constexpr int GROUPS = 4 / RUNS;                        // groups of a block of 128 values
    __shared__ float red[WARPS][MT * 8][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r = lane >> 2;
    const int n0 = blockIdx.x * 16;
    const size_t row0 = min(n0 + r, a.N - 1), row1 = min(n0 + r + 8, a.N - 1);            // (a row past the end is read, never stored)
    const unsigned char* w0 = a.w + row0 * a.ldw + quad * 16;
    const unsigned char* w1 = a.w + row1 * a.ldw + quad * 16;
    const bf16* xr[MT];
    bool xok[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        xok[m] = m * 8 + r < a.M;
        xr[m] = a.x + (size_t)(xok[m] ? m * 8 + r : 0) * a.ldx + quad * 8;
    }
    float acc[MT][4] = {};
    const int blocks = (a.K + BLOCK_K - 1) / BLOCK_K, groups = (a.K + 32 * RUNS - 1) / (32 * RUNS);
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    pdl_wait();
    pdl_launch_dependents();
    for (int c = warp; c < blocks; c += UNROLL * WARPS) {
        uint4 wa[UNROLL], wb[UNROLL];
#pragma unroll
        for (int q = 0; q < UNROLL; ++q) {
            const bool ok = c + q * WARPS < blocks;
            wa[q] = ok ? load_stream(w0 + (size_t)(c + q * WARPS) * BLOCK_BYTES) : zero;
            wb[q] = ok ? load_stream(w1 + (size_t)(c + q * WARPS) * BLOCK_BYTES) : zero;
        }
#pragma unroll
        for (int q = 0; q < UNROLL; ++q) {
            const int block = c + q * WARPS;
            if (block >= blocks) break;
            const unsigned word0[4] = {wa[q].x, wa[q].y, wa[q].z, wa[q].w}, word1[4] = {wb[q].x, wb[q].y, wb[q].z, wb[q].w};
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const int group = block * GROUPS + g;
                if (group >= groups) break;                 // (behind K there are no scales)
                const float s0 = to_f32(a.scales[row0 * a.lds + group]), s1 = to_f32(a.scales[row1 * a.lds + group]);
                const __nv_bfloat162 z0 = bias_of(ZEROS ? a.zeros[row0 * a.lds + group] : 8u), z1 = bias_of(ZEROS ? a.zeros[row1 * a.lds + group] : 8u);
                float sum[MT][4] = {};
#pragma unroll
                for (int j = g * RUNS; j < (g + 1) * RUNS; ++j) {
                    const int k = block * BLOCK_K + j * 32;
                    unsigned v0[4], v1[4];
#pragma unroll
                    for (int p = 0; p < 4; ++p) { v0[p] = two_codes(word0[j], p, z0); v1[p] = two_codes(word1[j], p, z1); }
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint4 xv = xok[m] && k + quad * 8 < a.K ? *reinterpret_cast<const uint4*>(xr[m] + k) : zero;   // (K is a multiple of 8)
                        mma_bf16(sum[m], v0[0], v1[0], v0[1], v1[1], xv.x, xv.y);
                        mma_bf16(sum[m], v0[2], v1[2], v0[3], v1[3], xv.z, xv.w);
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(i < 2 ? s0 : s1, sum[m][i], acc[m][i]);
            }
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
        a.out[(size_t)tok * a.ldo + row] = __float2bfloat16_rn(v);
    }
}

// More tokens than the weight-streaming kernel takes at once.
template <int RUNS, bool ZEROS>
int launch_wide(const Args& a, cudaStream_t s) {
    wide::Args g{};
    g.out = a.out; g.ldo = a.ldo;
    g.M = a.M; g.N = a.N; g.K = a.K;
    g.scales = a.scales; g.zeros = a.zeros; g.lds = a.lds;
    g.vec_out = (uintptr_t)a.out % 8 == 0 && a.ldo % 4 == 0;
    if (int rc = wide::shape<true, RUNS, ZEROS>(g, nullptr)) return rc;
    const long long w_bytes = (a.K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES;
    alignas(64) CUtensorMap mw, mx;
    if (int rc = wide::make_map_swizzled(&mw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.N, w_bytes, a.ldw, BM, BLOCK_BYTES, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
    if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.M, a.K, a.ldx, g.nt, 64)) return rc;
    return wide::launch<true, RUNS, ZEROS>(mw, mx, g, s);
}

template <int RUNS, bool ZEROS>
int launch(const Args& a, cudaStream_t s) {
    if (a.M > 16) return launch_wide<RUNS, ZEROS>(a, s);
    const int rows = (a.N + 15) / 16;
    if (a.M <= 8) llme_launch(skinny_kernel<1, RUNS, ZEROS, 4, 8>, dim3(rows), dim3(256), 0, s, a);
    else llme_launch(skinny_kernel<2, RUNS, ZEROS, 2, 8>, dim3(rows), dim3(256), 0, s, a);
    LLME_LAUNCH_STATUS();
}
template <int RUNS>
int launch(const Args& a, cudaStream_t s) { return a.zeros ? launch<RUNS, true>(a, s) : launch<RUNS, false>(a, s); }

}  // namespace

// x [M,K] bfloat16 with row stride ldx (elements, a multiple of 8; K too); w the codes [N, ceil(K / 128) * 64] with row stride ldw (bytes,
// a multiple of 16); scales [N, ceil(K / group)] bfloat16 and zeros of the same shape (values 0..15) or NULL, row stride lds; out [M,N]
// bfloat16, row stride ldo.
LLME_API int llme_gemm_int4(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, long long lds,
                            int group, void* out, long long ldo, int M, int N, int K, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !w || !scales || !out) LLME_REFUSE("gemm_int4: null pointer");
    if (K <= 0 || K % 8 || ldx % 8 || ldx < K) LLME_REFUSE("gemm_int4: K=%d ldx=%lld is not supported (multiples of 8, rows that do not overlap)", K, ldx);
    if (group != 32 && group != 64 && group != 128) LLME_REFUSE("gemm_int4: groups of %d values are not supported (32, 64 or 128)", group);
    if (ldw % 16 || ldw < (K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES) LLME_REFUSE("gemm_int4: rows of %lld bytes do not hold %d values in whole blocks", ldw, K);
    if (lds < (K + group - 1LL) / group) LLME_REFUSE("gemm_int4: rows of %lld scales are too short", lds);
    if (((uintptr_t)x | (uintptr_t)w) % 16) LLME_REFUSE("gemm_int4: operands must be 16-byte aligned");
    if (ldo < N) LLME_REFUSE("gemm_int4: output row stride shorter than the row");
    const long long groups = (K + group - 1LL) / group;
    if (meets(span(out, M, N, ldo, 2), {span(x, M, K, ldx, 2), span(w, N, (K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES, ldw, 1), span(scales, N, groups, lds, 2), span(zeros, N, groups, lds, 1)}))
        LLME_REFUSE("gemm_int4: the output lies over an operand");
    const Args a{(const bf16*)x, ldx, (const unsigned char*)w, ldw, (const bf16*)scales, (const unsigned char*)zeros, lds, (bf16*)out, ldo, M, N, K};
    if (group == 32) return launch<1>(a, stream);
    if (group == 64) return launch<2>(a, stream);
    return launch<4>(a, stream);
}

// 0 if no bounded wait has given up since the last call (synchronises the device).
LLME_API int llme_gemm_int4_status() { LLME_TAKE_STATUS(g_status); }
