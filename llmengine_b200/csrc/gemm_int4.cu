// out[M,N] = x[M,K] * w^T with w[n,k] = s[n,g] (c[n,k] - z[n,g]), g = k / G: bfloat16 rows times weights of 4 bits (c in 0..15) with a
// bfloat16 scale and a zero point (8 where none are given) for every G = 32, 64 or 128 neighbouring values of a weight row.
//
// How the codes lie: a row in blocks of 128 values (the last one filled up with zeros), 64 bytes each.  Word 4 q + j of a block's
// sixteen 32-bit words holds values 32 j + 8 q .. + 7, the even ones in the low half, the odd ones in the high half, four bits each, in
// order.  So lane q of a quad finds in ONE 16-byte load eight values of each of the block's four runs of 32: the 16 values of a matrix
// instruction always lie in one group, whichever G.  And (word >> 4 p) & 0x000f000f are the codes of two neighbouring values in the two
// halves of a register, from where one or two instructions make two bfloat16 numbers of them (eight_codes(), wide::Group).
//
// Up to 16 tokens: bound by reading the codes.  As in the bfloat16 product (gemm_skinny.cu) 16 weight rows are the M side of a
// mma.sync.m16n8k16 tile and the tokens its N side; the codes come through a ring in shared memory (weight_stream.cuh).  They enter the
// instruction as (c - z) 2^-6; a group's sums are multiplied by its scale, in 32-bit, when the group ends: no weight is rounded.
// 1 x 24576 x 4096, groups of 128: 13.6 us, 3.8 TB/s, where the loads alone take 10.1 and making numbers of the codes the rest; with zero points
// 15.4, in groups of 32 with zero points 21.8 (x in L2; from memory 14.8, 17.4, 22.9).  1 x 17408 x 5120 13.0 us, 1 x 4096 x 4096 4.4.
// More: tcgen05, the weights made into bfloat16 numbers in tensor memory, on single SMs (gemm_wide.cuh) or on pairs (gemm_int4_pair.cuh).
//
// The reference's weight-only product has 8-bit blocks (src/runtime/kernels/cuda_kernels.cu:296-358); it has none of 4 bits.
#include <cuda.h>
#include <type_traits>

#include "common.cuh"
#include "operands.cuh"

LLME_API const char* llme_last_error() { return llme_error_buffer(); }

namespace {

#include "umma.cuh"
#include "gemm_wide.cuh"
#include "weight_stream.cuh"
#include "gemm_int4_pair.cuh"

constexpr int BLOCK_K = 128, BLOCK_BYTES = 64;

int g_form = 0;                   // llme_gemm_int4_form()

struct Args {
    const bf16* x; long long ldx;
    const unsigned char* w; long long ldw;                  // bytes from row to row
    const bf16* scales; const unsigned char* zeros; long long lds;      // values from row to row of both
    void* out; long long ldo;
    int M, N, K;
    int together;                                           // scales and zero points that lie on their size: 2 a piece's, 1 a block's, 0 one
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A word's eight codes less the zero point, in the order of their values, as bfloat16 numbers of 2^-6: without a shift for half of them.  As
// bits of a bfloat16 number a code in the low four bits is c 2^-133, and one in the next four 16 c 2^-133 (the numbers below 2^-125 all have
// the same distance); the factors 2^127 and 2^123 make both c 2^-6, and the addend takes z 2^-6 off in the same instruction, exactly.
// (Arithmetic bounds this kernel: a logical instruction, a shift and one on two bfloat16 numbers all take two cycles a warp.)
__device__ __forceinline__ void eight_codes(unsigned word, __nv_bfloat162 minus_z, unsigned (&v)[4]) {
    const unsigned up = word >> 8;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const unsigned code = (p < 2 ? word : up) & (p & 1 ? 0x00f000f0u : 0x000f000fu), factor = p & 1 ? 0x7d007d00u : 0x7f007f00u;
        const __nv_bfloat162 w = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&code), *reinterpret_cast<const __nv_bfloat162*>(&factor), minus_z);
        v[p] = *reinterpret_cast<const unsigned*>(&w);
    }
}
// -z 2^-6, twice, of byte i of `z`: as bits of a bfloat16 number z is z 2^-133, and -2^127 of it is exact.
__device__ __forceinline__ __nv_bfloat162 minus_zero_point(unsigned z, int i) {
    const unsigned code = __byte_perm(z, 0u, 0x4040u | (unsigned)i * 0x0101u), factor = 0xff00ff00u;
    return __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&code), *reinterpret_cast<const __nv_bfloat162*>(&factor), __floats2bfloat162_rn(0.0f, 0.0f));
}

// BYTES neighbouring bytes, AT at a time.
template <int BYTES, int AT>
__device__ __forceinline__ void take(unsigned* to, const unsigned char* p) {
#pragma unroll
    for (int i = 0; i < BYTES; i += AT) {
        if constexpr (AT == 16) *reinterpret_cast<uint4*>(to + i / 4) = *reinterpret_cast<const uint4*>(p + i);
        else if constexpr (AT == 8) *reinterpret_cast<uint2*>(to + i / 4) = *reinterpret_cast<const uint2*>(p + i);
        else if constexpr (AT == 4) to[i / 4] = *reinterpret_cast<const unsigned*>(p + i);
        else if constexpr (AT == 2) to[i / 4] |= (unsigned)*reinterpret_cast<const unsigned short*>(p + i) << (8 * (i % 4));
        else to[i / 4] |= (unsigned)p[i] << (8 * (i % 4));
    }
}

// What goes with two rows' codes: the scales and zero points of a piece of COUNT groups.  (A load for every row brings all of them where they lie
// on their size: a load meets eight rows, which takes as long whatever it brings of each.)
template <int COUNT, bool ZEROS>
struct Factors {
    alignas(16) unsigned s[2][COUNT / 2], z[2][(COUNT + 3) / 4];
    template <int S_AT, int Z_AT>
    __device__ __forceinline__ void whole(const unsigned char* const (&scales)[2], const unsigned char* const (&zeros)[2], int first) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            take<2 * COUNT, S_AT>(s[r], scales[r] + 2 * (size_t)first);
            if (ZEROS) take<COUNT, Z_AT>(z[r], zeros[r] + first);
        }
    }
    __device__ __forceinline__ void fetch(const Args& a, const unsigned char* const (&scales)[2], const unsigned char* const (&zeros)[2], int first, int groups) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (unsigned& v : s[r]) v = 0;
#pragma unroll
            for (unsigned& v : z[r]) v = 0;
        }
        if (first + COUNT <= groups) {
            if (a.together == 2) whole<2 * COUNT, COUNT>(scales, zeros, first);
            else if (COUNT > 2 && a.together == 1) whole<COUNT, COUNT / 2>(scales, zeros, first);
            else whole<2, 1>(scales, zeros, first);
        } else {                                            // (behind K there are no scales, and what they would multiply is zero)
#pragma unroll
            for (int i = 0; i < COUNT; ++i)
                if (first + i < groups)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        s[r][i / 2] |= (unsigned)*reinterpret_cast<const unsigned short*>(scales[r] + 2 * (size_t)(first + i)) << (16 * (i % 2));
                        if (ZEROS) z[r][i / 4] |= (unsigned)zeros[r][first + i] << (8 * (i % 4));
                    }
        }
    }
    __device__ __forceinline__ float scale(int r, int i) const { return __uint_as_float(i & 1 ? s[r][i / 2] & 0xffff0000u : s[r][i / 2] << 16); }
    __device__ __forceinline__ __nv_bfloat162 minus_zero(int r, int i) const { return ZEROS ? minus_zero_point(z[r][i / 4], i % 4) : __floats2bfloat162_rn(-0.125f, -0.125f); }
};

// MT: 8-token tiles.  RUNS: runs of 32 values in a group (1, 2 or 4).  O: the output's type.  SHARE: warps that share a row group; AN_SM: warps an SM is to hold.
template <int MT, int RUNS, bool ZEROS, typename O, int SHARE, int AN_SM>
__global__ void __launch_bounds__(SHARE * 32, AN_SM / SHARE) skinny_kernel(Args a) {
    constexpr int GROUPS = 4 / RUNS, PAIR = 2 * BLOCK_K;          // a piece of 128 bytes is two blocks of codes
    extern __shared__ __align__(128) unsigned char rings[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, r = lane >> 2, part = warp;
    const int n0 = blockIdx.x * 16;
    const size_t row0 = min(n0 + r, a.N - 1), row1 = min(n0 + r + 8, a.N - 1);            // (a row past the end is read, never stored)
    const unsigned char* w0 = a.w + row0 * a.ldw + quad * 16;
    const unsigned char* w1 = a.w + row1 * a.ldw + quad * 16;
    const unsigned char* const scales[2] = {reinterpret_cast<const unsigned char*>(a.scales + row0 * a.lds), reinterpret_cast<const unsigned char*>(a.scales + row1 * a.lds)};
    const unsigned char* const zeros[2] = {ZEROS ? a.zeros + row0 * a.lds : nullptr, ZEROS ? a.zeros + row1 * a.lds : nullptr};
    // (lanes without a token read the first one: a token's sums are its own, and theirs are not stored)
    const bf16* xp[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xp[m] = a.x + (size_t)(m * 8 + r < a.M ? m * 8 + r : 0) * a.ldx + quad * 8 + part * PAIR;
    float acc[MT][4] = {};
    const int blocks = (a.K + BLOCK_K - 1) / BLOCK_K, pieces = (blocks + 1) / 2, groups = (a.K + 32 * RUNS - 1) / (32 * RUNS);
    const stream::Ring ring(rings);
    // (The kernel before may write what is taken for weights here: ahead of it goes only a request to have the first ones in L2.)
    if (quad == 0)
        for (int i = 0, t = part; i < stream::DEPTH - 1 && t < pieces; ++i, t += SHARE) { stream::prefetch_l2(w0 + (size_t)t * stream::PIECE); stream::prefetch_l2(w1 + (size_t)t * stream::PIECE); }
    pdl_wait();
    pdl_launch_dependents();
    int ahead = part;                                       // the piece that is brought next
    w0 += (size_t)part * stream::PIECE;
    w1 += (size_t)part * stream::PIECE;
    auto bring = [&](int slot) {
        if (ahead < pieces) ring.bring(slot, w0, w1, true, 2 * ahead + 1 < blocks);
        stream::Ring::close();
        ahead += SHARE;
        w0 += SHARE * stream::PIECE;
        w1 += SHARE * stream::PIECE;
    };
#pragma unroll
    for (int i = 0; i < stream::DEPTH - 1; ++i) bring(i);
    Factors<2 * GROUPS, ZEROS> next, now;
    next.fetch(a, scales, zeros, 2 * part * GROUPS, groups);
    // a piece's products; `last`: the piece in which K ends
    auto multiply = [&](int slot, int t, auto last) {
        constexpr bool LAST = decltype(last)::value;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            // (the second block of the last piece may not be there: whatever codes lie in its place meet zeros)
            const uint4 c0 = ring.read(slot, b, 0), c1 = ring.read(slot, b, 1);
            const unsigned word0[4] = {c0.x, c0.y, c0.z, c0.w}, word1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                const float f0 = now.scale(0, b * GROUPS + g), f1 = now.scale(1, b * GROUPS + g);
                const __nv_bfloat162 z0 = now.minus_zero(0, b * GROUPS + g), z1 = now.minus_zero(1, b * GROUPS + g);
                float sum[MT][4] = {};
#pragma unroll
                for (int j = g * RUNS; j < (g + 1) * RUNS; ++j) {
                    const int k = b * BLOCK_K + j * 32;
                    unsigned v0[4], v1[4];
                    eight_codes(word0[j], z0, v0);
                    eight_codes(word1[j], z1, v1);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        uint4 xv = make_uint4(0u, 0u, 0u, 0u);
                        if (!LAST || t * PAIR + k + quad * 8 < a.K) xv = *reinterpret_cast<const uint4*>(xp[m] + k);      // (K is a multiple of 8)
                        mma_bf16(sum[m], v0[0], v1[0], v0[1], v1[1], xv.x, xv.y);
                        mma_bf16(sum[m], v0[2], v1[2], v0[3], v1[3], xv.z, xv.w);
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][i] = fmaf(i < 2 ? f0 : f1, sum[m][i], acc[m][i]);
            }
        }
    };
    int slot = 0;
    for (int t = part; t < pieces; t += SHARE) {
        bring(slot == 0 ? stream::DEPTH - 1 : slot - 1);
        now = next;
        next.fetch(a, scales, zeros, 2 * (t + SHARE) * GROUPS, groups);
        stream::Ring::wait();
        if ((t + 1) * PAIR <= a.K) multiply(slot, t, std::false_type{});
        else multiply(slot, t, std::true_type{});
        slot = slot + 1 == stream::DEPTH ? 0 : slot + 1;
#pragma unroll
        for (int m = 0; m < MT; ++m) xp[m] += SHARE * PAIR;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] *= 64.0f;                            // (the codes were numbers of 2^-6)
    // the sums of the warps that share a row group, added in their order
    float (*red)[16] = reinterpret_cast<float (*)[16]>(rings);                     // [warp * 8 MT + token][row]: over the rings, which are empty now
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp * MT * 8 + m * 8 + quad * 2 + (i & 1)][r + (i >> 1) * 8] = acc[m][i];
    __syncthreads();
    for (int i = part * 32 + lane; i < MT * 8 * 16; i += SHARE * 32) {
        const int tok = i >> 4, row = n0 + (i & 15);
        if (tok >= a.M || row >= a.N) continue;
        float v = red[tok][i & 15];
#pragma unroll
        for (int w = 1; w < SHARE; ++w) v += red[w * MT * 8 + tok][i & 15];
        reinterpret_cast<O*>(a.out)[(size_t)tok * a.ldo + row] = from_f32<O>(v);
    }
}

template <int MT, int RUNS, bool ZEROS, typename O, int SHARE, int AN_SM>
int launch_skinny(const Args& a, cudaStream_t s) {
    constexpr size_t smem = SHARE * stream::RING;
    static_assert(MT * 8 * 16 * 4 <= stream::RING, "the sums lie over the rings");
    auto kernel = skinny_kernel<MT, RUNS, ZEROS, O, SHARE, AN_SM>;
    static LlmeGrants grants;
    if (cudaError_t e = llme_grant_smem(grants, kernel, smem)) LLME_REFUSE("gemm_int4: cannot reserve %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    llme_launch(kernel, dim3((a.N + 15) / 16), dim3(SHARE * 32), smem, s, a);
    LLME_LAUNCH_STATUS();
}
template <int MT, int RUNS, bool ZEROS, typename O>
int launch_skinny(const Args& a, cudaStream_t s) {
    return stream::with(stream::sharing((a.N + 15) / 16, (a.K + 2 * BLOCK_K - 1) / (2 * BLOCK_K), sm_count()), [&](auto warps, auto an_sm) {
        return launch_skinny<MT, RUNS, ZEROS, O, decltype(warps)::value, decltype(an_sm)::value>(a, s);
    });
}

// More tokens than the weight-streaming kernel takes at once: pairs of SMs, or single ones with K cut over a cluster, whichever a model of its
// time says is faster.
template <int RUNS, bool ZEROS, typename O>
int launch_wide(const Args& a, cudaStream_t s) {
    const long long w_bytes = (a.K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES;
    alignas(64) CUtensorMap mw, mx;
    if (int rc = wide::make_map_swizzled(&mw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.N, w_bytes, a.ldw, BM, BLOCK_BYTES, CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
    wide::Args g{};
    g.out = a.out; g.ldo = a.ldo; g.out_f32 = sizeof(O) == 4;
    g.M = a.M; g.N = a.N; g.K = a.K;
    g.scales = a.scales; g.zeros = a.zeros; g.lds = a.lds;
    g.vec_out = (uintptr_t)a.out % (4 * sizeof(O)) == 0 && a.ldo % 4 == 0;
    double single, paired;
    if (int rc = wide::shape<true, RUNS, ZEROS>(g, &single)) return rc;
    pair::PairArgs p{a.out, a.ldo, a.M, a.N, a.K, 0, 0, 0, a.scales, a.zeros, a.lds};
    if (int rc = pair::shape<RUNS, ZEROS>(p, &paired)) return rc;
    if (g_form == 2 || (g_form == 0 && paired < single)) {
        if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.M, a.K, a.ldx, p.nt / 2, 64)) return rc;
        return pair::launch<RUNS, ZEROS, O>(mw, mx, p, s);
    }
    if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.M, a.K, a.ldx, g.nt, 64)) return rc;
    return wide::launch<true, RUNS, ZEROS>(mw, mx, g, s);
}

template <int RUNS, bool ZEROS, typename O>
int launch(const Args& a, cudaStream_t s) {
    if (a.M > 16) return launch_wide<RUNS, ZEROS, O>(a, s);
    return a.M <= 8 ? launch_skinny<1, RUNS, ZEROS, O>(a, s) : launch_skinny<2, RUNS, ZEROS, O>(a, s);
}
template <int RUNS, typename O>
int launch(const Args& a, cudaStream_t s) { return a.zeros ? launch<RUNS, true, O>(a, s) : launch<RUNS, false, O>(a, s); }

// What both entry points check and launch; O: the output's type.
template <typename O>
int product(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, long long lds, int group, void* out, long long ldo,
            int M, int N, int K, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (!x || !w || !scales || !out) LLME_REFUSE("gemm_int4: null pointer");
    if (M > MOST || N > MOST || K > MOST) LLME_REFUSE("gemm_int4: %d x %d x %d, at most %d of each", M, N, K, MOST);
    if (K <= 0 || K % 8 || ldx % 8 || ldx < K) LLME_REFUSE("gemm_int4: K=%d ldx=%lld is not supported (multiples of 8, rows that do not overlap)", K, ldx);
    if (group != 32 && group != 64 && group != 128) LLME_REFUSE("gemm_int4: groups of %d values are not supported (32, 64 or 128)", group);
    if (ldw % 16 || ldw < (K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES) LLME_REFUSE("gemm_int4: rows of %lld bytes do not hold %d values in whole blocks", ldw, K);
    if (lds < (K + group - 1LL) / group) LLME_REFUSE("gemm_int4: rows of %lld scales are too short", lds);
    if (((uintptr_t)x | (uintptr_t)w) % 16) LLME_REFUSE("gemm_int4: operands must be 16-byte aligned");
    if (ldo < N) LLME_REFUSE("gemm_int4: output row stride shorter than the row");
    const long long groups = (K + group - 1LL) / group;
    if (meets(span(out, M, N, ldo, sizeof(O)), {span(x, M, K, ldx, 2), span(w, N, (K + BLOCK_K - 1LL) / BLOCK_K * BLOCK_BYTES, ldw, 1), span(scales, N, groups, lds, 2), span(zeros, N, groups, lds, 1)}))
        LLME_REFUSE("gemm_int4: the output lies over an operand");
    Args a{(const bf16*)x, ldx, (const unsigned char*)w, ldw, (const bf16*)scales, (const unsigned char*)zeros, lds, out, ldo, M, N, K, 0};
    auto aligned = [&](int count) { return lds % count == 0 && (uintptr_t)scales % (2 * count) == 0 && (uintptr_t)zeros % count == 0; };
    a.together = aligned(256 / group) ? 2 : (aligned(128 / group) ? 1 : 0);
    if (group == 32) return launch<1, O>(a, stream);
    if (group == 64) return launch<2, O>(a, stream);
    return launch<4, O>(a, stream);
}

}  // namespace

// x [M,K] bfloat16 with row stride ldx (elements, a multiple of 8; K too); w the codes [N, ceil(K / 128) * 64] with row stride ldw (bytes,
// a multiple of 16); scales [N, ceil(K / group)] bfloat16 and zeros of the same shape (values 0..15) or NULL, row stride lds; out [M,N]
// bfloat16, row stride ldo.
LLME_API int llme_gemm_int4(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, long long lds,
                            int group, void* out, long long ldo, int M, int N, int K, cudaStream_t stream) {
    return product<bf16>(x, ldx, w, ldw, scales, zeros, lds, group, out, ldo, M, N, K, stream);
}
// The same with a 32-bit out: a sum on its way into the residual stream.
LLME_API int llme_gemm_int4_f32(const void* x, long long ldx, const void* w, long long ldw, const void* scales, const void* zeros, long long lds,
                                int group, void* out, long long ldo, int M, int N, int K, cudaStream_t stream) {
    return product<float>(x, ldx, w, ldw, scales, zeros, lds, group, out, ldo, M, N, K, stream);
}

// More than 16 tokens: 0 (the default): whichever kernel should be faster; 1: single SMs, K cut over clusters; 2: pairs of SMs.  For tests and
// measurements.
LLME_API int llme_gemm_int4_form(int how) {
    if (how >= 0 && how <= 2) g_form = how;
    return g_form;
}

// 0 if no bounded wait has given up since the last call (synchronises the device).
LLME_API int llme_gemm_int4_status() { LLME_TAKE_STATUS(g_status); }
