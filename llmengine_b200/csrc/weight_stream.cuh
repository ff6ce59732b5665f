// Weights on their way from memory to a warp that multiplies them by a handful of tokens (gemm_e4m3.cu, gemm_int4.cu).
//
// A warp owns 16 weight rows and walks over them in pieces of 128 bytes a row; lane (r, quad) = (lane / 4, lane % 4) needs of every piece the
// 16 bytes at quad * 16 and at 64 + quad * 16 of rows r and r + 8.  The pieces of the next steps lie in a ring in shared memory, brought by
// asynchronous copies: every lane copies what it will read itself, so nothing has to be shared and no barrier is met, and how much is under
// way does not cost registers.  (24576 x 4096 in 4 bits, one token: 13.6 us, the loads alone 10.1; with the pieces in registers a warp's loads and
// its arithmetic took turns, 18.1 us.  A ring of three, four or six steps gains nothing.)
// Where the row groups alone do not fill the GPU, several warps share a group: warp p of n takes the pieces p, p + n, ..., and their sums are
// added in the order of the warps.  How many share follows from the weights' shape alone, so a token's result does not depend on the others.
// A block is one group: blocks of several came out less even over the SMs.
#pragma once

namespace stream {

constexpr int PIECE = 128, DEPTH = 2, RING = DEPTH * 16 * PIECE;      // bytes of a row in a step; steps in the ring; bytes of a warp's ring

struct Ring {
    unsigned at;                                  // this lane's place in its warp's ring (shared-memory address)
    __device__ __forceinline__ explicit Ring(unsigned char* rings) {
        at = (unsigned)__cvta_generic_to_shared(rings) + (threadIdx.x >> 5) * RING + (threadIdx.x & 31) * 16;
    }
    // The copies of a step's piece, 16 bytes each where `half0` / `half1` say that the row goes on so far.
    __device__ __forceinline__ void bring(int slot, const unsigned char* row0, const unsigned char* row1, bool half0, bool half1) const {
        const unsigned to = at + slot * (16 * PIECE);
        if (half0) { copy(to, row0); copy(to + 512, row1); }
        if (half1) { copy(to + 1024, row0 + 64); copy(to + 1536, row1 + 64); }
    }
    static __device__ __forceinline__ void copy(unsigned to, const unsigned char* from) {
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    }
    static __device__ __forceinline__ void close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // the copies of all steps but the last DEPTH - 1 that were closed have landed
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory"); }
    __device__ __forceinline__ uint4 read(int slot, int half, int row) const {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at + slot * (16 * PIECE) + half * 1024 + row * 512) : "memory");
        return v;
    }
};

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// How many warps share a row group, and how many warps an SM should hold.  Few groups: many warps each; many groups: few warps each, so that the
// last blocks to run are short (1,536 groups of 4,096 4-bit values, one token: 14.1 us with two warps, 15.3 with four, 15.4 with eight).  Of the
// warps an SM may hold those that leave the last round of blocks fullest, and the fewest of these: the others' room is registers (4-bit values in
// groups of 32 with zero points, eight tokens: 448 groups of 5,120 9.8 us with room for four blocks of four warps, 12.6 for five, 14.9 for six; 864
// groups of 5,120 17.9, 23.7 and 16.5; 2,000 groups of 4,096, two warps each, 27.3 us with room for eight blocks, 37.6 for ten, 44.7 for twelve.  256
// groups of 12,288, groups of 128, one token: 9.4 us with room for two blocks of eight warps, 10.8 for three).
struct Shares { int warps, an_sm; };
inline Shares sharing(int groups, int pieces, int sms) {
    const int each = (groups + sms - 1) / sms;              // blocks that an SM should hold
    if (each <= 1 && pieces >= 16) return {16, 16};
    if (each <= 3) return {8, each <= 2 ? 16 : 24};
    Shares by{each <= 6 ? 4 : 2, 0};
    double fullest = 0.0;
    for (int an_sm = 16; an_sm <= 24; an_sm += 4) {
        const long long held = (long long)an_sm / by.warps * sms, rounds = (groups + held - 1) / held;
        const double full = (double)groups / (double)(rounds * held);
        if (full > fullest) { fullest = full; by.an_sm = an_sm; }
    }
    return by;
}
// launch(warps, an_sm), both as compile-time numbers
template <typename F>
int with(Shares by, F launch) {
    using std::integral_constant;
    auto held = [&](auto warps) {
        if (by.an_sm == 16) return launch(warps, integral_constant<int, 16>{});
        if (by.an_sm == 20) return launch(warps, integral_constant<int, 20>{});
        return launch(warps, integral_constant<int, 24>{});
    };
    if (by.warps == 16) return launch(integral_constant<int, 16>{}, integral_constant<int, 16>{});
    if (by.warps == 8) return by.an_sm == 16 ? launch(integral_constant<int, 8>{}, integral_constant<int, 16>{}) : launch(integral_constant<int, 8>{}, integral_constant<int, 24>{});
    return by.warps == 4 ? held(integral_constant<int, 4>{}) : held(integral_constant<int, 2>{});
}

}  // namespace stream
