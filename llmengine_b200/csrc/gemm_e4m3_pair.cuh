// The product of 8-bit rows and weights for many tokens on pairs of SMs: 256 x 256 tiles, tcgen05.mma.cta_group::2 of kind f8f6f4.
// Included by gemm_e4m3.cu inside its unnamed namespace, behind umma.cuh and gemm_wide.cuh.
//
// Persistent: every pair of blocks (a cluster of two) walks over the tiles, the tiles of the same 256 weight rows one after another.  A
// block loads its own 128 tokens' rows and half of the tile's weight rows, 128 values of K (one swizzle row) at a time, six stages deep; the
// instructions, issued by the pair's first block alone, read both blocks' shared memory and add into both blocks' tensor memory, where the
// accumulator is double-buffered.  Eight warps of each block read it back, multiply by the two scales and store through shared memory
// (TMA; value by value where the output's rows do not begin on 16 bytes): 2048 x 24576 x 128, which is little else, 29 us in bfloat16 and
// 37 in 32 bits (5.4 TB/s of output); rows of an odd length, 2048 x 10423 x 2576 in bfloat16, 58 us, straight from registers 256.  2048 x 24576 x
// 4096 takes 138 to 148 us (2.8 to 3.0 PFLOP/s) at 1.5 GHz, to which the power limit brings the clock within one launch, the tensor pipe busy for
// 91 % of the cycles in which its SM works and 82 % of all; after a second of it, at 1.15 GHz, 178.  The plumbing is that of the bfloat16 product on pairs
// (gemm_tcgen05.cu); a step moves the same bytes and does twice the work.
#pragma once

namespace pair {

constexpr int BN = 256, STAGES = 6, STEP = 128, TILE_M = 2 * BM;
constexpr int A_BYTES = BM * STEP, B_BYTES = BN / 2 * STEP, STAGING = 8 * 4096;              // what one block holds of a stage; 8 warps x (32 rows x 128 bytes)
constexpr int BLOCK = 10 * 32;
constexpr unsigned TMEM = 512;

struct Barriers {
    unsigned long long full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
    unsigned tmem_base;
    int abort_flag;
};
constexpr size_t SMEM = 1024 + (size_t)STAGES * (A_BYTES + B_BYTES) + STAGING + sizeof(Barriers);
static_assert(SMEM <= wide::MOST_SMEM, "the block's shared memory must fit an SM");

__device__ __forceinline__ void mma_pair(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

template <typename O, bool TMA_STORE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(BLOCK, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_o, const Args a) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* a_tiles = smem;
    unsigned char* b_tiles = smem + STAGES * A_BYTES;
    unsigned char* staging = b_tiles + STAGES * B_BYTES;
    Barriers* bar = reinterpret_cast<Barriers*>(staging + STAGING);
    volatile int* abort_flag = &bar->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int steps = (a.K + STEP - 1) / STEP, m_tiles = (a.M + TILE_M - 1) / TILE_M, n_tiles = (a.N + BN - 1) / BN;
    const int tiles = m_tiles * n_tiles;             // (65,536 outputs each: fewer than 2^31 in any memory)
    const unsigned rank = cluster_rank();                              // 0: the block that issues the pair's instructions
    const int walker = (int)(blockIdx.x >> 1), walkers = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bar->full[s], 1);
            mbar_init(&bar->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar->acc_full[b], 1);
            mbar_init(&bar->acc_empty[b], 16);                         // one arrival per epilogue warp of both blocks
        }
        bar->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();                                                    // the partner's barriers are initialised before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bar->tmem_base;
    pdl_wait();

    if (warp == 0) {
        // ------------------------------------------------------------------ loads
        unsigned it = 0;
        bool ok = true;
        for (int t = walker; t < tiles && ok; t += walkers) {
            const int m0 = t % m_tiles * TILE_M + (int)rank * BM, n0 = t / m_tiles * BN + (int)rank * (BN / 2);
            for (int c = 0; c < steps; ++c, ++it) {
                const unsigned s = it % STAGES;
                ok = mbar_wait(&bar->empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, 11) && !*abort_flag;
                if (!ok) break;
                if (wide::elect_one()) {
                    // both blocks' bytes are counted on the first block's barrier, which that block arms
                    const unsigned full = map_to_cta(smem_u32(&bar->full[s]), 0);
                    if (rank == 0) mbar_expect_tx(&bar->full[s], 2 * (A_BYTES + B_BYTES));
                    tma_load_2d_pair(a_tiles + s * A_BYTES, &map_x, c * STEP, m0, full);
                    tma_load_2d_pair(b_tiles + s * B_BYTES, &map_w, c * STEP, n0, full);
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // gave up somewhere: let the copies that may still be in flight land before the block exits (the second block has no
            // barrier of its own to watch: it sleeps for far longer than a copy takes)
            if (rank != 0) {
                for (int i = 0; i < 200; ++i) __nanosleep(5000);
            } else {
                for (unsigned j = it > STAGES ? it - STAGES : 0; j < it; ++j)
                    for (unsigned i = 0; i < WAIT_LIMIT && !mbar_try_wait(&bar->full[j % STAGES], (j / STAGES) & 1); ++i) {}
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ instructions
        if (rank == 0) {
            constexpr unsigned id = wide::idesc_e4m3(TILE_M, BN);
            unsigned it = 0;
            bool ok = true;
            int i = 0;
            for (int t = walker; t < tiles && ok; t += walkers, ++i) {
                const int b = i & 1;
                ok = mbar_wait(&bar->acc_empty[b], ((i >> 1) & 1) ^ 1, abort_flag, 14);      // the epilogue has drained this buffer
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned d = tmem + (unsigned)(b * BN);
                for (int c = 0; c < steps; ++c, ++it) {
                    const unsigned s = it % STAGES;
                    ok = mbar_wait(&bar->full[s], (it / STAGES) & 1, abort_flag, 12);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (wide::elect_one()) {
                        const unsigned long long da = umma_desc(a_tiles + s * A_BYTES), db = umma_desc(b_tiles + s * B_BYTES);
#pragma unroll
                        for (int k = 0; k < STEP / 32; ++k) mma_pair(d, da + 2 * k, db + 2 * k, id, c > 0 || k > 0);
                        umma_commit_pair(&bar->empty[s]);              // the stage is free in both blocks once these have read it
                        if (c == steps - 1) umma_commit_pair(&bar->acc_full[b]);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ the way out (warps 2..9: two for every 32 lanes, half of the columns each)
        const int quarter = warp & 3;             // the lanes of tensor memory this warp may read
        constexpr int PIECES = (int)sizeof(O) / 2, COLS = 32 / PIECES;             // 64-byte pieces of 32 columns; columns of a piece
        const int col0 = ((warp - 2) >> 2) * (BN / 2), swizzle = (lane >> 1) & 3;
        unsigned char* own = staging + (warp - 2) * 4096;                              // two pieces of 32 rows x 64 bytes
        const unsigned acc_empty_first = map_to_cta(smem_u32(&bar->acc_empty[0]), 0);
        int i = 0;
        for (int t = walker; t < tiles; t += walkers, ++i) {
            const int m0 = t % m_tiles * TILE_M + (int)rank * BM + quarter * 32, n0 = t / m_tiles * BN + col0, b = i & 1, row = m0 + lane;
            // (the scales are on their way while the tile is worked on: column `lane` of every 32, handed round below)
            const float xs = row < a.M ? a.xs[row] : 0.0f;
            float ws[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) ws[j] = n0 + j * 32 + lane < a.N ? a.ws[n0 + j * 32 + lane] : 0.0f;
            if (!mbar_wait(&bar->acc_full[b], (i >> 1) & 1, abort_flag, 13)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned mine = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(b * BN + col0);
            unsigned v[2][32];
            tmem_ld_32x32(mine, v[0]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned (&f)[32] = v[j & 1];
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (j < 3) tmem_ld_32x32(mine + (unsigned)(j * 32 + 32), v[(j + 1) & 1]);
                else {                                                                        // its half of the tile has left tensor memory
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) wide::mbar_arrive_remote(acc_empty_first + (unsigned)(b * 8));
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) f[e] = __float_as_uint(__uint_as_float(f[e]) * xs * __shfl_sync(0xffffffffu, ws[j], e));
#pragma unroll
                for (int h = 0; h < PIECES; ++h) {
                    unsigned char* buf = own + (j * PIECES + h & 1) * 2048;
                    if (TMA_STORE && lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");     // the store before the last has read its piece
                    __syncwarp();
                    // row `lane` of the piece; its 16-byte chunk q goes to position q ^ (lane / 2 % 4): the 64-byte swizzle
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        unsigned w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (PIECES == 2) w[e] = f[h * 16 + 4 * q + e];
                            else {
                                const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(f[(8 * q + 2 * e) & 31]), __uint_as_float(f[(8 * q + 2 * e + 1) & 31]));
                                w[e] = *reinterpret_cast<const unsigned*>(&two);
                            }
                        }
                        *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ swizzle) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    const int col = n0 + j * 32 + h * COLS;
                    if (TMA_STORE) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");          // the writes above, seen by the TMA
                        __syncwarp();
                        if (lane == 0) {
                            // rows or columns of the piece that lie outside the matrix are clipped
                            if (m0 < a.M && col < a.N) tma_store_2d(&map_o, buf, col, m0);
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    } else if (h == PIECES - 1) {
                        // an output whose rows begin anywhere: value by value, the 32 lanes along a row (all rows wherever there are so many)
                        __syncwarp();
                        const int last = a.M - m0, left = a.N - (n0 + j * 32), chunk = lane * (int)sizeof(O) % 64 / 16, byte = lane * (int)sizeof(O) % 16;
                        const unsigned char* from = (PIECES == 2 ? own + lane / 16 * 2048 : buf) + byte;
                        O* to = reinterpret_cast<O*>(a.out) + (long long)m0 * a.ldo + (n0 + j * 32 + lane);
                        if (lane < left) {
                            if (last >= 32) {
#pragma unroll
                                for (int r = 0; r < 32; ++r, to += a.ldo) *to = *reinterpret_cast<const O*>(from + r * 64 + ((chunk ^ (r >> 1 & 3)) << 4));
                            } else {
                                for (int r = 0; r < last; ++r, to += a.ldo) *to = *reinterpret_cast<const O*>(from + r * 64 + ((chunk ^ (r >> 1 & 3)) << 4));
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (TMA_STORE && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    pdl_launch_dependents();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // a pair leaves together: no instruction of the first block still reads the second's shared memory or writes its tensor memory, and no
    // arrive is on its way to a block that has gone
    cluster_sync();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM));
    }
}

template <typename O, bool TMA_STORE>
int launch_kernel(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mo, const Args& a, cudaStream_t s) {
    auto kernel = pair_kernel<O, TMA_STORE>;
    static LlmeGrants grants;
    if (cudaError_t e = llme_grant_smem(grants, kernel, SMEM)) LLME_REFUSE("gemm_e4m3: cannot reserve %zu bytes of shared memory: %s", SMEM, cudaGetErrorString(e));
    // The two blocks of a pair need two free SMs of one GPC: a GPU may hold fewer pairs than half its SMs.  A pair that had to wait for
    // another to finish would double the kernel's time, so there are never more than fit.
    static std::atomic<int> held{0};
    int walkers = held.load(std::memory_order_relaxed);
    if (!walkers) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * 1024, 1, 1);
        cfg.blockDim = dim3(BLOCK);
        cfg.dynamicSmemBytes = SMEM;
        if (cudaOccupancyMaxActiveClusters(&walkers, kernel, &cfg) != cudaSuccess || walkers <= 0 || walkers > sm_count() / 2) {
            cudaGetLastError();
            walkers = sm_count() / 2;
        }
        held.store(walkers, std::memory_order_relaxed);
    }
    const long long tiles = (long long)((a.M + TILE_M - 1) / TILE_M) * ((a.N + BN - 1) / BN);
    llme_launch(kernel, dim3((unsigned)(tiles < walkers ? tiles : walkers) * 2), dim3(BLOCK), SMEM, s, mx, mw, mo, a);
    LLME_LAUNCH_STATUS();
}

template <typename O>
int launch(const Args& a, cudaStream_t s) {
    alignas(64) CUtensorMap mx, mw, mo;
    if (int rc = make_map(&mx, a.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.M, a.K, a.ldx, BM, STEP)) return rc;
    if (int rc = make_map(&mw, a.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.N, a.K, a.ldw, BN / 2, STEP)) return rc;
    if ((uintptr_t)a.out % 16 == 0 && a.ldo * (long long)sizeof(O) % 16 == 0) {
        if (int rc = wide::make_map_swizzled(&mo, a.out, sizeof(O) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (int)sizeof(O), a.M, a.N, a.ldo,
                                             32, 64 / (int)sizeof(O), CU_TENSOR_MAP_SWIZZLE_64B)) return rc;
        return launch_kernel<O, true>(mx, mw, mo, a, s);
    }
    mo = mx;
    return launch_kernel<O, false>(mx, mw, mo, a, s);
}

}  // namespace pair
