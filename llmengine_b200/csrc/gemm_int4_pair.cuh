// The product with 4-bit weights for many tokens on pairs of SMs: tiles of 256 weight rows x NT tokens, tcgen05.mma.cta_group::2.
// Included by gemm_int4.cu inside its unnamed namespace, behind umma.cuh and gemm_wide.cuh.
//
// What bounds the product on single SMs (gemm_wide.cuh) at many tokens is what a block brings from L2, 57 KB a step at 192 tokens against 768 cycles
// of instructions.  Of a pair each block brings its own 128 weight rows and HALF of the tokens' rows: 32 KB.
//
// Persistent: every pair (a cluster of two) walks over the tiles.  In each block
//   * one warp brings, 128 values of K at a time, the codes (counted on the block's own barrier) and the block's half of the tokens' rows
//     (counted on the first block's barrier);
//   * twelve warps, in three sets that take the steps in turn, make bfloat16 numbers s (c - z) of the codes, a weight row a lane, in the block's
//     tensor memory, and say so to the first block, where one warp issues the instructions for both (256 x NT x 16).  (A set needs 2,100
//     cycles from step to step, a third of them waits and messages: two sets were slower than the instructions, which take 768 at 192 tokens);
//   * four warps read the block's half of the accumulator, which is double-buffered, and store it, a token's 32 neighbouring values at a time
//     (1999 x 8192 x 256, little else: 17 us; through shared memory and TMA 25).
// 1900 x 7168 x 5120 takes 92 to 94 us (1.5 PFLOP/s) at 1.53 GHz, to which the power limit brings the clock within one launch, the tensor pipe busy for
// 88 % of the cycles in which its SM works and 77 % of all (280 tiles, 74 pairs); after a second of it, at 1.37 GHz, 114.  In groups of 32 with zero
// points 108 and 130.
// The accumulators take 2 NT columns of tensor memory and the weights the rest, 64 columns a step: NT is at most 192.
// All waits are bounded (umma.cuh).
#pragma once

namespace pair {

using wide::elect_one;
constexpr int STEP = wide::STEP, MOST_STAGES = 6, MOST_NT = 192, SETS = 3, WORKERS = 4 * SETS, PRODUCER = WORKERS, ISSUER = WORKERS + 1, FIRST_OUT = WORKERS + 2, OUT_WARPS = 4;
constexpr int BLOCK = (FIRST_OUT + OUT_WARPS) * 32, W_BYTES = BM * STEP / 2, TILE_N = 2 * BM;
constexpr unsigned TMEM = 512;

struct PairArgs {
    void* out; long long ldo;
    int M, N, K, nt, stages, w_stages;
    const bf16* scales; const unsigned char* zeros; long long lds;
};

struct Barriers {
    unsigned long long w_full[MOST_STAGES], x_full[MOST_STAGES], done[MOST_STAGES];     // x_full: the first block's, for both halves
    unsigned long long ready[MOST_STAGES], acc_full[2], acc_empty[2];                   // ready and acc_empty: the first block's, for both
    unsigned tmem_base;
    int abort_flag;
};

// A step's eight instructions, 16 values each: the weights' columns follow one another, the tokens' tile has 32 bytes more each, and its second
// half, 64 values on, is a tile of its own.  In one piece, so that little stands between them: the warp that issues shares its scheduler with
// four others, and a step is 768 cycles.
__device__ __forceinline__ void mma_step(unsigned d, unsigned w, unsigned long long x0, unsigned long long x1, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 q, %4, %4;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %4, p;\n\t"
        "add.u32 a, %1, 8;\n\tadd.u64 b, %2, 2;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t"
        "add.u32 a, %1, 16;\n\tadd.u64 b, %2, 4;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t"
        "add.u32 a, %1, 24;\n\tadd.u64 b, %2, 6;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t"
        "add.u32 a, %1, 32;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], %3, %4, q;\n\t"
        "add.u32 a, %1, 40;\n\tadd.u64 b, %3, 2;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t"
        "add.u32 a, %1, 48;\n\tadd.u64 b, %3, 4;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t"
        "add.u32 a, %1, 56;\n\tadd.u64 b, %3, 6;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], [a], b, %4, q;\n\t}"
        ::"r"(d), "r"(w), "l"(x0), "l"(x1), "r"(idesc), "r"(accumulate) : "memory");
}

// O: the output's type, float or bfloat16
template <int RUNS, bool ZEROS, typename O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(BLOCK, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const PairArgs g) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nt = g.nt, x_bytes = nt / 2 * STEP * 2, stages = g.stages;              // the block's half of the tokens' rows of a step
    unsigned char* w_tiles = smem;
    unsigned char* x_tiles = smem + stages * W_BYTES;
    Barriers* bar = reinterpret_cast<Barriers*>(x_tiles + stages * x_bytes);
    volatile int* abort_flag = &bar->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
    const unsigned rank = cluster_rank();                                             // 0: the block that issues the pair's instructions
    const int steps = (g.K + STEP - 1) / STEP, m_tiles = (g.M + nt - 1) / nt, n_tiles = (g.N + TILE_N - 1) / TILE_N;
    const int tiles = m_tiles * n_tiles;                                              // (16,384 outputs each at least: fewer than 2^31 in any memory)
    const int walker = (int)(blockIdx.x >> 1), walkers = (int)(gridDim.x >> 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&bar->w_full[s], 1);
            mbar_init(&bar->x_full[s], 1);
            mbar_init(&bar->done[s], 1);
        }
        for (int s = 0; s < g.w_stages; ++s) mbar_init(&bar->ready[s], 8);            // four warps of a set of both blocks
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar->acc_full[b], 1);
            mbar_init(&bar->acc_empty[b], 2 * OUT_WARPS);
        }
        bar->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync();                                                                   // the partner's barriers are there before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bar->tmem_base, tmem_w = tmem + (unsigned)(2 * nt);         // two accumulators, then 64 columns of weights a step
    pdl_wait();

    if (warp == PRODUCER) {
        wide::Ring at(stages);
        unsigned it = 0;
        bool ok = true;
        for (int t = walker; t < tiles && ok; t += walkers) {
            const int m0 = t % m_tiles * nt + (int)rank * (nt / 2), n0 = t / m_tiles * TILE_N + (int)rank * BM;
            for (int c = 0; c < steps; ++c, ++it, at.next()) {
                const int s = at.stage;
                ok = mbar_wait(&bar->done[s], at.phase ^ 1, abort_flag, 21) && !*abort_flag;
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&bar->w_full[s], W_BYTES);
                    tma_load_2d(w_tiles + s * W_BYTES, &map_w, c * (STEP / 2), n0, &bar->w_full[s]);
                    const unsigned full = map_to_cta(smem_u32(&bar->x_full[s]), 0);
                    if (rank == 0) mbar_expect_tx(&bar->x_full[s], 2 * x_bytes);
                    tma_load_2d_pair(x_tiles + s * x_bytes, &map_x, c * STEP, m0, full);
                    tma_load_2d_pair(x_tiles + s * x_bytes + x_bytes / 2, &map_x, c * STEP + 64, m0, full);
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // gave up somewhere: let the copies that may still be in flight land before the block exits (the codes' barrier is the block's
            // own; what the tokens' rows are counted on may be the partner's: far longer than a copy takes)
            for (unsigned j = it > (unsigned)stages ? it - stages : 0; j < it; ++j)
                for (unsigned i = 0; i < WAIT_LIMIT && !mbar_try_wait(&bar->w_full[j % stages], (j / stages) & 1); ++i) {}
            for (int i = 0; i < 200; ++i) __nanosleep(5000);
        }
    } else if (warp == ISSUER) {
        if (rank == 0) {
            const unsigned id = umma_idesc(TILE_N, nt);
            wide::Ring at(stages), made(g.w_stages);
            bool ok = true;
            int i = 0;
            for (int t = walker; t < tiles && ok; t += walkers, ++i) {
                const int b = i & 1;
                ok = mbar_wait(&bar->acc_empty[b], ((i >> 1) & 1) ^ 1, abort_flag, 24);      // this accumulator has been read
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned d = tmem + (unsigned)(b * nt);
                for (int c = 0; c < steps; ++c, at.next(), made.next()) {
                    ok = mbar_wait(&bar->ready[made.stage], made.phase, abort_flag, 23);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
                        const unsigned long long x = umma_desc(x_tiles + at.stage * x_bytes);
                        mma_step(d, tmem_w + (unsigned)(made.stage * 64), x, x + (unsigned)(x_bytes / 2 >> 4), id, c > 0);
                        umma_commit_pair(&bar->done[at.stage]);                       // the stage, and the weights made of it, are free in both blocks
                        if (c == steps - 1) umma_commit_pair(&bar->acc_full[b]);
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp < WORKERS) {
        // ------------------------------------------------------------------ codes to numbers: a lane has a weight row
        const int set = warp >> 2, row = quarter * 32 + lane, groups = (g.K + 32 * RUNS - 1) / (32 * RUNS);
        const unsigned mine = tmem_w + ((unsigned)(quarter * 32) << 16), ready_first = map_to_cta(smem_u32(&bar->ready[0]), 0);
        // step `it` of the walk, counted over all tiles, lies in stage it % stages and leaves its weights in place it % w_stages, where those of
        // step it - w_stages lay: its instructions must be done, which is said where their stage is given back
        int stage = set, place = set % g.w_stages;
        unsigned phase = 0;
        bool ok = true, first = set < g.w_stages;                                     // (first: nothing lay in the place before)
        auto next = [&] {
            first = first && place + SETS < g.w_stages;
            stage += SETS;
            if (stage >= stages) { stage -= stages; phase ^= 1; }
            place = (place + SETS) % g.w_stages;
        };
        // the set's next step is step c of tile t: its scales are on their way before the step's codes are looked at, over the end of a tile too
        int c = set, t = walker;
        const bf16* scales = nullptr;
        const unsigned char* zeros = nullptr;
        auto locate = [&] {
            for (; c >= steps; c -= steps) t += walkers;
            const long long weight_row = min(t / m_tiles * TILE_N + (int)rank * BM + row, g.N - 1);
            scales = g.scales + weight_row * g.lds;
            if (ZEROS) zeros = g.zeros + weight_row * g.lds;
        };
        locate();
        wide::Group<RUNS, ZEROS> ahead;
        if (t < tiles) ahead.fetch(scales, zeros, c, groups);
        while (t < tiles) {
            const int s = stage;
            const wide::Group<RUNS, ZEROS> now = ahead;
            c += SETS;
            if (c >= steps) locate();
            if (t < tiles) ahead.fetch(scales, zeros, c, groups);
            ok = mbar_wait(&bar->w_full[s], phase, abort_flag, 25);
            if (!ok) break;
            // unit q holds word 4 q + j; the 64-byte swizzle put it at q ^ (row / 2 % 4), so that eight lanes meet no bank twice
            const unsigned char* src = w_tiles + s * W_BYTES + row * 64;
            unsigned words[4][4], v[4][16];
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(words[q]) = *reinterpret_cast<const uint4*>(src + ((q ^ ((row >> 1) & 3)) << 4));
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) now.numbers(words[q][j], j / RUNS, v[j] + q * 4);
            // (the numbers wait in registers for their place, of which there are few: from one step's end to the next one's beginning in a
            // place only the way into tensor memory and the messages take time)
            if (!first) {
                const int before = stage - g.w_stages;
                ok = mbar_wait(&bar->done[before < 0 ? before + stages : before], before < 0 ? phase ^ 1 : phase, abort_flag, 26);
            }
            // (one warp also sees that the tokens' rows are there, for the warp that issues: a wait takes that one some 300 cycles of a step)
            if (ok && rank == 0 && quarter == 0) ok = mbar_wait(&bar->x_full[s], phase, abort_flag, 22);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j) wide::tmem_store16(mine + (unsigned)(place * 64 + j * 16), v[j]);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) wide::mbar_arrive_remote(ready_first + (unsigned)(place * 8));
            next();
        }
    } else {
        // ------------------------------------------------------------------ the way out: a warp for every 32 weight rows
        const unsigned acc_empty_first = map_to_cta(smem_u32(&bar->acc_empty[0]), 0);
        int i = 0;
        for (int t = walker; t < tiles; t += walkers, ++i) {
            const int m0 = t % m_tiles * nt, n = t / m_tiles * TILE_N + (int)rank * BM + quarter * 32 + lane, b = i & 1;
            if (!mbar_wait(&bar->acc_full[b], (i >> 1) & 1, abort_flag, 27)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned mine = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)(b * nt);
            // 32 tokens' values of this lane's weight row (all of them wherever there are so many: a test at every store took twice as long)
            auto put = [&](const unsigned (&v)[32], int j) {
                if (n >= g.N) return;
                const int left = g.M - m0 - j;
                O* to = reinterpret_cast<O*>(g.out) + (long long)(m0 + j) * g.ldo + n;
                if (left >= 32) {
#pragma unroll
                    for (int e = 0; e < 32; ++e, to += g.ldo) *to = from_f32<O>(__uint_as_float(v[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e, to += g.ldo)
                        if (e < left) *to = from_f32<O>(__uint_as_float(v[e]));
                }
            };
            // the next values are on their way out of tensor memory while these are stored; behind the last the accumulator may be filled again
            auto next = [&](unsigned (&v)[32], int j) {
                __syncwarp();
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (j < nt) tmem_ld_32x32(mine + (unsigned)j, v);
                else {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) wide::mbar_arrive_remote(acc_empty_first + (unsigned)(b * 8));
                }
            };
            unsigned v0[32], v1[32];
            tmem_ld_32x32(mine, v0);
            for (int j = 0; j < nt; j += 64) {
                next(v1, j + 32);
                put(v0, j);
                if (j + 32 >= nt) break;
                next(v0, j + 64);
                put(v1, j + 32);
            }
        }
    }
    __syncwarp();
    pdl_launch_dependents();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // a pair leaves together: no instruction of the first block still reads the second's memory, and no arrive is on its way to a block that has gone
    cluster_sync();
    if (warp == ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM));
    }
}

inline size_t smem_of(int nt, int stages) { return 1024 + (size_t)stages * (W_BYTES + (size_t)nt / 2 * STEP * 2) + sizeof(Barriers); }

template <int RUNS, bool ZEROS, typename O>
int grant() {
    static LlmeGrants grants;
    if (cudaError_t e = llme_grant_smem(grants, pair_kernel<RUNS, ZEROS, O>, wide::MOST_SMEM)) LLME_REFUSE("gemm_int4: cannot reserve %zu bytes of shared memory: %s", wide::MOST_SMEM, cudaGetErrorString(e));
    return 0;
}

// How many pairs the GPU holds at once, of whichever output type (asked of bfloat16's kernel): the two blocks of a pair need two free SMs of one GPC.
template <int RUNS, bool ZEROS>
int pairs_held() {
    static std::atomic<int> known{0};
    int n = known.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * 1024, 1, 1);
    cfg.blockDim = dim3(BLOCK);
    cfg.dynamicSmemBytes = wide::MOST_SMEM;
    if (cudaOccupancyMaxActiveClusters(&n, pair_kernel<RUNS, ZEROS, bf16>, &cfg) != cudaSuccess || n <= 0 || n > sm_count() / 2) {
        cudaGetLastError();
        n = sm_count() / 2;
    }
    known.store(n, std::memory_order_relaxed);
    return n;
}

// The tile width that takes the fewest cycles (as in wide::shape(): microseconds times 1,870), and how many: a step takes 780 and one for every token of the tile (1900 x 7168 x 5120, tiles of 64 /
// 128 / 160 / 192: 226 / 124 / 113 / 92 us), the way from one tile to the next 1,500; all tiles but the last take 4,000 and three for every token at
// least, which the way out of the one before takes (768 / 1600 x 24576 x 256: 17.8 / 32.7 us); starting takes 3,300, the last one's way out 23 for
// every token.
template <int RUNS, bool ZEROS>
int shape(PairArgs& g, double* cycles) {
    if (int rc = grant<RUNS, ZEROS, bf16>()) return rc;
    const int held = pairs_held<RUNS, ZEROS>(), n_tiles = (g.N + TILE_N - 1) / TILE_N;
    *cycles = -1.0;
    for (int nt = 64; nt <= MOST_NT; nt += 32) {
        const long long tiles = (long long)n_tiles * ((g.M + nt - 1) / nt);
        const double tile = ((g.K + STEP - 1) / STEP) * (780.0 + nt) + 1500.0, out = 4000.0 + 3.0 * nt;
        const double cost = (double)((tiles + held - 1) / held - 1) * (tile > out ? tile : out) + tile + 3300.0 + 23.0 * nt;
        if (*cycles < 0.0 || cost < *cycles) { *cycles = cost; g.nt = nt; }
    }
    g.w_stages = (512 - 2 * g.nt) / 64 < MOST_STAGES ? (512 - 2 * g.nt) / 64 : MOST_STAGES;
    g.stages = MOST_STAGES;
    while (smem_of(g.nt, g.stages) > wide::MOST_SMEM) --g.stages;
    if (g.w_stages > g.stages) g.w_stages = g.stages;
    return 0;
}

template <int RUNS, bool ZEROS, typename O>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, const PairArgs& g, cudaStream_t s) {
    if (int rc = grant<RUNS, ZEROS, O>()) return rc;
    const long long tiles = (long long)((g.M + g.nt - 1) / g.nt) * ((g.N + TILE_N - 1) / TILE_N);
    const int held = pairs_held<RUNS, ZEROS>();
    llme_launch(pair_kernel<RUNS, ZEROS, O>, dim3((unsigned)(tiles < held ? tiles : held) * 2), dim3(BLOCK), smem_of(g.nt, g.stages), s, mw, mx, g);
    LLME_LAUNCH_STATUS();
}

}  // namespace pair
