// Products with weights of 8 or 4 bits on the fifth-generation tensor cores, the weights on the lanes of tensor memory: a block takes 128
// weight rows and NT tokens, so a tile is as narrow as the tokens are few, and the segments of K are a cluster's blocks, so that few
// tiles still fill the SMs.  Included by gemm_e4m3.cu and gemm_int4.cu inside their unnamed namespaces, behind umma.cuh.
//
//   * one warp brings, 128 values of K at a time, the weights and the tokens' rows into shared memory (TMA);
//   * 4-bit weights: eight warps, in two sets that take the steps in turn, make bfloat16 numbers s (c - z) of the codes, a weight row a
//     lane, and leave them in TENSOR memory, from where the instructions take their first operand.  c - z is exact; its product with
//     the scale is rounded to bfloat16 once, half a step of 2^-8 at most, as a model with bfloat16 weights would hold it;
//   * one warp issues the instructions (128 x NT x 16 bfloat16, 128 x NT x 32 e4m3) into one accumulator in tensor memory;
//   * at the end eight warps read the accumulator.  One segment: they store it.  Several: each block leaves its sums in shared memory and
//     adds a share of the outputs over the cluster's blocks in their order.
// Bound by the weights' way from memory where the tokens are few, by what a block brings from L2 and, with 4 bits, by the making of numbers where
// they are more: 77 x 4096 x 12288 in 8 bits 14.6 us (3.6 TB/s), 40 / 200 x 7168 x 5120 in 8 bits 11.3 / 15.4 us, in 4 bits 14.1 / 22.3.
// All waits are bounded (umma.cuh).
#pragma once

namespace wide {

constexpr int STEP = 128;                        // values of K a stage holds
constexpr int WORKERS = 8, PRODUCER = 8, ISSUER = 9, BLOCK = (WORKERS + 2) * 32, MOST_STAGES = 8, MOST_SEGMENTS = 8;
constexpr size_t MOST_SMEM = 232448, HALF_SMEM = 115712;      // of a block that has an SM to itself; of one of two (1 KB each is the system's)

struct Args {
    void* out; long long ldo; int out_f32;
    int M, N, K, nt, segments, segment_steps, stages, d_cols, tmem_cols, per_sm, vec_out;
    const float* xs; const float* ws;                                                      // 8 bits
    const bf16* scales; const unsigned char* zeros; long long lds;                         // 4 bits
};

struct Barriers {
    unsigned long long full[MOST_STAGES], ready[MOST_STAGES], done[MOST_STAGES], acc;
    unsigned tmem_base;
    int abort_flag;
};

// A stage and how often the ring has come round (a division by the number of stages takes longer than much of a step).
struct Ring {
    int stages, stage = 0;
    unsigned phase = 0;
    __device__ __forceinline__ explicit Ring(int n) : stages(n) {}
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; phase ^= 1; }
    }
};

__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_e4m3_tile(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_from_tmem(unsigned d, unsigned a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// kind::f8f6f4: D = F32, A = B = E4M3 (type 0), both K-major
__device__ constexpr unsigned idesc_e4m3(int M, int N) { return (1u << 4) | ((unsigned)(N >> 3) << 17) | ((unsigned)(M >> 4) << 24); }

__device__ __forceinline__ void tmem_store16(unsigned addr, const unsigned (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}
__device__ __forceinline__ void tmem_load8(unsigned addr, unsigned (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(addr));
}
// An arrival at another block's barrier (`bar`: an address in the cluster's shared window) that passes on nothing but tensor memory, which
// tcgen05.wait and tcgen05.fence order: released to the cluster (mbar_arrive_cluster) it would wait for all of the thread's loads and stores
// first, some 1,500 cycles.
__device__ __forceinline__ void mbar_arrive_remote(unsigned bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// A request to bring a box into L2: it holds nothing back and may come ahead of what is written there.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
// Eight tokens' values of a weight row, of which `left` are there.
template <typename O>
__device__ __forceinline__ void store8(O* to, long long ldo, int left, const float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e, to += ldo)
        if (e < left) *to = from_f32<O>(f[e]);
}
__device__ __forceinline__ void store_value(const Args& g, long long m, int n, float v) {
    if (g.out_f32) reinterpret_cast<float*>(g.out)[m * g.ldo + n] = v;
    else reinterpret_cast<bf16*>(g.out)[m * g.ldo + n] = __float2bfloat16_rn(v);
}

// What the lanes of a warp set make of a weight row's 128 codes: RUNS runs of 32 values share a scale.
template <int RUNS, bool ZEROS>
struct Group {
    static constexpr int COUNT = 4 / RUNS;
    __nv_bfloat162 scale[COUNT], bias[COUNT];
    // the scales of step `step` of K; behind the last group there is nothing but zeros to multiply
    __device__ __forceinline__ void fetch(const bf16* scales, const unsigned char* zeros, int step, int groups) {
#pragma unroll
        for (int g = 0; g < COUNT; ++g) {
            const int at = step * COUNT + g;
            scale[g] = at < groups ? __bfloat162bfloat162(scales[at]) : __floats2bfloat162_rn(0.0f, 0.0f);
            const unsigned z = ZEROS ? (at < groups ? zeros[at] : 0u) : 8u, b = 0x43004300u | z | z << 16;
            bias[g] = *reinterpret_cast<const __nv_bfloat162*>(&b);
        }
    }
    // a word's eight numbers, in order, of its group g
    __device__ __forceinline__ void numbers(unsigned word, int g, unsigned* v) const {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const unsigned code = ((word >> (4 * p)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 w = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&code), bias[g]), scale[g]);
            v[p] = *reinterpret_cast<const unsigned*>(&w);
        }
    }
};

// INT4: bfloat16 tokens and 4-bit weights; else both e4m3.
template <bool INT4, int RUNS, bool ZEROS>
__global__ void __launch_bounds__(BLOCK, 2)
wide_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Args g) {
    constexpr int W_BYTES = INT4 ? BM * STEP / 2 : BM * STEP;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int nt = g.nt, x_bytes = nt * STEP * (INT4 ? 2 : 1), stages = g.stages;
    unsigned char* w_tiles = smem;                                 // stages x the weights of a step; the sums at the end
    unsigned char* x_tiles = smem + stages * W_BYTES;
    Barriers* bar = reinterpret_cast<Barriers*>(x_tiles + stages * x_bytes);
    volatile int* abort_flag = &bar->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3, rank = (int)blockIdx.z;
    // (the tiles of the same weight rows follow one another)
    const int m_tiles = (g.M + nt - 1) / nt, m0 = (int)(blockIdx.x % (unsigned)m_tiles) * nt, n0 = (int)(blockIdx.x / (unsigned)m_tiles) * BM;
    const int step0 = rank * g.segment_steps, steps = min(g.segment_steps, (g.K + STEP - 1) / STEP - step0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&bar->full[s], 1);
            mbar_init(&bar->ready[s], 5);                          // four warps of a set, and the copy of the tokens' rows
            mbar_init(&bar->done[s], 1);
        }
        mbar_init(&bar->acc, 1);
        bar->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == ISSUER) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar->tmem_base)), "r"(g.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bar->tmem_base, tmem_w = tmem + (unsigned)g.d_cols;        // the accumulator; 64 columns of weights a stage
    // (The kernel before may write what is taken for weights here: ahead of it goes only a request to have the first ones in L2.)
    if (warp == PRODUCER && elect_one())
        for (int c = 0; c < min(stages, steps); ++c) tma_prefetch_2d(&map_w, (step0 + c) * (INT4 ? STEP / 2 : STEP), n0);
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();        // (a block of the next kernel comes in when a block of this one has left its shared memory)

    if (warp == PRODUCER) {
        Ring at(stages);
        int c = 0;
        for (; c < steps; ++c, at.next()) {
            const int s = at.stage;
            if (!mbar_wait(&bar->done[s], at.phase ^ 1, abort_flag, 1) || *abort_flag) break;
            if (elect_one()) {
                // (4-bit weights: the tokens' bytes are counted where the numbers made of the codes are, for the instructions wait there)
                unsigned long long* x_full = INT4 ? &bar->ready[s] : &bar->full[s];
                mbar_expect_tx(&bar->full[s], INT4 ? W_BYTES : W_BYTES + x_bytes);
                tma_load_2d(w_tiles + s * W_BYTES, &map_w, (step0 + c) * (INT4 ? STEP / 2 : STEP), n0, &bar->full[s]);
                if (INT4) mbar_expect_tx(x_full, x_bytes);
                tma_load_2d(x_tiles + s * x_bytes, &map_x, (step0 + c) * STEP, m0, x_full);
                if (INT4) tma_load_2d(x_tiles + s * x_bytes + x_bytes / 2, &map_x, (step0 + c) * STEP + 64, m0, x_full);
            }
            __syncwarp();
        }
        if (c < steps) {                                           // gave up: the copies that may still be in flight land first
            for (int j = max(0, c - stages); j < c; ++j)
                for (unsigned n = 0; n < WAIT_LIMIT && !mbar_try_wait(&bar->full[j % stages], (unsigned)(j / stages) & 1); ++n) {}
            if (INT4) for (int i = 0; i < 200; ++i) __nanosleep(5000);         // (the tokens' barriers may lack an arrival: far longer than a copy takes)
        }
    } else if (warp == ISSUER) {
        const unsigned id = INT4 ? umma_idesc(BM, nt) : idesc_e4m3(BM, nt);
        Ring at(stages);
        for (int c = 0; c < steps; ++c, at.next()) {
            const int s = at.stage;
            if (!mbar_wait(INT4 ? &bar->ready[s] : &bar->full[s], at.phase, abort_flag, 2)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                const unsigned long long x = umma_desc(x_tiles + s * x_bytes);
                if (INT4) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)                     // 16 values each; the second half of the values is a tile of its own
                        mma_from_tmem(tmem, tmem_w + (unsigned)(s * 64 + k * 8), x + (unsigned)((k >> 2) * (x_bytes / 2) >> 4) + 2 * (k & 3), id, c > 0 || k > 0);
                } else {
                    const unsigned long long w = umma_desc(w_tiles + s * W_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_e4m3_tile(tmem, w + 2 * k, x + 2 * k, id, c > 0 || k > 0);
                }
                umma_commit(&bar->done[s]);
                if (c == steps - 1) umma_commit(&bar->acc);
            }
            __syncwarp();
        }
    } else if (INT4) {
        // ------------------------------------------------------------------ codes to numbers: a lane has a weight row
        const int set = warp >> 2, row = quarter * 32 + lane;
        const long long weight_row = min(n0 + row, g.N - 1);
        const bf16* scales = g.scales + weight_row * g.lds;
        const unsigned char* zeros = ZEROS ? g.zeros + weight_row * g.lds : nullptr;
        const int groups = (g.K + 32 * RUNS - 1) / (32 * RUNS);
        const unsigned mine = tmem_w + ((unsigned)(quarter * 32) << 16);
        Group<RUNS, ZEROS> next;
        next.fetch(scales, zeros, step0 + set, groups);
        Ring at(stages);
        if (set) at.next();
        for (int c = set; c < steps; c += 2, at.next(), at.next()) {
            const int s = at.stage;
            const Group<RUNS, ZEROS> now = next;
            next.fetch(scales, zeros, step0 + c + 2, groups);
            if (!mbar_wait(&bar->full[s], at.phase, abort_flag, 4)) break;
            // unit q holds word 4 q + j; the 64-byte swizzle put it at q ^ (row / 2 % 4), so that eight lanes meet no bank twice
            const unsigned char* src = w_tiles + s * W_BYTES + row * 64;
            unsigned words[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(words[q]) = *reinterpret_cast<const uint4*>(src + ((q ^ ((row >> 1) & 3)) << 4));
            // (the instructions that read these columns before are through: the copy waited for them)
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                unsigned v[16];
#pragma unroll
                for (int q = 0; q < 4; ++q) now.numbers(words[q][j], j / RUNS, v + q * 4);
                tmem_store16(mine + (unsigned)(s * 64 + j * 16), v);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar->ready[s]);
        }
    }
    __syncwarp();
    float* part = reinterpret_cast<float*>(smem);                  // [token][128 weight rows]
    if (warp < WORKERS) {
        const int row = quarter * 32 + lane, n = n0 + row, half = nt / 2, col0 = (warp >> 2) * half;
        const int first = m0 + col0, left = n < g.N ? min(half, g.M - first) : 0;       // the half's first token; how many of its values are stored
        // (the scales are there before the sums are: token 32 i + lane's, handed round below)
        const float ws = !INT4 && g.segments == 1 && n < g.N ? g.ws[n] : 1.0f;
        float xs[4];
        if (!INT4)
#pragma unroll
            for (int i = 0; i < 4; ++i) xs[i] = g.segments == 1 && 32 * i + lane < half && first + 32 * i + lane < g.M ? g.xs[first + 32 * i + lane] : 0.0f;
        const bool sum = mbar_wait(&bar->acc, 0, abort_flag, 5);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned mine = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)col0;
        auto put = [&](const unsigned (&v)[8], int j) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(v[e]);
            if (g.segments > 1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) part[(col0 + j + e) * BM + row] = f[e];
                return;
            }
            if (!INT4) {
                const float scales = j < 32 ? xs[0] : (j < 64 ? xs[1] : (j < 96 ? xs[2] : xs[3]));
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = f[e] * __shfl_sync(0xffffffffu, scales, (j & 31) + e) * ws;
            }
            if (g.out_f32) {
                store8(reinterpret_cast<float*>(g.out) + (long long)(first + j) * g.ldo + n, g.ldo, left - j, f);
            } else {
                store8(reinterpret_cast<bf16*>(g.out) + (long long)(first + j) * g.ldo + n, g.ldo, left - j, f);
            }
        };
        // the next values are on their way out of tensor memory while these are stored
        auto next = [&](unsigned (&v)[8], int j) {
            __syncwarp();
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (j < half) tmem_load8(mine + (unsigned)j, v);
        };
        if (sum) {
            unsigned v0[8], v1[8];
            tmem_load8(mine, v0);
            for (int j = 0; j < half; j += 16) {
                next(v1, j + 8);
                put(v0, j);
                if (j + 8 >= half) break;
                next(v0, j + 16);
                put(v1, j + 8);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == ISSUER) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(g.tmem_cols));
    }
    if (g.segments == 1) return;
    cluster_sync();
    // a share of the outputs over all segments in their order
    const unsigned from_here = smem_u32(smem);
    for (int e = rank * BLOCK + (int)threadIdx.x; e < nt * (BM / 4); e += g.segments * BLOCK) {
        const int m = m0 + e / (BM / 4), n = n0 + (e % (BM / 4)) * 4;
        if (m >= g.M || n >= g.N) continue;
        // (all of a place's loads are under way before the first is added: one after the other each takes some 700 cycles)
        float4 f[MOST_SEGMENTS];
#pragma unroll
        for (int from = 0; from < MOST_SEGMENTS; ++from)
            if (from < g.segments)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(f[from].x), "=f"(f[from].y), "=f"(f[from].z), "=f"(f[from].w) : "r"(map_to_cta(from_here + 16u * (unsigned)e, (unsigned)from)));
        float v[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
        for (int from = 1; from < MOST_SEGMENTS; ++from)
            if (from < g.segments) { v[0] += f[from].x; v[1] += f[from].y; v[2] += f[from].z; v[3] += f[from].w; }
        if (!INT4) {
            const float xs = g.xs[m];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < g.N) v[i] = v[i] * xs * g.ws[n + i];
        }
        if (g.vec_out && n + 4 <= g.N) {
            if (g.out_f32) {
                *reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + m * g.ldo + n) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                uint2 raw;
                *reinterpret_cast<__nv_bfloat162*>(&raw.x) = __floats2bfloat162_rn(v[0], v[1]);
                *reinterpret_cast<__nv_bfloat162*>(&raw.y) = __floats2bfloat162_rn(v[2], v[3]);
                *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(g.out) + m * g.ldo + n) = raw;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < g.N) store_value(g, m, n + i, v[i]);
        }
    }
    cluster_sync();                                                // nobody leaves while its sums are read
}

// The same as make_map() with a choice of swizzle.
int make_map_swizzled(CUtensorMap* map, const void* base, CUtensorMapDataType type, int elem_bytes, long long rows, long long cols, long long ld,
                      int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) LLME_REFUSE("gemm_wide: cuTensorMapEncodeTiled is not available in this driver");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * elem_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) LLME_REFUSE("gemm_wide: cuTensorMapEncodeTiled failed with code %d", (int)r);
    return 0;
}

// How many clusters of `segments` blocks the GPU holds at once, `per_sm` blocks an SM: a cluster's blocks need SMs of one GPC, and what is
// left of a GPC stays empty.  (Asked once for every size of cluster.)
template <bool INT4, int RUNS, bool ZEROS>
int clusters_held(int segments, int per_sm) {
    static std::atomic<int> known[2][MOST_SEGMENTS + 1];
    std::atomic<int>& one = known[per_sm - 1][segments];
    int n = one.load(std::memory_order_relaxed);
    if (n) return n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024, 1, segments);
    cfg.blockDim = dim3(BLOCK);
    cfg.dynamicSmemBytes = per_sm == 1 ? MOST_SMEM : HALF_SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = (unsigned)segments;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int all = per_sm * sm_count() / segments;
    if (segments == 1 || cudaOccupancyMaxActiveClusters(&n, wide_kernel<INT4, RUNS, ZEROS>, &cfg) != cudaSuccess || n <= 0 || n > all) {
        cudaGetLastError();
        n = all;
    }
    one.store(n, std::memory_order_relaxed);
    return n;
}

// Tile width, segments, blocks an SM and stages of a product: what a model of its time says is least, in cycles.  The blocks that run at once
// (as many as are held) share the memory's 4,000 bytes a cycle for the weights; an SM's blocks share its 60 bytes a cycle from L2 (52 beside the
// making of numbers) and its tensor core, where a step takes twice nt cycles (128 e4m3 values) or four times (bfloat16); making numbers of a step's
// codes keeps an SM busy for 850.  Starting and ending a block cost about 4,000 cycles and 22 for every token, the cluster's sums 3,000 and 10.
// All of these models count microseconds times 1,870.  (The clock is 1,965 MHz until the power limit holds it: many tokens' products run at 1.5 GHz, and
// what is 972 here, a step of 192 tokens on pairs in 4 bits, is some 780 of the SM's own cycles, its instructions' 768 and little else.)
// Over 42 products of 40 to 1,600 tokens and all of their tilings the model is off by 12 % (standard deviation), and its choice took 1 % longer than
// the best with 8 bits, 2 % with 4.  (200 x 4096 x 4096 in 8 bits, tiles of 208 tokens in four segments, 11.3 us; 96 x 7168 x 5120 in 4 bits, two
// segments, 15.6, where tiles of 48, two blocks an SM, take 31.)
// Widths: as few tiles along the tokens as a width of 256 allows, and one, two and three more, one by one; from there in steps of half of what has been
// reached, up to four times the fewest and three, for few weight rows, whose wide tiles would leave SMs idle (2048 x 264 x 1616 in 8 bits 7.2 us, with
// tiles of 192 to 256 alone 9.1).  Not every width: a call asks the model about each.
template <bool INT4, int RUNS, bool ZEROS>
int shape(Args& g, double* cycles) {
    const int steps = (g.K + STEP - 1) / STEP, n_tiles = (g.N + BM - 1) / BM, w_bytes = INT4 ? BM * STEP / 2 : BM * STEP, x_width = STEP * (INT4 ? 2 : 1);
    const int least = (g.M + 255) / 256;
    static LlmeGrants grants;
    if (cudaError_t e = llme_grant_smem(grants, wide_kernel<INT4, RUNS, ZEROS>, MOST_SMEM)) LLME_REFUSE("gemm_wide: cannot reserve %zu bytes of shared memory: %s", MOST_SMEM, cudaGetErrorString(e));
    double best = -1.0;
    for (int m_tiles = least; m_tiles <= 4 * least + 3; m_tiles += m_tiles < least + 3 ? 1 : (least + 3) / 2) {
        const int nt = ((g.M + m_tiles - 1) / m_tiles + 15) / 16 * 16;
        const long long tiles = (long long)n_tiles * ((g.M + nt - 1) / nt);
        for (int per_sm = 1; per_sm <= (nt <= 64 ? 2 : 1); ++per_sm)
            for (int segments = 1; segments <= MOST_SEGMENTS && segments <= steps && (segments == 1 || tiles < sm_count()); ++segments) {
                const int each = (steps + segments - 1) / segments;
                if ((steps + each - 1) / each != segments) continue;
                const int held = clusters_held<INT4, RUNS, ZEROS>(segments, per_sm);
                const double rounds = (double)((tiles + held - 1) / held), at_once = (double)(tiles < held ? tiles : held) * segments;
                const double share = at_once > sm_count() ? at_once / sm_count() : 1.0;                   // blocks on an SM
                double step = share * (INT4 ? 4.0 : 2.0) * nt;
                if (INT4 && step < 850.0 * (at_once > sm_count() ? 2.0 : 1.0)) step = 850.0 * (at_once > sm_count() ? 2.0 : 1.0);
                if (step < share * (w_bytes + nt * x_width) / (INT4 ? 52.0 : 60.0)) step = share * (w_bytes + nt * x_width) / (INT4 ? 52.0 : 60.0);
                if (step < at_once * w_bytes / 4000.0) step = at_once * w_bytes / 4000.0;
                const double cost = rounds * (each * step + 4000.0 + 22.0 * nt + (segments > 1 ? 3000.0 + 10.0 * nt : 0.0));
                if (best < 0.0 || cost < best) { best = cost; g.nt = nt; g.segments = segments; g.segment_steps = each; g.per_sm = per_sm; }
            }
    }
    g.d_cols = g.nt <= 64 ? 64 : (g.nt <= 128 ? 128 : 256);
    g.tmem_cols = INT4 && g.per_sm == 1 ? 512 : 256;
    const int fit = (int)(((g.per_sm == 1 ? MOST_SMEM : HALF_SMEM) - 1024 - sizeof(Barriers)) / (w_bytes + g.nt * x_width));
    g.stages = fit < MOST_STAGES ? fit : MOST_STAGES;
    if (INT4 && g.stages > (g.tmem_cols - g.d_cols) / 64) g.stages = (g.tmem_cols - g.d_cols) / 64;
    if (cycles) *cycles = best;
    return 0;
}

template <bool INT4, int RUNS, bool ZEROS>
int launch(const CUtensorMap& mw, const CUtensorMap& mx, const Args& g, cudaStream_t stream) {
    const size_t smem = 1024 + (size_t)g.stages * ((INT4 ? BM * STEP / 2 : BM * STEP) + (size_t)g.nt * STEP * (INT4 ? 2 : 1)) + sizeof(Barriers);
    auto kernel = wide_kernel<INT4, RUNS, ZEROS>;
    const long long blocks = (long long)((g.M + g.nt - 1) / g.nt) * ((g.N + BM - 1) / BM);
    if (blocks > 2147483647LL) LLME_REFUSE("gemm_wide: %d x %d outputs are too many for one launch", g.M, g.N);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks, 1, g.segments);
    cfg.blockDim = dim3(BLOCK);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = llme_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = (unsigned)g.segments;
    cfg.attrs = attr;
    cfg.numAttrs = g.segments > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, mw, mx, g);
    LLME_LAUNCH_STATUS();
}

}  // namespace wide
