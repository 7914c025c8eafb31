// An adapter's gradient from an input that is held in 8 bits (act8.cuh):
//
//     C[m][f] (+)= alpha * col[f] * sum_t A[t][m] * q[t][f] * 2^k(t, f / 32)
//
// A [tokens][M] BF16 (dh of the adapter, or of several that share the input), q / scale [tokens][N].  The sum runs over
// tokens, the slow axis of both operands, and the scale changes along it, so it cannot be taken out of the sum.  e4m3 is
// widened to BF16 (exact) in registers, the power of two goes to the few values of A instead (exact as well, down to BF16's
// subnormals: 2^-134 * 448 a term), and mma.sync (m16n8k16, FP32 accumulators) multiplies: columns are its rows, ranks its
// columns.  Where |A| * 2^k passes BF16's range - a product with the block's largest element then passes FP32's - the block's
// columns become infinite or NaN.
#include <cooperative_groups.h>

#include <algorithm>

#include "act8.cuh"
#include "ctx.h"

namespace ta {
namespace {

namespace cg = cooperative_groups;

// A CTA has WF warps side by side along the columns, 64 columns each, and WT along the tokens.  Its operands come through a ring
// of ST stages in shared memory filled by cp.async; a stage holds KS steps of 16 tokens for each warp.
template <int WF, int WT, int NT, int KS, int ST>
struct Tile {
    static constexpr int kThreads = 32 * WF * WT, kFeat = 64 * WF, kTokens = 16 * WT * KS, kStages = ST;
    static constexpr int kBlk = kFeat / kQ8Block;
    // a thread reads 4 bytes of tokens t, t + 4, t + 8, t + 12: rows an odd multiple of 32 bytes apart do not collide
    static constexpr int kQRow = kFeat + 32;
    static constexpr int kARow = NT * 16 + 16;                       // 16-byte chunks an odd number apart for ldmatrix
    static constexpr int kQ = kTokens * kQRow, kA = kTokens * kARow, kS = kTokens * kBlk;
    static constexpr int kStage = kQ + kA + kS;
    static constexpr int kRegions = WT > 1 ? WT / 2 : 1, kPitch = kFeat + 4;
    static constexpr int kRed = kRegions * NT * 8 * kPitch * 4;
    static constexpr int kSmem = kStages * kStage > kRed ? kStages * kStage : kRed;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t saddr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(on ? 8 : 0) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Two e4m3 values (a word's low or high half) as FP32; NaN stays NaN.
__device__ __forceinline__ float2 widen2(uint32_t w, int high) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(high ? w >> 16 : w)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// One step of 16 tokens on 64 columns: acc += A^T x.  w[b][j]: four columns of block b for the thread's j-th token, sb[b] the four
// tokens' scales, a: A's fragments.  Tokens 0, 1 of a thread are a fragment's low pair, 2, 3 its high pair.
template <int NT>
__device__ __forceinline__ void multiply(float (&acc)[4][NT][4], const uint32_t (&a)[NT / 2][4], const uint32_t (&w)[2][4], const uint32_t (&sb)[2]) {
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const uint32_t s0 = __byte_perm(sb[b], 0, 0x4140) << 7, s1 = __byte_perm(sb[b], 0, 0x4342) << 7;   // BF16's 2^k, two tokens
        uint32_t x[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float2 v0 = widen2(w[b][0], h), v1 = widen2(w[b][1], h), v2 = widen2(w[b][2], h), v3 = widen2(w[b][3], h);
            x[h][0] = pack_bf16x2(v0.x, v1.x);
            x[h][1] = pack_bf16x2(v0.y, v1.y);
            x[h][2] = pack_bf16x2(v2.x, v3.x);
            x[h][3] = pack_bf16x2(v2.y, v3.y);
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint32_t b0 = mul_bf16x2(a[n / 2][n % 2 * 2], s0), b1 = mul_bf16x2(a[n / 2][n % 2 * 2 + 1], s1);
            mma_bf16(acc[2 * b][n], x[0], b0, b1);
            mma_bf16(acc[2 * b + 1][n], x[1], b0, b1);
        }
    }
}

// The sums of the WT warps on a column, then of the cluster's CTAs, in a fixed order (the same bits every time), and the output.
// Warps from WF * WT on hold no sums.
template <int WF, int WT, int NT>
__device__ __forceinline__ void join(const float (&acc)[4][NT][4], unsigned char* smem, cg::cluster_group& cluster, int f0, int m0,
                                     const __nv_bfloat16* __restrict__ col, float* __restrict__ C, long ldc, int M, int N, float alpha, int accumulate) {
    constexpr int kFeat = 64 * WF, kPitch = kFeat + 4, kRegions = WT > 1 ? WT / 2 : 1, kThreads = 32 * WF * WT;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, wf = warp % WF, wt = warp / WF;
    const int cs = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    float* red = reinterpret_cast<float*>(smem);
    __syncthreads();
#pragma unroll
    for (int half = WT > 1 ? 1 : 0; half >= 0; half--) {
        if (wt < WT && wt / kRegions == half) {
            float* to = red + (wt % kRegions) * NT * 8 * kPitch + wf * 64 + 4 * g;
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float4* at = reinterpret_cast<float4*>(to + (n * 8 + 2 * t + e) * kPitch + 32 * b);
                        float4 sum = make_float4(acc[2 * b][n][e], acc[2 * b][n][e + 2], acc[2 * b + 1][n][e], acc[2 * b + 1][n][e + 2]);
                        if (WT > 1 && half == 0) {
                            const float4 o = *at;
                            sum.x += o.x; sum.y += o.y; sum.z += o.z; sum.w += o.w;
                        }
                        *at = sum;
                    }
        }
        __syncthreads();
    }
    if (kRegions > 1 && tid < kThreads) {
        for (int o = tid; o < NT * 8 * kFeat; o += kThreads) {
            float* at = red + o / kFeat * kPitch + o % kFeat;
            float sum = at[0];
#pragma unroll
            for (int r = 1; r < kRegions; r++) sum += at[r * NT * 8 * kPitch];
            at[0] = sum;
        }
    }
    cluster.sync();
    if (tid < kThreads) {
        for (int o = rank * kThreads + tid; o < NT * 8 * kFeat; o += cs * kThreads) {
            const int m = o / kFeat, c = o % kFeat;
            if (m0 + m >= M || f0 + c >= N) continue;
            float sum = 0.f;
            for (int r = 0; r < cs; r++) sum += cluster.map_shared_rank(red, r)[m * kPitch + c];
            sum *= alpha;
            if (col) sum *= __bfloat162float(col[f0 + c]);
            float* out = C + size_t(m0 + m) * ldc + f0 + c;
            *out = accumulate ? *out + sum : sum;
        }
    }
    cluster.sync();   // nobody leaves while its sums are read
}

template <int WF, int WT, int NT, int KS, int ST>
__global__ void __launch_bounds__(32 * WF * WT) gemm_tokens_q8_any_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                                      const __nv_bfloat16* __restrict__ A, long lda,
                                                                      const __nv_bfloat16* __restrict__ col, float* __restrict__ C, long ldc,
                                                                      int M, int N, int K, float alpha, int accumulate) {
    using T = Tile<WF, WT, NT, KS, ST>;
    constexpr int kThreads = T::kThreads;
    extern __shared__ __align__(128) unsigned char smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int wf = warp % WF, wt = warp / WF;
    const int f0 = int(blockIdx.x) / cs * T::kFeat, m0 = int(blockIdx.y) * NT * 8;
    const int nblk = (N + kQ8Block - 1) / kQ8Block;
    const int chunks = (K + T::kTokens - 1) / T::kTokens;
    const int mine = chunks > rank ? (chunks - rank + cs - 1) / cs : 0;   // chunks rank, rank + cs, ...
    const uint32_t base = smem_u32(smem);

    // A thread's copies of a stage of q lie in one column group, kRowStep rows apart.
    const bool wide = N % 16 == 0;
    const int per = wide ? 16 : 8, lanes = T::kFeat / per;
    const int q_row = tid / lanes, q_col = tid % lanes * per, row_step = kThreads / lanes;
    const bool q_on = f0 + q_col < N;
    const uint8_t* q_src = q + size_t(q_row) * N + f0 + q_col;
    const uint32_t q_dst = uint32_t(q_row * T::kQRow + q_col);

    constexpr int kScales = T::kS / kThreads;     // scale bytes a thread brings into a stage
    static_assert(T::kS % kThreads == 0 && kThreads % T::kBlk == 0, "");
    const int s_blk = tid % T::kBlk;
    const bool s_on = f0 / kQ8Block + s_blk < nblk;
    const uint8_t* s_src = scale + size_t(tid / T::kBlk) * nblk + f0 / kQ8Block + s_blk;
    uint8_t held[kScales];
    // Issues the copies of the CTA's i-th chunk into stage i % kStages; its scales go to registers (too small and unaligned for
    // cp.async) and from there to shared memory one stage later.
    auto fetch = [&](int i) {
        if (i < mine) {
            const int tok0 = (i * cs + rank) * T::kTokens;
            const uint32_t st = base + (i % T::kStages) * T::kStage;
            const uint8_t* src = q_src + size_t(tok0) * N;
            if (wide) {
#pragma unroll
                for (int j = 0; j < T::kTokens * T::kFeat / 16 / kThreads; j++) {
                    const int r = j * (kThreads / (T::kFeat / 16));
                    const bool on = q_on && tok0 + q_row + r < K;
                    cp_async16(st + q_dst + r * T::kQRow, on ? src + size_t(r) * N : q, on);
                }
            } else {
                for (int j = 0; j < T::kTokens * T::kFeat / 8 / kThreads; j++) {
                    const int r = j * row_step;
                    const bool on = q_on && tok0 + q_row + r < K;
                    cp_async8(st + q_dst + r * T::kQRow, on ? src + size_t(r) * N : q, on);
                }
            }
#pragma unroll
            for (int c = tid; c < T::kTokens * NT; c += kThreads) {
                const int tok = c / NT, m = m0 + c % NT * 8;
                const bool on = tok0 + tok < K && m < M;
                cp_async16(st + T::kQ + tok * T::kARow + c % NT * 16, on ? A + size_t(tok0 + tok) * lda + m : A, on);
            }
#pragma unroll
            for (int c = 0; c < kScales; c++) {
                constexpr int kStep = kThreads / T::kBlk;
                const bool on = s_on && tok0 + tid / T::kBlk + c * kStep < K;
                held[c] = on ? s_src[size_t(tok0 + c * kStep) * nblk] : uint8_t(127);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Scale bytes of a step of 16 tokens lie as [block][t][i] for token t + 4 i: a thread's four in one word.
    auto put_scales = [&](int i) {
        if (i >= mine) return;
        unsigned char* st = smem + (i % T::kStages) * T::kStage + T::kQ + T::kA;
#pragma unroll
        for (int c = 0; c < kScales; c++) {
            const int tok = tid / T::kBlk + c * (kThreads / T::kBlk);
            st[(tok / 16 * T::kBlk + s_blk) * 16 + (tok & 3) * 4 + (tok >> 2 & 3)] = held[c];
        }
    };

    float acc[4][NT][4] = {};
#pragma unroll
    for (int i = 0; i < T::kStages - 1; i++) {
        fetch(i);
        put_scales(i);
    }
    // the token that row k of a fragment stands for: pairs (2t, 2t+1) are t, t + 4 and (2t+8, 2t+9) are t + 8, t + 12
    const int frag_tok = ((lane & 7) >> 1) + (lane & 1) * 4 + (lane >> 3 & 1) * 8;
    for (int i = 0; i < mine; i++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(T::kStages - 2) : "memory");
        __syncthreads();                       // stage i is there; stage i - 1 is read by nobody
        fetch(i + T::kStages - 1);
        const uint32_t st = base + (i % T::kStages) * T::kStage;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const int tok = (wt * KS + k) * 16;
            const uint32_t at = st + (tok + t) * T::kQRow + wf * 64 + g * 4;
            const uint32_t sat = st + T::kQ + T::kA + (tok / 16 * T::kBlk + wf * 2) * 16 + t * 4;
            const uint32_t rows = st + T::kQ + (tok + frag_tok) * T::kARow + (lane >> 4) * 16;
            uint32_t a[NT / 2][4], w[2][4], sb[2];
#pragma unroll
            for (int n = 0; n < NT / 2; n++) ldmatrix_x4_trans(a[n], rows + n * 32);
#pragma unroll
            for (int b = 0; b < 2; b++) {
#pragma unroll
                for (int j = 0; j < 4; j++) w[b][j] = lds32(at + 4 * j * T::kQRow + b * 32);
                sb[b] = lds32(sat + b * 16);
            }
            multiply<NT>(acc, a, w, sb);
        }
        put_scales(i + T::kStages - 1);        // read two barriers on at the earliest
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    join<WF, WT, NT>(acc, smem, cluster, f0, m0, col, C, ldc, M, N, alpha, accumulate);
}

// ── the same with TMA ───────────────────────────────────────────────────────
// For rows of q that TMA can address (N % 16 == 0).  A warp for each stage fills it: q and A as boxes (zeros outside the arrays),
// the scale bytes by hand, read one round ahead; with one warp for all stages the latency of those reads was the time of a stage
// (1.5 us).  The WF * WT others wait for nothing but their data.
template <int WF, int WT, int NT, int KS, int ST>
struct TmaTile {
    static constexpr int kThreads = 32 * (WF * WT + ST), kFeat = 64 * WF, kTokens = 16 * WT * KS, kStages = ST;
    static constexpr int kBlk = kFeat / kQ8Block;
    static constexpr int kBox = kFeat < 128 ? kFeat : 128;            // bytes of a q row in one box, the box's swizzle span
    static constexpr int kCols = NT == 2 ? 16 : NT == 4 ? 32 : 64;    // of A in a box: 32, 64 or 128 bytes
    static constexpr int kQ = kTokens * kFeat, kA = kTokens * kCols * 2, kS = kTokens * kBlk;
    static constexpr int kStage = (kQ + kA + kS + 1023) / 1024 * 1024;
    static constexpr int kRed = (WT > 1 ? WT / 2 : 1) * NT * 8 * (kFeat + 4) * 4;
    static constexpr int kSmem = (kStages * kStage > kRed ? kStages * kStage : kRed) + 1024;
    static_assert(kTokens <= 256 && kBox * kTokens % 1024 == 0 && kQ % 1024 == 0 && kA % 1024 == 0, "");
};

template <int WF, int WT, int NT, int KS, int ST>
__global__ void __launch_bounds__(32 * (WF * WT + ST)) gemm_tokens_q8_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap a_map,
                                                                           const uint8_t* __restrict__ scale, const __nv_bfloat16* __restrict__ col,
                                                                           float* __restrict__ C, long ldc, int M, int N, int K, float alpha,
                                                                           int accumulate, int* status) {
    using T = TmaTile<WF, WT, NT, KS, ST>;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
    __shared__ uint64_t full[ST], empty[ST];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int f0 = int(blockIdx.x) / cs * T::kFeat, m0 = int(blockIdx.y) * NT * 8;
    const int chunks = (K + T::kTokens - 1) / T::kTokens;
    const int mine = chunks > rank ? (chunks - rank + cs - 1) / cs : 0;   // chunks rank, rank + cs, ...
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], WF * WT);
        }
        abort_word = 0;
        fence_barrier_init();
    }
    __syncthreads();

    // A thread's four tokens of a step of 16 and its place in the swizzled rows of q: with 128-byte rows 2t + {0, 1, 8, 9}, with
    // 64-byte rows {0, 4, 1, 5}[t] + {0, 2, 8, 10}, so that the four rows a load touches fall on different banks.
    auto token = [](int tt, int j) {
        return WF > 1 ? 2 * tt + (j & 1) + (j >> 1) * 8 : (tt & 1) * 4 + (tt >> 1) + (j & 1) * 2 + (j >> 1) * 8;
    };
    float acc[4][NT][4] = {};
    if (warp >= WF * WT) {
        const int nblk = (N + kQ8Block - 1) / kQ8Block;
        constexpr int kWords = T::kS / 4 / 32;       // words of four tokens' scales a lane brings into a stage
        static_assert(T::kS % 128 == 0, "");
        uint8_t held[kWords][4];
        auto read_scales = [&](int i) {
            const int tok0 = (i * cs + rank) * T::kTokens;
#pragma unroll
            for (int c = 0; c < kWords; c++) {
                const int word = c * 32 + lane, blk = word % T::kBlk, tt = word / T::kBlk & 3, step = word / T::kBlk / 4;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int tok = tok0 + step * 16 + token(tt, j), b = f0 / kQ8Block + blk;
                    held[c][j] = tok < K && b < nblk ? scale[size_t(tok) * nblk + b] : uint8_t(127);
                }
            }
        };
        const int st = warp - WF * WT;
        if (st < mine) read_scales(st);
        for (int i = st; i < mine; i += ST) {
            if (!mbar_wait(&empty[st], (i / ST & 1) ^ 1, abort_flag, status, DS_TIMEOUT_PRODUCER)) break;
            unsigned char* at = smem + st * T::kStage;
#pragma unroll
            for (int c = 0; c < kWords; c++) {
                const int word = c * 32 + lane, blk = word % T::kBlk, tt = word / T::kBlk & 3, step = word / T::kBlk / 4;
                *reinterpret_cast<uint32_t*>(at + T::kQ + T::kA + ((step * T::kBlk + blk) * 4 + tt) * 4) =
                    held[c][0] | held[c][1] << 8 | held[c][2] << 16 | uint32_t(held[c][3]) << 24;
            }
            __syncwarp();
            if (lane == 0) {
                const int tok0 = (i * cs + rank) * T::kTokens;
                mbar_arrive_expect_tx(&full[st], T::kQ + T::kA);
#pragma unroll
                for (int x = 0; x < T::kFeat / T::kBox; x++) tma_load_2d(at + x * T::kTokens * T::kBox, &q_map, &full[st], f0 + x * T::kBox, tok0);
                tma_load_2d(at + T::kQ, &a_map, &full[st], m0, tok0);
            }
            if (i + ST < mine) read_scales(i + ST);
        }
    } else {
        const int wf = warp % WF, wt = warp / WF;
        // q: chunk of 16 bytes c of row r lies at c ^ (r & 7) (128-byte rows) or c ^ (r >> 1 & 3) (64-byte rows)
        auto q_at = [&](int j) {
            const int r = token(t, j), c = (wf * 64 % T::kBox + g * 4) / 16, s = T::kBox == 128 ? r & 7 : r >> 1 & 3;
            return wf * 64 / T::kBox * T::kTokens * T::kBox + r * T::kBox + ((c ^ s) * 16 | (g * 4 & 15));
        };
        const int q0 = q_at(0), q1 = q_at(1);
        constexpr int kHigh = 8 * T::kBox;           // tokens 2 and 3 lie eight rows below, same swizzle
        // A: row k of a fragment is token(k / 2 & 3, k & 1 + k / 8 * 2); chunk of 16 bytes c at c ^ swizzle of the row
        const int ar = token((lane & 7) >> 1, (lane & 1) + (lane >> 3 & 1) * 2);
        const int as = T::kCols == 16 ? ar >> 2 & 1 : T::kCols == 32 ? ar >> 1 & 3 : ar & 7;
        const int a0 = ar * T::kCols * 2 + (((lane >> 4) ^ as) * 16);
        for (int i = 0; i < mine; i++) {
            const int st = i % ST;
            if (!mbar_wait(&full[st], i / ST & 1, abort_flag, status, DS_TIMEOUT_MMA)) break;
            const uint32_t base = smem_u32(smem) + st * T::kStage;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                const int step = wt * KS + k;
                const uint32_t qb = base + step * 16 * T::kBox, ab = base + T::kQ + step * 16 * T::kCols * 2 + a0;
                const uint32_t sat = base + T::kQ + T::kA + (step * T::kBlk + wf * 2) * 16 + t * 4;
                uint32_t a[NT / 2][4], w[2][4], sb[2];
#pragma unroll
                for (int n = 0; n < NT / 2; n++) ldmatrix_x4_trans(a[n], ab ^ (n * 32));
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    w[b][0] = lds32(qb + (q0 ^ b * 32));
                    w[b][1] = lds32(qb + (q1 ^ b * 32));
                    w[b][2] = lds32(qb + kHigh + (q0 ^ b * 32));
                    w[b][3] = lds32(qb + kHigh + (q1 ^ b * 32));
                    sb[b] = lds32(sat + b * 16);
                }
                multiply<NT>(acc, a, w, sb);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
    }
    __syncwarp();
    if (*abort_flag) {
        // give copies already in flight time to land before shared memory is reused
        for (int i = 0; i < 200; i++) __nanosleep(1000);
    }
    join<WF, WT, NT>(acc, smem, cluster, f0, m0, col, C, ldc, M, N, alpha, accumulate);
}

struct Call {
    ta_ctx* ctx;
    cudaStream_t stream;
    const uint8_t *q, *scale;
    const __nv_bfloat16* A;
    long lda;
    const __nv_bfloat16* col;
    float* C;
    long ldc;
    int M, N, K;
    float alpha;
    int accumulate;
};

template <typename T>
cudaLaunchConfig_t config(const Call& c, int NT, int cs, cudaLaunchAttribute& at) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned((c.N + T::kFeat - 1) / T::kFeat * cs), unsigned((c.M + NT * 8 - 1) / (NT * 8)));
    cfg.blockDim = dim3(T::kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = c.stream;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(cs); at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cfg;
}

template <int WF, int WT, int NT, int KS, int ST>
int launch_any(const Call& c) {
    using T = Tile<WF, WT, NT, KS, ST>;
    ta_ctx* ctx = c.ctx;
    const auto kernel = gemm_tokens_q8_any_kernel<WF, WT, NT, KS, ST>;
    TA_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
    // as many CTAs on a column tile as there are stages of tokens, 8 (the portable cluster) at most
    int cs = 8;
    while (cs > 1 && c.K <= cs / 2 * T::kTokens) cs /= 2;
    cudaLaunchAttribute at{};
    const cudaLaunchConfig_t cfg = config<T>(c, NT, cs, at);
    TA_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, c.q, c.scale, c.A, c.lda, c.col, c.C, c.ldc, c.M, c.N, c.K, c.alpha, c.accumulate));
    TA_LAUNCH_CHECK(ctx, "gemm_tokens_q8_any_kernel");
    return TA_OK;
}
template <int WF, int WT>
int any_for_rank(const Call& c) {
    constexpr int KS = WF == 1 ? 1 : 2;
    return c.M <= 16 ? launch_any<WF, WT, 2, KS, 4>(c) : c.M <= 32 ? launch_any<WF, WT, 4, KS, 4>(c) : c.M <= 48 ? launch_any<WF, WT, 6, KS, 4>(c) : launch_any<WF, WT, 8, KS, 4>(c);
}

template <int WF, int WT, int NT, int KS, int ST>
int launch_tma(const Call& c, int force_cs = 0) {
    using T = TmaTile<WF, WT, NT, KS, ST>;
    ta_ctx* ctx = c.ctx;
    const auto kernel = gemm_tokens_q8_kernel<WF, WT, NT, KS, ST>;
    TA_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
    int cs = 8;
    while (cs > 1 && c.K <= cs / 2 * T::kTokens) cs /= 2;
    if (force_cs) cs = force_cs;
    CUtensorMap q_map, a_map;
    if (int rc = encode_tmap_2d(ctx, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.q, c.N, c.K, c.N, T::kBox, T::kTokens, T::kBox, &q_map)) return rc;
    if (int rc = encode_tmap_2d(ctx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.A, c.M, c.K, c.lda * 2, T::kCols, T::kTokens, T::kCols * 2, &a_map)) return rc;
    cudaLaunchAttribute at{};
    const cudaLaunchConfig_t cfg = config<T>(c, NT, cs, at);
    TA_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, q_map, a_map, c.scale, c.col, c.C, c.ldc, c.M, c.N, c.K, c.alpha, c.accumulate, ctx->d_status));
    TA_LAUNCH_CHECK(ctx, "gemm_tokens_q8_kernel");
    return TA_OK;
}
template <int WF, int WT>
int tma_for_rank(const Call& c) {
    constexpr int KS = WF == 1 ? 1 : 2;
    return c.M <= 16 ? launch_tma<WF, WT, 2, KS, 4>(c) : c.M <= 32 ? launch_tma<WF, WT, 4, KS, 4>(c) : c.M <= 48 ? launch_tma<WF, WT, 6, KS, 4>(c) : launch_tma<WF, WT, 8, KS, 4>(c);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_gemm_tokens_q8_f32(ta_ctx* ctx, int M, int N, int K, float alpha, const void* A, long lda, const void* q, const void* scale,
                                     const void* col, float* C, long ldc, int accumulate, void* stream) {
    if (!ctx || !A || !q || !scale || !C || M <= 0 || N <= 0 || K < 0)
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: null argument or bad size");
    if (M % 8 || N % 8 || lda % 8 || lda < M || ldc < N)
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: M, N and lda must be multiples of 8, lda >= M, ldc >= N");
    if ((reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(q) & 15))
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: pointers must be 16-byte aligned");
    if (int rc = on_ctx_device(ctx, "gemm_tokens_q8_f32")) return rc;
    const Call c{ctx, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale),
                 static_cast<const __nv_bfloat16*>(A), lda, static_cast<const __nv_bfloat16*>(col), C, ldc, M, N, K, alpha, accumulate};
    // four warps abreast share a stage's rows of A; where that leaves SMs without a CTA, one
    const bool wide = (N + 255) / 256 * 8 >= ctx->sm_count;
    if (N % 16 == 0 && K > 0) return wide ? tma_for_rank<2, 4>(c) : tma_for_rank<1, 8>(c);
    return wide ? any_for_rank<4, 2>(c) : any_for_rank<1, 8>(c);
}
