// An adapter's gradient from an input that is held in 8 bits (act8.cuh):
//
//     C[m][f] (+)= alpha * col[f] * sum_t A[t][m] * q[t][f] * 2^k(t, f / 32)
//
// A [tokens][M] BF16 (dh of the adapter, or of several that share the input), q / scale [tokens][N].  The sum runs over
// tokens, the slow axis of both operands, and the scale changes along it, so it cannot be taken out of the sum: a value is
// widened to BF16 (exact) in registers and multiplied by mma.sync (m16n8k16, FP32 accumulators).
#include <cooperative_groups.h>

#include <algorithm>

#include "act8.cuh"
#include "ctx.h"

namespace ta {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8;
constexpr int kFeat = 64;      // columns of q per CTA
constexpr int kPitch = kFeat + 1;

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
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// Two e4m3 values (byte j of each word, of two tokens) as a BF16 pair times 2^-120: sign and the seven other bits moved
// under BF16's eight exponent bits, subnormals included.  e4m3's NaN would come out as 480.
__device__ __forceinline__ uint32_t raw_pair(uint32_t a, uint32_t b, int j) {
    const uint32_t w = __byte_perm(a, b, j | j << 4 | (4 + j) << 8 | (4 + j) << 12);
    return (w & 0x80008000u) | ((w >> 4) & 0x07F007F0u);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (w & 0x7F7F7F7Fu) + 0x01010101u; }   // bit 7 of a NaN's byte

struct Step {
    uint2 q[4];        // eight columns of tokens 2t, 2t+1, 2t+8, 2t+9
    uint32_t byte[4];  // their blocks' scales
};

template <int NT>
__global__ void __launch_bounds__(kWarps * 32) gemm_tokens_q8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                                     const __nv_bfloat16* __restrict__ A, long lda,
                                                                     const __nv_bfloat16* __restrict__ col, float* __restrict__ C, long ldc,
                                                                     int M, int N, int K, float alpha, int accumulate) {
    constexpr int kRow = NT * 16 + 16;             // bytes of a staged row of A: 16-byte chunks an odd number apart
    constexpr int kStage = 16 * kRow;
    constexpr int kSmem = kWarps * 2 * kStage > NT * 8 * kPitch * 4 ? kWarps * 2 * kStage : NT * 8 * kPitch * 4;
    __shared__ __align__(16) unsigned char smem[kSmem];
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int f0 = int(blockIdx.x) / cs * kFeat, m0 = int(blockIdx.y) * NT * 8;
    const int nblk = (N + kQ8Block - 1) / kQ8Block;
    const int f = f0 + 8 * g;
    const bool f_on = f < N;
    const int steps = (K + 15) / 16, stride = cs * kWarps;
    const uint32_t stage = smem_u32(smem) + warp * 2 * kStage;

    float acc[4][NT][4] = {};

    auto fetch = [&](int step, int buf, Step& s) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int tok = step * 16 + 2 * t + (i & 1) + (i >> 1) * 8;
            const bool on = f_on && tok < K;
            s.q[i] = on ? *reinterpret_cast<const uint2*>(q + size_t(tok) * N + f) : make_uint2(0, 0);
            s.byte[i] = on ? scale[size_t(tok) * nblk + f / kQ8Block] : 127u;
        }
#pragma unroll
        for (int i = 0; i < NT / 2; i++) {
            const int c = lane + i * 32, row = c / NT, m = m0 + c % NT * 8, tok = step * 16 + row;
            const bool on = tok < K && m < M;
            cp_async16(stage + buf * kStage + row * kRow + c % NT * 16, on ? A + size_t(tok) * lda + m : A, on);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    Step cur, next;
    int step = rank * kWarps + warp, buf = 0;
    if (step < steps) fetch(step, 0, cur);
    for (; step < steps; step += stride, buf ^= 1) {
        if (step + stride < steps) {
            fetch(step + stride, buf ^ 1, next);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncwarp();
        uint32_t odd = 0, top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            odd |= nan_bytes(cur.q[i].x) | nan_bytes(cur.q[i].y);
            top = max(top, cur.byte[i]);
        }
        // 2^(k + 120) is a BF16 number for k <= 7 (amax <= 57344): one multiplication.  Larger scales and NaN the long way.
        const bool plain = !__any_sync(0xffffffffu, (odd & 0x80808080u) != 0 || top > 134);
        uint32_t s01, s89;
        if (plain) {
            s01 = (cur.byte[0] + 120) << 7 | (cur.byte[1] + 120) << 23;
            s89 = (cur.byte[2] + 120) << 7 | (cur.byte[3] + 120) << 23;
        } else {
            s01 = cur.byte[0] << 7 | cur.byte[1] << 23;
            s89 = cur.byte[2] << 7 | cur.byte[3] << 23;
        }
        uint32_t x[4][4];   // [pair of columns][fragment register]
#pragma unroll
        for (int j = 0; j < 8; j++) {
            auto word = [&](int i) { return j < 4 ? cur.q[i].x : cur.q[i].y; };
            uint32_t lo = raw_pair(word(0), word(1), j & 3), hi = raw_pair(word(2), word(3), j & 3);
            if (!plain) {
                auto settle = [](uint32_t v) {   // times 2^120, NaN restored
                    const bool n0 = (v & 0x7FF0u) == 0x07F0u, n1 = (v & 0x7FF00000u) == 0x07F00000u;
                    v = mul_bf16x2(v, 0x7B807B80u);
                    if (n0) v = (v & 0xFFFF0000u) | 0x7FC0u;
                    if (n1) v = (v & 0x0000FFFFu) | 0x7FC00000u;
                    return v;
                };
                lo = settle(lo);
                hi = settle(hi);
            }
            x[j >> 1][j & 1] = mul_bf16x2(lo, s01);
            x[j >> 1][2 + (j & 1)] = mul_bf16x2(hi, s89);
        }
        const uint32_t rows = stage + buf * kStage + ((lane >> 3 & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16;
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, rows + n * 16);
#pragma unroll
            for (int p = 0; p < 4; p++) {
                mma_bf16(acc[p][n], x[p], b[0], b[1]);
                mma_bf16(acc[p][n + 1], x[p], b[2], b[3]);
            }
        }
        __syncwarp();   // this buffer is filled again two steps on
        cur = next;
    }

    // The warps' sums, then the CTAs' of the cluster, in a fixed order: the same bits every time.
    float* red = reinterpret_cast<float*>(smem);
    for (int w = 0; w < kWarps; w++) {
        __syncthreads();
        if (warp != w) continue;
#pragma unroll
        for (int p = 0; p < 4; p++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float* at = red + (n * 8 + 2 * t + (e & 1)) * kPitch + 8 * g + 2 * p + (e >> 1);
                    *at = w ? *at + acc[p][n][e] : acc[p][n][e];
                }
    }
    cluster.sync();
    for (int o = rank * kWarps * 32 + int(threadIdx.x); o < NT * 8 * kFeat; o += cs * kWarps * 32) {
        const int m = o / kFeat, c = o % kFeat;
        if (m0 + m >= M || f0 + c >= N) continue;
        float sum = 0.f;
        for (int r = 0; r < cs; r++) sum += cluster.map_shared_rank(red, r)[m * kPitch + c];
        sum *= alpha;
        if (col) sum *= __bfloat162float(col[f0 + c]);
        float* out = C + size_t(m0 + m) * ldc + f0 + c;
        *out = accumulate ? *out + sum : sum;
    }
    cluster.sync();   // nobody leaves while its sums are read
}

template <int NT>
int launch(ta_ctx* ctx, cudaStream_t s, const uint8_t* q, const uint8_t* scale, const __nv_bfloat16* A, long lda, const __nv_bfloat16* col,
           float* C, long ldc, int M, int N, int K, float alpha, int accumulate) {
    // as many CTAs on a column tile as have a step of 16 tokens for each of their warps, 8 (the portable cluster) at most
    int cs = 8;
    while (cs > 1 && K < cs * kWarps * 16) cs /= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned((N + kFeat - 1) / kFeat * cs), unsigned((M + NT * 8 - 1) / (NT * 8)));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(cs); at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    TA_CUDA(ctx, cudaLaunchKernelEx(&cfg, gemm_tokens_q8_kernel<NT>, q, scale, A, lda, col, C, ldc, M, N, K, alpha, accumulate));
    TA_LAUNCH_CHECK(ctx, "gemm_tokens_q8_kernel");
    return TA_OK;
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
    const auto run = [&](auto f) {
        return f(ctx, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale),
                 static_cast<const __nv_bfloat16*>(A), lda, static_cast<const __nv_bfloat16*>(col), C, ldc, M, N, K, alpha, accumulate);
    };
    return M <= 16 ? run(launch<2>) : M <= 32 ? run(launch<4>) : M <= 48 ? run(launch<6>) : run(launch<8>);
}
