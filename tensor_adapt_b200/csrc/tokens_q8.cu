// An adapter's gradient from an input that is held in 8 bits (act8.cuh):
//
//     C[m][f] (+)= alpha * col[f] * sum_t A[t][m] * q[t][f] * 2^k(t, f / 32)
//
// A [tokens][M] BF16 (dh of the adapter, or of several that share the input), q / scale [tokens][N].  The sum runs over
// tokens, the slow axis of both operands, and the scale changes along it, so it cannot be taken out of the sum.
//
// A CTA takes 128 columns of q and a share of the tokens, 128 at a time (a chunk).  q, its scales and the matching rows of A come
// into shared memory asynchronously.  Warps widen q to BF16 with its scale (exact), pairing tokens on the way, and store it to
// tensor memory as the K-major first operand [128 columns][tokens] of tcgen05.mma; A is the second, MN-major, from shared memory;
// D [128 columns][M ranks] is in tensor memory too.  The CTAs on the same columns are a cluster, which adds its sums through
// distributed shared memory in a fixed order: no partial sums in global memory, no second launch, the same bits every time.
//
// tcgen05.mma cuts its sums off instead of rounding them: 8e-6 of the result after 512 products in a row, 1.4e-6 after 128.  So
// after every four chunks, 32 products, D is added to a running sum beside it, rounded, and starts again (3e-7 in all).
//
// What bounds it, at 16384 tokens x 18944 columns and rank 16: the way of q through memory (5.5 TB/s while it runs), with the scale
// bytes beside it, of whose 32-byte sectors a tile uses four.  In-kernel clocks show the widening warps waiting for data most of the
// time; issue slots are 60 % busy, the ALU 42 %, the tensor cores 7 %.  6 to 8 us any call has: launch, first loads, join.  Measured
// (us a call; the bytes at the copy rate in parentheses): 16384 x 18944, rank 16, 75 (49); 8192 x 8960, rank 64, 28 (12); 8192 x 896,
// rank 48, 12 (1.3); 8192 x 3584, rank 192, 25 (5).  Other arrangements at the first, on the device, where this one takes 63: mma.sync
// from registers 66 and at the second 50, where its products alone take 17; the widened operand in shared memory instead, 97 (6 bytes
// of its traffic an element); q straight to the widening warps' registers, 94 (the proxy fence after a chunk waits for the loads in
// flight).
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <mutex>

#include "act8.cuh"
#include "ctx.h"

namespace ta {
namespace {

namespace cg = cooperative_groups;

constexpr int kFeat = 128, kTok = 128;      // a chunk: columns of q, tokens
constexpr int kConv = 8;                    // warps that widen q, in two sets; behind them the loaders, one that issues TMA copies, one that multiplies
constexpr int kPitch = kFeat + 4;           // of the sums in shared memory

constexpr int kRun = 4;                     // chunks that D takes in a row

// NB: room for ranks, 16, 32, 64, 128 or 192.  Rings: RS chunks of q and scales, BS of A's rows, two of the widened operand.  The sets of
// widening warps and the loaders of the TMA form take chunks in turn.  A wait on a barrier's parity cannot tell phases two apart, so
// nobody may come to a slot whose phase before last is not complete: with an even ring and two of each, a slot is always the same
// set's and the same loader's, which has waited for that phase itself.
// WIDE: rows of q start on 16 bytes (N % 16 == 0) and come by TMA; otherwise on 8, by cp.async, which takes more warps.
template <int NB, bool WIDE, int RS, int BS>
struct Tile {
    static constexpr int kLoad = WIDE ? 2 : 6, kThreads = 32 * (kConv + kLoad + 2);
    static_assert(RS % 2 == 0, "");
    static constexpr int kWide = NB < 64 ? NB : 64, kRow = 2 * kWide; // of a box of A: ranks, bytes
    static constexpr int kBoxes = NB / kWide;
    static constexpr int kQ = kFeat * kTok, kBox = kTok * kRow, kB = kBoxes * kBox;
    static constexpr int kScale = kTok * (kFeat / kQ8Block) * 2;     // as BF16
    static constexpr int kAtB = RS * kQ, kAtS = kAtB + BS * kB;
    static constexpr int kRings = kAtS + RS * kScale, kRed = NB * kPitch * 4;
    static constexpr int kSmem = (kRings > kRed ? kRings : kRed) + 1024;
    static constexpr int kX = kTok / 2;                             // tensor-memory columns of a widened chunk
    static constexpr int kTmem = 2 * NB + 2 * kX <= 256 ? 256 : 512;  // D, the running sum, two widened chunks
};

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
// Registers of 16 x 4 fragments of 32-bit values side by side (lane / 4 the row, lane % 4 the column, rows 8 on in the odd registers) to
// 16 lanes and 16 columns of tensor memory.
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(on ? 8 : 0) : "memory");
}
// One of the barrier's arrivals, once this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int NB, bool WIDE, int RS, int BS>
__global__ void __launch_bounds__(Tile<NB, WIDE, RS, BS>::kThreads, NB <= 64 ? 2 : 1) gemm_tokens_q8_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap a_map,
                                                                     const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                                     const __nv_bfloat16* __restrict__ col, float* __restrict__ C, long ldc, int M,
                                                                     int N, int K, float alpha, int accumulate, int* status) {
    using T = Tile<NB, WIDE, RS, BS>;
    constexpr int kLoad = T::kLoad, kThreads = T::kThreads;
    extern __shared__ unsigned char raw_smem[];
    unsigned char* smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
    __shared__ uint64_t q_full[RS], q_empty[RS], x_full[2], x_empty[2], b_full[BS], b_empty[BS], d_full, d_empty, done;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    cg::cluster_group cluster = cg::this_cluster();
    const int cs = int(cluster.num_blocks()), rank = int(cluster.block_rank());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int f0 = int(blockIdx.x) / cs * kFeat, m0 = int(blockIdx.y) * NB;
    const int chunks = (K + kTok - 1) / kTok;
    const int mine = chunks > rank ? (chunks - rank + cs - 1) / cs : 0;   // chunks rank, rank + cs, ...
    auto copy_q = [&](int j) {
        mbar_arrive_expect_tx(&q_full[j % RS], T::kQ);
        tma_load_2d(smem + j % RS * T::kQ, &q_map, &q_full[j % RS], f0, (j * cs + rank) * kTok);
    };
    auto copy_a = [&](int i) {
        mbar_arrive_expect_tx(&b_full[i % BS], T::kB);
#pragma unroll
        for (int c = 0; c < T::kBoxes; c++)
            tma_load_2d(smem + T::kAtB + i % BS * T::kB + c * T::kBox, &a_map, &b_full[i % BS], m0 + T::kWide * c, (i * cs + rank) * kTok);
    };
    if (threadIdx.x == 32 * (kConv + kLoad)) {
        for (int i = 0; i < RS; i++) {
            mbar_init(&q_full[i], WIDE ? 2 : 1 + 32 * kLoad);
            mbar_init(&q_empty[i], kConv / 2);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&x_full[i], kConv / 2);
            mbar_init(&x_empty[i], 1);
        }
        for (int i = 0; i < BS; i++) {
            mbar_init(&b_full[i], 1);
            mbar_init(&b_empty[i], 1);
        }
        mbar_init(&d_full, 1);
        mbar_init(&d_empty, kConv / 2);
        mbar_init(&done, 1);
        abort_word = 0;
        fence_barrier_init();
        fence_proxy_async_smem();
        // the first round of the rings: this thread's copies need nobody else
        for (int i = 0; i < RS && i < mine; i++) {
            if (WIDE) copy_q(i);
            if (i < BS) copy_a(i);
        }
    }
    // Where q comes by TMA the loaders have its scales alone and take chunks in turn; by cp.async all work on every chunk, and the
    // first has the scales.  Those are too small and unaligned for an asynchronous copy: a lane reads the four blocks' bytes of
    // tokens 2t, 2t + 1, 2t + 8 and 2t + 9 of a step of 16 (t: lane % 4, the step: lane / 4) one chunk ahead, and stores them as
    // BF16 pairs.  (Two ahead is slower by 1 to 2 us, the lines of L1 that the reads in flight hold are too many; so is a prefetch
    // to L2, by 5.)
    const int nblk = int((unsigned(N) + kQ8Block - 1) / kQ8Block), blk0 = f0 / kQ8Block, me = warp - kConv;
    constexpr int kTurn = WIDE ? kLoad : 1;
    const int first = WIDE ? me : 0;
    const bool words = nblk % 4 == 0 && (reinterpret_cast<uintptr_t>(scale) & 3) == 0;    // then so are four blocks of a row
    uint32_t held[4];
    auto read = [&](int i, uint32_t (&h)[4]) {
        const int tok0 = (i * cs + rank) * kTok + (lane >> 2) * 16 + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int tok = tok0 + (j & 1) + (j >> 1) * 8;
            h[j] = 0x7F7F7F7Fu;
            if (i >= mine || tok >= K || (!WIDE && me != 0)) continue;
            const uint8_t* p = scale + size_t(tok) * nblk + blk0;
            if (words) {
                h[j] = __ldg(reinterpret_cast<const uint32_t*>(p));
            } else {
#pragma unroll
                for (int b = 0; b < 4; b++)
                    if (blk0 + b < nblk) h[j] = (h[j] & ~(0xFFu << 8 * b)) | uint32_t(p[b]) << 8 * b;
            }
        }
    };
    if (warp >= kConv && warp < kConv + kLoad) read(first, held);
    if (warp == kConv + kLoad + 1) {
        tmem_alloc(&tmem_slot, T::kTmem);
        tmem_relinquish();
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    tcgen05_fence_after_sync();
    const uint32_t d_tmem = tmem_slot, s_tmem = d_tmem + NB, x_tmem = s_tmem + NB, base = smem_u32(smem);
    const int ranks = min(NB, M - m0);
    const uint32_t quarter = uint32_t((warp & 3) * 32) << 16;       // the lanes of tensor memory that this warp may touch

    // A wait that gives up leaves its code in `status`, raises the flag and lets the others give up in turn.  A warp leaves its loop
    // as one: none may arrive on a barrier once more than its phase expects.
    auto warp_wait = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code)) != 0; };
    if (warp < kConv) {
        // A set of four warps widens every other chunk.  A warp has the 32 lanes of tensor memory, that is the block of 32 columns,
        // that its number allows.  Of each step of 16 tokens a thread reads four columns of tokens 2t, 2t + 1, 2t + 8 and 2t + 9
        // (t: lane % 4, g: lane / 4): columns 4g and 4g + 1 become rows g and g + 8 of a fragment, 4g + 2 and 4g + 3 those of a
        // second one.  128-byte rows are swizzled, chunk of 16 bytes c of row r at c ^ (r & 7): the four rows of a load fall on
        // different banks.
        const int g = lane >> 2, t = lane & 3, blk = warp & 3, set = warp >> 2;
        const uint32_t even = 2 * t * 128 + (((blk * 2 + (g >> 2)) ^ (2 * t)) * 16 | (g * 4 & 15)), odd = (even + 128) ^ 16;
        const uint32_t s_src = base + T::kAtS + (t * 4 + blk) * 8, x_dst = x_tmem + set * T::kX + quarter;
        int rs = set;
        uint32_t r_phase = 0, x_phase = 1;
        for (int i = set; i < mine; i += 2) {
            if (!warp_wait(&q_full[rs], r_phase, DS_TIMEOUT_MMA)) break;
            if (!warp_wait(&x_empty[set], x_phase, DS_TIMEOUT_PRODUCER)) break;
            tcgen05_fence_after_sync();
            const uint32_t src = base + rs * T::kQ, ssrc = s_src + rs * T::kScale;
#pragma unroll
            for (int k = 0; k < kTok / 32; k++) {      // two steps
                uint32_t w[2][4];
                uint2 s[2];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t at = src + (2 * k + u) * 2048;
                    w[u][0] = lds32(at + even);
                    w[u][1] = lds32(at + odd);
                    w[u][2] = lds32(at + even + 1024);
                    w[u][3] = lds32(at + odd + 1024);
                    s[u] = lds64(ssrc + (2 * k + u) * 128);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t x[8];
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const float2 v0 = widen2(w[u][0], h), v1 = widen2(w[u][1], h), v2 = widen2(w[u][2], h), v3 = widen2(w[u][3], h);
                        x[4 * u] = mul_bf16x2(pack_bf16x2(v0.x, v1.x), s[u].x);
                        x[4 * u + 1] = mul_bf16x2(pack_bf16x2(v0.y, v1.y), s[u].x);
                        x[4 * u + 2] = mul_bf16x2(pack_bf16x2(v2.x, v3.x), s[u].y);
                        x[4 * u + 3] = mul_bf16x2(pack_bf16x2(v2.y, v3.y), s[u].y);
                    }
                    tmem_st_frag(x_dst + k * 16 + (uint32_t(h * 16) << 16), x);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_empty[rs]);
            tmem_st_wait();
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&x_full[set]);
            if (i > 0 && i % kRun == 0) {      // the run before this chunk
                if (!warp_wait(&d_full, (i / kRun - 1) & 1, DS_TIMEOUT_EPILOGUE)) break;
                tcgen05_fence_after_sync();
                for (int n = 0; n < ranks; n += 16) {
                    uint32_t d[16], old[16];
                    tmem_ld_x16(d_tmem + n + quarter, d);
                    if (i > kRun) tmem_ld_x16(s_tmem + n + quarter, old);
                    tmem_ld_wait();
                    uint32_t lo[8], hi[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        lo[e] = i > kRun ? __float_as_uint(__uint_as_float(d[e]) + __uint_as_float(old[e])) : d[e];
                        hi[e] = i > kRun ? __float_as_uint(__uint_as_float(d[e + 8]) + __uint_as_float(old[e + 8])) : d[e + 8];
                    }
                    tmem_st_x8(s_tmem + n + quarter, lo);
                    tmem_st_x8(s_tmem + n + 8 + quarter, hi);
                }
                tmem_st_wait();
                tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty);
            }
            if ((rs += 2) >= RS) { rs -= RS; r_phase ^= 1; }
            x_phase ^= 1;
        }
    } else if (warp < kConv + kLoad) {
        auto copy = [&](int i, const uint32_t (&h)[4]) {
            const int rs = i % RS;
            if (!warp_wait(&q_empty[rs], (i / RS & 1) ^ 1, DS_TIMEOUT_PRODUCER)) return false;
            if constexpr (!WIDE) {
                // a lane has eight columns of every 2 kLoad-th token
                const int f = lane % 16 * 8, tok1 = lane / 16 + 2 * me, tok0 = (i * cs + rank) * kTok;
                const uint8_t* src = q + size_t(tok0 + tok1) * N + f0 + f;
                const uint32_t dst = base + rs * T::kQ + (f & 8);
#pragma unroll 4
                for (int r = tok1; r < kTok; r += 2 * kLoad, src += size_t(2 * kLoad) * N) {
                    const bool on = tok0 + r < K && f0 + f < N;
                    cp_async8(dst + r * 128 + (f / 16 ^ (r & 7)) * 16, on ? src : q, on);
                }
                cp_async_arrive(&q_full[rs]);
                if (me != 0) return true;
            }
            uint32_t pair[8];       // BF16's 2^k of tokens 2t and 2t + 1, and of 2t + 8 and 2t + 9, for each block
#pragma unroll
            for (int b = 0; b < 4; b++) {
                pair[2 * b] = (h[0] >> 8 * b & 0xFF) << 7 | (h[1] >> 8 * b & 0xFF) << 23;
                pair[2 * b + 1] = (h[2] >> 8 * b & 0xFF) << 7 | (h[3] >> 8 * b & 0xFF) << 23;
            }
            uint4* to = reinterpret_cast<uint4*>(smem + T::kAtS + rs * T::kScale) + lane * 2;
            to[0] = make_uint4(pair[0], pair[1], pair[2], pair[3]);
            to[1] = make_uint4(pair[4], pair[5], pair[6], pair[7]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[rs]);
            return true;
        };
        for (int i = first; i < mine; i += kTurn) {
            if (!copy(i, held)) break;
            read(i + kTurn, held);
        }
    } else if (warp == kConv + kLoad) {
        if (lane == 0) {
            // Chunk j of q by TMA, then chunk i of A, as many chunks behind as its ring is shorter: the slot of A is given back
            // by the products of the chunk whose widening gave back q's.  (q from the warps that have its scales, and so behind
            // their reads: 1 to 2 % slower.)
            constexpr int kLag = WIDE ? RS - BS : 0;
            for (int j = BS + kLag; j < mine + kLag; j++) {      // BS + kLag is RS where q comes by TMA
                if (WIDE && j < mine) {
                    if (!mbar_wait(&q_empty[j % RS], (j / RS & 1) ^ 1, abort_flag, status, DS_TIMEOUT_PRODUCER)) break;
                    copy_q(j);
                }
                const int i = j - kLag;
                if (!mbar_wait(&b_empty[i % BS], (i / BS & 1) ^ 1, abort_flag, status, DS_TIMEOUT_PRODUCER)) break;
                copy_a(i);
            }
        }
    } else if (lane == 0) {
        const uint32_t idesc = umma_idesc_bf16(kFeat, (ranks + 15) / 16 * 16, false, true);
        bool ok = true;
        for (int i = 0; i < mine && ok; i++) {
            const int xs = i & 1, bs = i % BS;
            ok = mbar_wait(&b_full[bs], i / BS & 1, abort_flag, status, DS_TIMEOUT_MMA) && mbar_wait(&x_full[xs], i >> 1 & 1, abort_flag, status, DS_TIMEOUT_MMA);
            if (ok && i > 0 && i % kRun == 0) ok = mbar_wait(&d_empty, (i / kRun - 1) & 1, abort_flag, status, DS_TIMEOUT_MMA);
            if (!ok) break;
            tcgen05_fence_after_sync();
            const uint64_t bd = smem_desc(T::kRow, base + T::kAtB + bs * T::kB, T::kBox, 8 * T::kRow);
#pragma unroll
            for (int k = 0; k < kTok / 16; k++) umma_bf16_ts(d_tmem, x_tmem + xs * T::kX + k * 8, bd + k * T::kRow, idesc, uint32_t(i % kRun + k > 0));
            umma_commit(&x_empty[xs]);
            umma_commit(&b_empty[bs]);
            if (i % kRun == kRun - 1 && i + 1 < mine) umma_commit(&d_full);
        }
        if (ok && mine > 0) umma_commit(&done);
    }
    __syncwarp();
    if (mine > 0 && warp < kConv) mbar_wait(&done, 0, abort_flag, status, DS_TIMEOUT_EPILOGUE);
    if constexpr (!WIDE) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    if (*abort_flag) {
        // give copies and products already in flight time to land before shared memory is reused
        for (int i = 0; i < 200; i++) __nanosleep(1000);
    }
    __syncthreads();

    // D to shared memory, [rank][column]; tensor memory is given back before anything waits for another CTA
    float* red = reinterpret_cast<float*>(smem);
    if (warp < kConv) {
        tcgen05_fence_after_sync();
        float* to = red + (warp & 3) * 32 + (lane & 7) * 4 + (lane >> 3);   // row 8 j + g of a block is column 4 g + j
#pragma unroll 1
        for (int n = (warp >> 2) * 16; n < ranks; n += 32) {
            uint32_t r[16], old[16];
            if (mine > 0) tmem_ld_x16(d_tmem + n + quarter, r);
            if (mine > kRun) tmem_ld_x16(s_tmem + n + quarter, old);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; e++) {
                float v = mine > 0 ? __uint_as_float(r[e]) : 0.f;
                if (mine > kRun) v += __uint_as_float(old[e]);
                to[(n + e) * kPitch] = v;
            }
        }
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == kConv + kLoad + 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc(d_tmem, T::kTmem);
    }
    cluster.sync();
    // Four columns a thread; the reads of the cluster's sums are issued together.
    const bool whole = ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
    for (int o = rank * kThreads + int(threadIdx.x); o < ranks * (kFeat / 4); o += cs * kThreads) {
        const int m = o / (kFeat / 4), c = o % (kFeat / 4) * 4;
        if (f0 + c >= N) continue;                     // N is a multiple of 8: all four or none
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int from = 0; from < cs; from += 8) {
            float4 part[8];
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (from + r < cs) part[r] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(red, from + r) + m * kPitch + c);
#pragma unroll
            for (int r = 0; r < 8; r++)
                if (from + r < cs) { sum[0] += part[r].x; sum[1] += part[r].y; sum[2] += part[r].z; sum[3] += part[r].w; }
        }
        float* out = C + size_t(m0 + m) * ldc + f0 + c;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sum[e] *= alpha;
            if (col) sum[e] *= __bfloat162float(col[f0 + c + e]);
        }
        if (whole) {
            float4 v = make_float4(sum[0], sum[1], sum[2], sum[3]);
            if (accumulate) {
                const float4 old = *reinterpret_cast<const float4*>(out);
                v.x += old.x; v.y += old.y; v.z += old.z; v.w += old.w;
            }
            *reinterpret_cast<float4*>(out) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) out[e] = accumulate ? out[e] + sum[e] : sum[e];
        }
    }
    // Nobody leaves while its sums are read.  A relaxed arrival does not wait for the stores above (0.2 to 0.3 us); the reads are done,
    // since the stores take their values.
    asm volatile("barrier.cluster.arrive.relaxed;\nbarrier.cluster.wait;" ::: "memory");
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

// Clusters of 1 to 16 CTAs that the device holds at a time with one CTA on an SM (`alone`) and in all, asked once for each kernel and
// device.  The answer counts one CTA an SM for these kernels, two of which run on one (NB <= 64: counters show 24 warps active of 2 x
// 12); clusters of cs at two CTAs an SM are then as many as clusters of cs / 2 at one.  Above 8 that did not hold: 12 clusters of 16 take
// 13.5 us at 1536 columns x 8192 tokens, of 8 11.9.
constexpr int kMostCtas = 16;
struct Residency {
    int alone[kMostCtas + 1] = {}, all[kMostCtas + 1] = {};
    bool known = false;
};
std::mutex residency_lock;   // contexts of several host threads share the answers
template <typename F>
void ask(F kernel, cudaLaunchConfig_t cfg, cudaLaunchAttribute& at, int per_sm, int sm_count, Residency& r) {
    int n[kMostCtas + 1] = {};
    for (int cs = 1; cs <= kMostCtas; cs++) {
        at.val.clusterDim.x = unsigned(cs);
        cfg.gridDim = dim3(unsigned(cs));
        if (cudaOccupancyMaxActiveClusters(&n[cs], kernel, &cfg) != cudaSuccess) n[cs] = 0;
    }
    (void)cudaGetLastError();
    const bool both = n[1] > sm_count;      // it did count two
    for (int cs = 1; cs <= kMostCtas; cs++) {
        r.alone[cs] = both ? n[cs] / 2 : n[cs];
        r.all[cs] = both || per_sm == 1 || cs > 8 ? n[cs] : cs == 1 ? 2 * n[1] : std::max(n[cs], n[(cs + 1) / 2]);
    }
    r.known = true;
}

template <int NB, bool WIDE, int RS, int BS>
int launch(const Call& c) {
    using T = Tile<NB, WIDE, RS, BS>;
    ta_ctx* ctx = c.ctx;
    const auto kernel = gemm_tokens_q8_kernel<NB, WIDE, RS, BS>;
    static Residency resident[64];
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(T::kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = c.stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    Residency fit;
    {
        std::lock_guard<std::mutex> hold(residency_lock);
        Residency& known = resident[ctx->device & 63];
        if (!known.known) {
            TA_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem));
            TA_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            ask(kernel, cfg, at, NB <= 64 ? 2 : 1, ctx->sm_count, known);
        }
        fit = known;
    }
    // CTAs on a column tile: the least time by what was measured (us): 6 whatever the chunks, 7 in a cluster above 8, and a CTA's chunk
    // 0.72 alone on its SM, 1.05 with another.  E.g. 8192 tokens: 896 columns (7 tiles) 16 CTAs a tile 10.0 (8: 11.9); 1536, 8 11.9 (6
    // 13.7, 16 13.5); 4864, 6 16.6 (4 20.3, 8 23.2); 8960, 4 24.8 (2 29.6, 8 41).
    const unsigned tiles = (unsigned(c.N) + kFeat - 1) / kFeat, rows = (unsigned(c.M) + NB - 1) / NB;
    const int chunks = (c.K + kTok - 1) / kTok;
    const long clusters = long(tiles) * rows;
    int cs = 0;
    long least = 0;
    for (int k = 1; k <= kMostCtas && k <= chunks; k++) {
        if (fit.all[k] <= 0) continue;
        const long rounds = (clusters + fit.all[k] - 1) / fit.all[k], mine = (chunks + k - 1) / k;
        const long cost = rounds * ((k > 8 ? 700 : 600) + mine * (clusters > fit.alone[k] ? 105 : 72));
        if (cs == 0 || cost < least) { least = cost; cs = k; }
    }
    if (cs == 0) return fail(ctx, TA_ERR_CUDA, "gemm_tokens_q8_f32: the kernel cannot be resident on this device");
    at.val.clusterDim.x = unsigned(cs);
    cfg.gridDim = dim3(tiles * unsigned(cs), rows);
    CUtensorMap q_map{}, a_map;
    if (WIDE)
        if (int rc = encode_tmap_2d(ctx, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.q, c.N, c.K, c.N, kFeat, kTok, 128, &q_map, false)) return rc;
    if (int rc = encode_tmap_2d(ctx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.A, c.M, c.K, c.lda * 2, T::kWide, kTok, T::kRow, &a_map)) return rc;
    ProfScope prof(ctx, c.stream, PROF_GEMM_SKINNY, 2.0 * c.M * c.N * c.K);
    TA_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, q_map, a_map, c.q, c.scale, c.col, c.C, c.ldc, c.M, c.N, c.K, c.alpha, c.accumulate, ctx->d_status));
    TA_LAUNCH_CHECK(ctx, "gemm_tokens_q8_kernel");
    return TA_OK;
}
// Room for 16 or 32 ranks beside 64: boxes of A as wide as they, since a box is filled whatever the rank (16384 x 18944, rank 16, us on
// the device: 62.7 against 70.2; rank 32 65.3).  Rings: four slots of q by TMA (two: 72 at rank 16, and 78 against 74 at rank 64); two
// by cp.async, where L1 and not the latency is short (8960 x 8192, rank 64: 31.7, with four 36.5).  Above 192 ranks, passes of 128.
template <bool WIDE>
int launch_for_rank(const Call& c) {
    constexpr int RS = WIDE ? 4 : 2;
    return c.M <= 16 ? launch<16, WIDE, RS, 2>(c) : c.M <= 32 ? launch<32, WIDE, RS, 2>(c) : c.M <= 64 ? launch<64, WIDE, RS, 2>(c)
         : c.M <= 128 ? launch<128, WIDE, 4, 2>(c) : c.M <= 192 ? launch<192, WIDE, 4, 2>(c) : launch<128, WIDE, 4, 2>(c);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" int ta_gemm_tokens_q8_f32(ta_ctx* ctx, int M, int N, int K, float alpha, const void* A, long lda, const void* q, const void* scale,
                                     const void* col, float* C, long ldc, int accumulate, void* stream) {
    if (!ctx || !A || !q || !scale || !C || M <= 0 || N <= 0 || K < 0)
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: null argument or bad size");
    if (K > INT_MAX - 64 * kTok) return fail(ctx, TA_ERR_UNSUPPORTED, "gemm_tokens_q8_f32: more than 2^31 - 8193 tokens");
    if (M > 65535 * 128) return fail(ctx, TA_ERR_UNSUPPORTED, "gemm_tokens_q8_f32: more than 65535 * 128 ranks");
    if (M % 8 || N % 8 || lda % 8 || lda < M || ldc < N)
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: M, N and lda must be multiples of 8, lda >= M, ldc >= N");
    if ((reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(q) & 15))
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: pointers must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(C) & 3) || (reinterpret_cast<uintptr_t>(col) & 1))
        return fail(ctx, TA_ERR_INVALID, "gemm_tokens_q8_f32: C and col must be aligned to their elements");
    if (int rc = on_ctx_device(ctx, "gemm_tokens_q8_f32")) return rc;
    const Call c{ctx, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(scale),
                 static_cast<const __nv_bfloat16*>(A), lda, static_cast<const __nv_bfloat16*>(col), C, ldc, M, N, K, alpha, accumulate};
    if (K == 0) {   // an empty sum
        if (!accumulate) TA_CUDA(ctx, cudaMemset2DAsync(C, size_t(ldc) * 4, 0, size_t(N) * 4, size_t(M), c.stream));
        return TA_OK;
    }
    return N % 16 == 0 ? launch_for_rank<true>(c) : launch_for_rank<false>(c);
}
