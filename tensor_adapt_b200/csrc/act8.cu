// Activations held in 8 bits between the forward and the backward pass: the residual add + RMSNorm that also leaves its
// normalised rows in 8 bits and the backward that reads them, SwiGLU forward / backward the same way, and the plain store
// and load.  The form is described in act8.cuh.  All are bound by memory: each element is read once and written once,
// 16-byte vectors of BF16 (8 columns a lane), FP32 inside, sums in FP32.
#include <algorithm>
#include <initializer_list>
#include <string>

#include "act8.cuh"
#include "ctx.h"

namespace ta {
namespace {

// n / d for n < 2^31 with one high multiply (Granlund and Montgomery, "Division by invariant integers using multiplication")
struct FastDiv {
    uint32_t d = 1, mul = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        while ((1ull << shift) < d) shift++;
        mul = uint32_t(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// Where the element-wise kernels' vectors lie.  A row has nvec vectors of 8 columns; four make a block of 32, and a row that
// ends inside a block is padded to whole blocks in the numbering (lanes of the padding load and store nothing), so the four
// lanes of a block are neighbours.  With D % 32 == 0 nothing is padded and no division is needed.
struct Rows {
    uint32_t total;      // numbered vectors, < 2^31
    uint32_t nvec, nblk;
    FastDiv padded;      // vectors of a row, padding included
};
struct Place {
    bool on;
    size_t vec;          // index of the 8-column vector in BF16 (16 bytes) and q (8 bytes)
    size_t blk;          // index of the scale byte
    uint32_t col;        // vector within the row
};
template <bool RAGGED>
__device__ __forceinline__ Place place(const Rows& r, uint32_t i) {
    Place p;
    if constexpr (RAGGED) {
        const uint32_t row = r.padded.div(i);
        p.col = i - row * r.padded.d;
        p.on = i < r.total && p.col < r.nvec;
        p.vec = size_t(row) * r.nvec + p.col;
        p.blk = size_t(row) * r.nblk + (p.col >> 2);
    } else {
        p.on = i < r.total;
        p.vec = i;
        p.blk = i >> 2;
        p.col = 0;
    }
    return p;
}

constexpr int kThreads = 256;

template <bool RAGGED, int U>
__global__ void __launch_bounds__(kThreads) q8_store_kernel(Rows r, const uint4* x, uint2* q, uint8_t* scale) {
    const uint32_t base = blockIdx.x * (kThreads * U) + threadIdx.x;
    Place p[U];
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        p[u] = place<RAGGED>(r, base + u * kThreads);
        v[u] = p[u].on ? x[p[u].vec] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float f[8];
        unpack8(v[u], f);
        int byte;
        const uint2 o = narrow8(f, byte);
        if (p[u].on) {
            q[p[u].vec] = o;
            if ((threadIdx.x & 3) == 0) scale[p[u].blk] = uint8_t(byte);
        }
    }
}

template <bool RAGGED, int U>
__global__ void __launch_bounds__(kThreads) q8_load_kernel(Rows r, const uint2* __restrict__ q, const uint8_t* __restrict__ scale,
                                                           const uint4* __restrict__ col, FastDiv nvec, uint4* __restrict__ out) {
    const uint32_t base = blockIdx.x * (kThreads * U) + threadIdx.x;
    Place p[U];
    uint2 v[U];
    int b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        p[u] = place<RAGGED>(r, base + u * kThreads);
        v[u] = p[u].on ? q[p[u].vec] : make_uint2(0, 0);
        b[u] = p[u].on ? scale[p[u].blk] : 127;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (!p[u].on) continue;
        float f[8];
        widen8(v[u], b[u], f);
        if (col) {
            const uint32_t c = RAGGED ? p[u].col : uint32_t(p[u].vec) - nvec.div(uint32_t(p[u].vec)) * nvec.d;
            float w[8];
            unpack8(__ldg(col + c), w);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] *= w[e];
        }
        out[p[u].vec] = pack8(f);
    }
}

// 1 / (1 + 2^(-g log2 e)) by the special-function unit: relative error under 8 + 1.5 |g| halves of FP32's step (the product's
// rounding is |g| of them, its constant half as many, ex2 and rcp four each), and at -88 and below, where the sum passes FLT_MAX,
// zero for at most 2^-127.  The results are rounded to BF16's 2^-8 next.  expf and a division instead make the kernels below bound
// by instructions: 448 against 363 us forward, 508 against 465 backward, at 16384 x 18944.
__device__ __forceinline__ float sigmoid(float g) {
    float e, r;
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}

// act = silu(gate) * up; gate and up to 8 bits: 4 bytes an element read, 4 + 1/16 written.  Two vectors a thread: with one the
// loads in flight do not cover the latency (419 us), four cost registers (385 us).
template <bool RAGGED, int U>
__global__ void __launch_bounds__(kThreads) silu_mul_q8_fwd_kernel(Rows r, const uint4* gate, const uint4* up, uint4* act, uint2* gate_q,
                                                                   uint8_t* gate_s, uint2* up_q, uint8_t* up_s) {
    const uint32_t base = blockIdx.x * (kThreads * U) + threadIdx.x;
    Place p[U];
    uint4 g[U], h[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        p[u] = place<RAGGED>(r, base + u * kThreads);
        g[u] = p[u].on ? gate[p[u].vec] : make_uint4(0, 0, 0, 0);
        h[u] = p[u].on ? up[p[u].vec] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float fg[8], fu[8], a[8];
        unpack8(g[u], fg);
        unpack8(h[u], fu);
        int bg, bu;
        const uint2 qg = narrow8(fg, bg), qu = narrow8(fu, bu);
#pragma unroll
        for (int e = 0; e < 8; e++) a[e] = fg[e] * sigmoid(fg[e]) * fu[e];
        if (p[u].on) {
            act[p[u].vec] = pack8(a);
            gate_q[p[u].vec] = qg;
            up_q[p[u].vec] = qu;
            if ((threadIdx.x & 3) == 0) {
                gate_s[p[u].blk] = uint8_t(bg);
                up_s[p[u].blk] = uint8_t(bu);
            }
        }
    }
}

template <bool RAGGED, int U>
__global__ void __launch_bounds__(kThreads) silu_mul_q8_bwd_kernel(Rows r, const uint4* dout, const uint2* __restrict__ gate_q,
                                                                   const uint8_t* __restrict__ gate_s, const uint2* __restrict__ up_q,
                                                                   const uint8_t* __restrict__ up_s, uint4* dgate, uint4* dup, uint4* act) {
    const uint32_t base = blockIdx.x * (kThreads * U) + threadIdx.x;
    Place p[U];
    uint4 d[U];
    uint2 g[U], h[U];
    int bg[U], bu[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        p[u] = place<RAGGED>(r, base + u * kThreads);
        d[u] = p[u].on ? dout[p[u].vec] : make_uint4(0, 0, 0, 0);
        g[u] = p[u].on ? gate_q[p[u].vec] : make_uint2(0, 0);
        h[u] = p[u].on ? up_q[p[u].vec] : make_uint2(0, 0);
        bg[u] = p[u].on ? gate_s[p[u].blk] : 127;
        bu[u] = p[u].on ? up_s[p[u].blk] : 127;
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (!p[u].on) continue;
        float fd[8], fg[8], fu[8], og[8], ou[8], oa[8];
        unpack8(d[u], fd);
        widen8(g[u], bg[u], fg);
        widen8(h[u], bu[u], fu);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float sig = sigmoid(fg[e]), s = fg[e] * sig;
            og[e] = fd[e] * fu[e] * (sig * (1.f + fg[e] * (1.f - sig)));
            ou[e] = fd[e] * s;
            oa[e] = s * fu[e];
        }
        dgate[p[u].vec] = pack8(og);
        dup[p[u].vec] = pack8(ou);
        if (act) act[p[u].vec] = pack8(oa);
    }
}

// ── RMSNorm ─────────────────────────────────────────────────────────────────
// A row belongs to TPR threads (a warp, four of which make a CTA, or a whole CTA), which hold it in registers: one read.  A thread
// has NV vectors of 8 columns, TPR vectors apart, so the four lanes of a block of 32 columns are neighbours.  Many small CTAs: one
// row's barrier and latencies are covered by the other rows on the SM, two or four rows a CTA are slower (67 / 83 us backward at
// 16384 x 3584, a warp a row 100).  All loads of a row stand before its sum, add_to's too (after it: 77 us).
//
// Sum over the threads of a row; every thread gets it.  A warp's sum needs no barrier; a CTA's one.
template <int TPR, typename T>
__device__ __forceinline__ T row_sum(T v, T* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < TPR / 32; w++) v += red[w];
    }
    return v;
}

// r = bf16(x + delta), n = r / rms(r), out = bf16(n * w), (q, scale) = n in 8 bits.  n and not n * w is held: the backward
// needs n, and a gradient over tokens of out = n * w has w as a factor of its columns (ta_gemm_tokens_q8_f32's `col`).
// 1 / rms is formed in 64 bits from sums of eight squares and multiplied as two FP32 parts, the product is cut off and its last bit
// set, so that its conversion to e4m3 and its comparison with 448 * 2^k come out as the unrounded product's: next to a border an
// error of 1e-7 gives another code, or to all 32 of a block another scale.  It costs 2 us of 87 at 16384 x 3584 (81 at the
// copy rate).
template <int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) add_rms_norm_q8_fwd_kernel(const uint4* x, const uint4* delta, const uint4* __restrict__ w,
                                                                                    uint4* res, uint4* out, uint2* q, uint8_t* scale,
                                                                                    float* rms_out, int rows, int D, double inv_d, float eps) {
    __shared__ double red[TPR / 32];
    const int lane = threadIdx.x % TPR;
    const int row = TPR == 32 ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (row >= rows) return;   // a whole warp's, or a whole CTA's
    const int nvec = D / 8, nblk = (D + kQ8Block - 1) / kQ8Block;
    const size_t at = size_t(row) * nvec;
    uint4 v[NV];
    double ss = 0;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = lane + j * TPR;
        v[j] = i < nvec ? x[at + i] : make_uint4(0, 0, 0, 0);
    }
    if (delta) {
        uint4 dv[NV];
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = lane + j * TPR;
            dv[j] = i < nvec ? delta[at + i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = lane + j * TPR;
            float a[8], b[8];
            unpack8(v[j], a);
            unpack8(dv[j], b);
#pragma unroll
            for (int e = 0; e < 8; e++) a[e] += b[e];
            v[j] = pack8(a);
            if (i < nvec) res[at + i] = v[j];
        }
    } else if (res) {
#pragma unroll
        for (int j = 0; j < NV; j++) {
            const int i = lane + j * TPR;
            if (i < nvec) res[at + i] = v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
        float f[8], eight = 0.f;
        unpack8(v[j], f);
#pragma unroll
        for (int e = 0; e < 8; e++) eight += f[e] * f[e];
        ss += double(eight);
    }
    ss = row_sum<TPR>(ss, red);
    const double exact = rsqrt(ss * inv_d + double(eps));
    const float rms = float(exact), rest = exact < double(CUDART_INF_F) ? float(exact - double(rms)) : 0.f;
    if (lane == 0) rms_out[row] = rms;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = lane + j * TPR;
        float f[8];
        unpack8(v[j], f);
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = __uint_as_float(__float_as_uint(__fmaf_rz(f[e], rms, f[e] * rest)) | 1u);
        int byte;
        const uint2 o = narrow8(f, byte);
        if (i < nvec) {
            q[at + i] = o;
            if ((lane & 3) == 0) scale[size_t(row) * nblk + (i >> 2)] = uint8_t(byte);
            if (out) {
                float g[8];
                unpack8(__ldg(w + i), g);
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] *= g[e];
                out[at + i] = pack8(f);
            }
        }
    }
}

// Eight values as four pairs
__device__ __forceinline__ void pairs(const uint4& u, uint64_t (&f)[4]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 t = unpack_bf16x2(w[i]);
        f[i] = pack_f32x2(t.x, t.y);
    }
}
__device__ __forceinline__ void codes(const uint2& q, uint64_t (&f)[4]) {
    float v[8];
    widen4(q.x, 1.f, v);
    widen4(q.y, 1.f, v + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
}

// dx = rms * (w*dy - n * mean(w*dy*n)) (+ add_to), n from 8 bits
// (The second bound 1 has the compiler take 166 registers at eight vectors a thread: 154 us at 8192 columns, with its own 156 160.)
template <int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR, NV == 8 ? 1 : 0) rms_norm_q8_bwd_kernel(const uint4* dy, const uint2* __restrict__ q,
                                                                                const uint8_t* __restrict__ scale, const uint4* __restrict__ w,
                                                                                const float* __restrict__ rms_saved, uint4* dx,
                                                                                const uint4* add_to, int rows, int D) {
    __shared__ float red[TPR / 32];
    const int lane = threadIdx.x % TPR;
    const int row = TPR == 32 ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
    if (row >= rows) return;
    const int nvec = D / 8, nblk = (D + kQ8Block - 1) / kQ8Block;
    const size_t at = size_t(row) * nvec;
    const float rms = rms_saved[row];
    uint4 d[NV], a[NV];
    uint2 n[NV];
    int b[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = lane + j * TPR;
        const bool on = i < nvec;
        d[j] = on ? dy[at + i] : make_uint4(0, 0, 0, 0);
        n[j] = on ? q[at + i] : make_uint2(0, 0);
        b[j] = on ? scale[size_t(row) * nblk + (i >> 2)] : 127;
        a[j] = on && add_to ? add_to[at + i] : make_uint4(0, 0, 0, 0);
    }
    constexpr bool kEarly = NV <= 2;   // the weights before the sum too, while registers allow it: 1 to 2 us
    uint4 wv[kEarly ? NV : 1];
    if constexpr (kEarly) {
#pragma unroll
        for (int j = 0; j < NV; j++) wv[j] = lane + j * TPR < nvec ? __ldg(w + lane + j * TPR) : make_uint4(0, 0, 0, 0);
    }
    // Pairs of columns, two to an instruction (one by one: 43.0 -> 45.3 us at 16384 x 2048, 154 -> 188 at 8192).  n = q * 2^k: the
    // block's power of two is taken once a vector, of the sum and of corr.
    auto weight = [&](int j, uint64_t (&f)[4]) {
        if constexpr (kEarly) pairs(wv[j], f);
        else pairs(__ldg(w + lane + j * TPR), f);
    };
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = lane + j * TPR;
        if (i >= nvec) continue;
        uint64_t fd[4], fq[4], fw[4], acc = 0;
        pairs(d[j], fd);
        codes(n[j], fq);
        weight(j, fw);
#pragma unroll
        for (int e = 0; e < 4; e++) acc = ffma2(fmul2(fd[e], fw[e]), fq[e], acc);
        const float2 t = unpack_f32x2(acc);
        dot += (t.x + t.y) * q8_step(b[j]);
    }
    dot = row_sum<TPR>(dot, red);
    const float corr = dot / float(D);
    const uint64_t rms2 = pack_f32x2(rms, rms);
    // d and n are widened again below: held as pairs they would take twice the registers
#pragma unroll
    for (int j = 0; j < NV; j++) asm volatile("" : "+r"(d[j].x), "+r"(d[j].y), "+r"(d[j].z), "+r"(d[j].w), "+r"(n[j].x), "+r"(n[j].y));
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int i = lane + j * TPR;
        if (i >= nvec) continue;
        uint64_t fd[4], fq[4], fw[4], fa[4];
        pairs(d[j], fd);
        codes(n[j], fq);
        weight(j, fw);
        pairs(a[j], fa);      // zeros without add_to; one rounding to BF16, at the store
        const float c = -corr * q8_step(b[j]);
        const uint64_t c2 = pack_f32x2(c, c);
        uint4 o;
        uint32_t* ow = &o.x;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 t = unpack_f32x2(ffma2(rms2, ffma2(fq[e], c2, fmul2(fd[e], fw[e])), fa[e]));
            ow[e] = pack_bf16x2(t.x, t.y);
        }
        dx[at + i] = o;
    }
}

// Calls launch(Rows, first row) for pieces whose vectors number fewer than 2^30.
template <typename F>
int over_rows(int rows, int D, F launch) {
    Rows r;
    r.nvec = uint32_t(D / 8);
    r.nblk = (uint32_t(D) + kQ8Block - 1) / kQ8Block;
    const uint32_t padded = r.nblk * 4;
    r.padded = FastDiv(padded);
    const int most = std::max(1, int((1u << 30) / padded));
    for (long at = 0; at < rows; at += most) {     // at may pass 2^31
        r.total = uint32_t(std::min(rows - int(at), most)) * padded;
        if (int rc = launch(r, int(at))) return rc;
    }
    return TA_OK;
}
unsigned blocks(uint32_t total, int per_block) { return unsigned((total + per_block - 1) / per_block); }

template <typename T>
T* rows_from(void* p, int row, int per_row) { return static_cast<T*>(p) + size_t(row) * per_row; }
template <typename T>
const T* rows_from(const void* p, int row, int per_row) { return static_cast<const T*>(p) + size_t(row) * per_row; }

bool aligned16(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}
int q8_args(ta_ctx* ctx, const char* what, bool all, int rows, int D, bool aligned) {
    if (!ctx || !all || rows < 0 || D <= 0) return fail(ctx, TA_ERR_INVALID, std::string(what) + ": null argument or bad size");
    if (D % 8) return fail(ctx, TA_ERR_INVALID, std::string(what) + ": D must be a multiple of 8");
    if (!aligned) return fail(ctx, TA_ERR_INVALID, std::string(what) + ": pointers must be 16-byte aligned");
    return on_ctx_device(ctx, what);
}

}  // namespace
}  // namespace ta

using namespace ta;

extern "C" {

int ta_q8_store(ta_ctx* ctx, const void* x, void* q, void* scale, int rows, int D, void* stream) {
    if (int rc = q8_args(ctx, "q8_store", x && q && scale, rows, D, aligned16({x, q}))) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return over_rows(rows, D, [&](const Rows& r, int at) {
        constexpr int U = 4;
        const auto X = rows_from<uint4>(x, at, D / 8);
        const auto Q = rows_from<uint2>(q, at, D / 8);
        const auto S = rows_from<uint8_t>(scale, at, r.nblk);
        if (D % kQ8Block) q8_store_kernel<true, U><<<blocks(r.total, kThreads * U), kThreads, 0, s>>>(r, X, Q, S);
        else              q8_store_kernel<false, U><<<blocks(r.total, kThreads * U), kThreads, 0, s>>>(r, X, Q, S);
        TA_LAUNCH_CHECK(ctx, "q8_store_kernel");
        return TA_OK;
    });
}

int ta_q8_load(ta_ctx* ctx, const void* q, const void* scale, const void* col, void* out, int rows, int D, void* stream) {
    if (int rc = q8_args(ctx, "q8_load", q && scale && out, rows, D, aligned16({q, col, out}))) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return over_rows(rows, D, [&](const Rows& r, int at) {
        constexpr int U = 4;
        const auto Q = rows_from<uint2>(q, at, D / 8);
        const auto S = rows_from<uint8_t>(scale, at, r.nblk);
        const auto O = rows_from<uint4>(out, at, D / 8);
        const auto C = static_cast<const uint4*>(col);
        if (D % kQ8Block) q8_load_kernel<true, U><<<blocks(r.total, kThreads * U), kThreads, 0, s>>>(r, Q, S, C, r.padded, O);
        else              q8_load_kernel<false, U><<<blocks(r.total, kThreads * U), kThreads, 0, s>>>(r, Q, S, C, r.padded, O);
        TA_LAUNCH_CHECK(ctx, "q8_load_kernel");
        return TA_OK;
    });
}

int ta_silu_mul_q8_fwd(ta_ctx* ctx, const void* gate, const void* up, void* out, void* gate_q, void* gate_scale, void* up_q, void* up_scale,
                       int rows, int D, void* stream) {
    if (int rc = q8_args(ctx, "silu_mul_q8_fwd", gate && up && out && gate_q && gate_scale && up_q && up_scale, rows, D,
                         aligned16({gate, up, out, gate_q, up_q})))
        return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return over_rows(rows, D, [&](const Rows& r, int at) {
        constexpr int U = 2;
        const auto G = rows_from<uint4>(gate, at, D / 8), H = rows_from<uint4>(up, at, D / 8);
        const auto O = rows_from<uint4>(out, at, D / 8);
        const auto GQ = rows_from<uint2>(gate_q, at, D / 8), UQ = rows_from<uint2>(up_q, at, D / 8);
        const auto GS = rows_from<uint8_t>(gate_scale, at, r.nblk), US = rows_from<uint8_t>(up_scale, at, r.nblk);
        const unsigned grid = blocks(r.total, kThreads * U);
        if (D % kQ8Block) silu_mul_q8_fwd_kernel<true, U><<<grid, kThreads, 0, s>>>(r, G, H, O, GQ, GS, UQ, US);
        else              silu_mul_q8_fwd_kernel<false, U><<<grid, kThreads, 0, s>>>(r, G, H, O, GQ, GS, UQ, US);
        TA_LAUNCH_CHECK(ctx, "silu_mul_q8_fwd_kernel");
        return TA_OK;
    });
}

int ta_silu_mul_q8_bwd(ta_ctx* ctx, const void* dout, const void* gate_q, const void* gate_scale, const void* up_q, const void* up_scale,
                       void* dgate, void* dup, void* act, int rows, int D, void* stream) {
    if (int rc = q8_args(ctx, "silu_mul_q8_bwd", dout && gate_q && gate_scale && up_q && up_scale && dgate && dup, rows, D,
                         aligned16({dout, gate_q, up_q, dgate, dup, act})))
        return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return over_rows(rows, D, [&](const Rows& r, int at) {
        constexpr int U = 2;
        const auto DO = rows_from<uint4>(dout, at, D / 8);
        const auto GQ = rows_from<uint2>(gate_q, at, D / 8), UQ = rows_from<uint2>(up_q, at, D / 8);
        const auto GS = rows_from<uint8_t>(gate_scale, at, r.nblk), US = rows_from<uint8_t>(up_scale, at, r.nblk);
        const auto DG = rows_from<uint4>(dgate, at, D / 8), DU = rows_from<uint4>(dup, at, D / 8);
        const auto A = act ? rows_from<uint4>(act, at, D / 8) : nullptr;
        const unsigned grid = blocks(r.total, kThreads * U);
        if (D % kQ8Block) silu_mul_q8_bwd_kernel<true, U><<<grid, kThreads, 0, s>>>(r, DO, GQ, GS, UQ, US, DG, DU, A);
        else              silu_mul_q8_bwd_kernel<false, U><<<grid, kThreads, 0, s>>>(r, DO, GQ, GS, UQ, US, DG, DU, A);
        TA_LAUNCH_CHECK(ctx, "silu_mul_q8_bwd_kernel");
        return TA_OK;
    });
}

// Threads a row and vectors a thread by the row's length, each the fastest of those measured on 16384 rows (us a call, L2 cold; in
// parentheses the next best).  Forward: 64 x 2 to 1024 columns 30.7, 96 x 2 at 1536 41.0 (128 x 2 43.0), 128 x 2 to 2048 53, 128 x
// 3 at 2560 65.6 (192 x 2 69.6, 128 x 4 71), 128 x 4 at 3584 86 (256 x 2 as much), 256 x 3 at 5120 125 (384 x 2 135, 256 x 4 141),
// 256 x 4 to 8192 186 (128 x 8 188).  Backward, which holds three arrays: 64 x 2 to 1024 24.6, 96 x 2 at 1536 32.8 (128 x 2 34.8),
// 128 x 2 to 2048 43, 192 x 2 at 2560 55 (128 x 3 57, 256 x 2 59), 256 x 2 at 3584 70 (128 x 4 80), 384 x 2 at 5120 106 (256 x 3
// 110, 128 x 8 119), 128 x 8 to 8192 154 (256 x 4 172, 512 x 2 184), 512 x 4 to 16384 389 (256 x 8 516).  As many warps as a row
// needs, a number known at launch, costs the constant offsets: 28.6 at 1024, 80 at 3584.
// Few rows, up to four an SM, leave most of the device idle and are bound by a row's own latency: more threads a row then (us,
// forward / backward, from L2: 1 x 896 1.7 / 1.5, with the others 2.1 / 1.6; 256 x 3584 2.9 / 2.8, 3.8 / 3.3; 64 x 8192 3.2 / 2.8, 3.8 /
// 4.5; 592 x 8192 11.3 / 10.0, 9.6 / 14.3; beyond, at 1024 x 3584, 8.8 / 7.0, 7.8 / 8.7).
#define TA_NORM_CASES(LAUNCH, AT_384, AT_512, AT_768, AT_1024, AT_2048)                 \
    do {                                                                                \
        const int nvec = D / 8;                                                         \
        const bool few = rows <= 4 * ctx->sm_count;                                     \
        if (nvec <= 32)        LAUNCH(32, 1);                                           \
        else if (nvec <= 64)   LAUNCH(32, 2);                                           \
        else if (nvec <= 128)  { if (few) LAUNCH(128, 1); else LAUNCH(64, 2); }         \
        else if (nvec <= 192)  { if (few) LAUNCH(256, 1); else LAUNCH(96, 2); }         \
        else if (nvec <= 256)  { if (few) LAUNCH(256, 1); else LAUNCH(128, 2); }        \
        else if (nvec <= 384)  { if (few) LAUNCH(512, 1); else LAUNCH AT_384; }         \
        else if (nvec <= 512)  { if (few) LAUNCH(512, 1); else LAUNCH AT_512; }         \
        else if (nvec <= 768)  { if (few) LAUNCH(512, 2); else LAUNCH AT_768; }         \
        else if (nvec <= 1024) { if (few) LAUNCH(512, 2); else LAUNCH AT_1024; }        \
        else                   { if (few) LAUNCH(512, 4); else LAUNCH AT_2048; }        \
    } while (0)

int ta_add_rms_norm_q8_fwd(ta_ctx* ctx, const void* x, const void* delta, const void* w, void* res_out, void* out, void* q, void* scale,
                           float* rms_out, int rows, int D, float eps, void* stream) {
    if (int rc = q8_args(ctx, "add_rms_norm_q8_fwd", x && w && q && scale && rms_out && (res_out || !delta), rows, D,
                         aligned16({x, delta, w, res_out, out, q})))
        return rc;
    if (D > 16384) return fail(ctx, TA_ERR_INVALID, "add_rms_norm_q8_fwd: D must be a multiple of 8 and <= 16384");
    if (reinterpret_cast<uintptr_t>(rms_out) & 3) return fail(ctx, TA_ERR_INVALID, "add_rms_norm_q8_fwd: rms_out must be 4-byte aligned");
    if (rows == 0) return TA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto X = static_cast<const uint4*>(x), De = static_cast<const uint4*>(delta), W = static_cast<const uint4*>(w);
    const auto R = static_cast<uint4*>(res_out), O = static_cast<uint4*>(out);
    const auto Q = static_cast<uint2*>(q);
    const auto S = static_cast<uint8_t*>(scale);
#define TA_LAUNCH(TPR, NV) \
    add_rms_norm_q8_fwd_kernel<TPR, NV><<<TPR == 32 ? (rows - 1) / 4 + 1 : rows, TPR == 32 ? 128 : TPR, 0, s>>>(X, De, W, R, O, Q, S, rms_out, rows, D, 1.0 / D, eps)
    TA_NORM_CASES(TA_LAUNCH, (128, 3), (128, 4), (256, 3), (256, 4), (256, 8));
#undef TA_LAUNCH
    TA_LAUNCH_CHECK(ctx, "add_rms_norm_q8_fwd_kernel");
    return TA_OK;
}

int ta_rms_norm_q8_bwd(ta_ctx* ctx, const void* dy, const void* q, const void* scale, const void* w, const float* rms_saved, void* dx,
                       const void* add_to, int rows, int D, void* stream) {
    if (int rc = q8_args(ctx, "rms_norm_q8_bwd", dy && q && scale && w && rms_saved && dx, rows, D, aligned16({dy, q, w, dx, add_to}))) return rc;
    if (D > 16384) return fail(ctx, TA_ERR_INVALID, "rms_norm_q8_bwd: D must be a multiple of 8 and <= 16384");
    if (reinterpret_cast<uintptr_t>(rms_saved) & 3) return fail(ctx, TA_ERR_INVALID, "rms_norm_q8_bwd: rms_saved must be 4-byte aligned");
    if (rows == 0) return TA_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto DY = static_cast<const uint4*>(dy), W = static_cast<const uint4*>(w), AT = static_cast<const uint4*>(add_to);
    const auto Q = static_cast<const uint2*>(q);
    const auto S = static_cast<const uint8_t*>(scale);
    const auto DX = static_cast<uint4*>(dx);
#define TA_LAUNCH(TPR, NV) \
    rms_norm_q8_bwd_kernel<TPR, NV><<<TPR == 32 ? (rows - 1) / 4 + 1 : rows, TPR == 32 ? 128 : TPR, 0, s>>>(DY, Q, S, W, rms_saved, DX, AT, rows, D)
    TA_NORM_CASES(TA_LAUNCH, (192, 2), (256, 2), (384, 2), (128, 8), (512, 4));
#undef TA_LAUNCH
    TA_LAUNCH_CHECK(ctx, "rms_norm_q8_bwd_kernel");
    return TA_OK;
}

}  // extern "C"
