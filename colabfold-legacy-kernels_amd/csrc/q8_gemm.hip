// 8-bit matrix product for gfx950 (CDNA4): out[m,n] = round16((sum_k q[m,k] w[n,k]) sx[m] sw[n] + b[n] +
// residual[m,n]), the integer sum exact in 32 bits. No counterpart in the reference; it stands beside
// output_projection and reads the 8-bit rows of rows8.hip.
//
// The products are v_mfma_i32_16x16x64_i8 with the weights as A operand (rows of D are channels) and the
// activations as B, so a lane holds four consecutive D rows of one activation row. Weights come in blocks
// of 64 channels by 64 inputs, laid out so that
//   - one MFMA operand (16 channels, 64 inputs) is 1024 contiguous bytes in lane order, and
//   - D row 4 g + i of the block's operand b is channel 16 g + 4 b + i: the four operands of a block give a
//     lane 16 consecutive channels, 32 bytes of its output row.
// Both operands' rows are padded with zeros to multiples of 64, so there is no tail in k and none in the
// weights' channels; rows past M read as zeros (the buffer's range) and are not stored.
#include "clk_common.h"

#include <algorithm>

namespace clk {

namespace {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef half8 half8u __attribute__((aligned(2)));
typedef half4 half4u __attribute__((aligned(2)));

// D[16x16] += A[16x64] B[64x16] in int32: lane l supplies A row and B column l % 16, inputs 16 (l / 16) .. + 15,
// and holds D rows 4 (l / 16) .. + 3 of column l % 16.
__device__ __forceinline__ int4v mfma_i8(int4v a, int4v b, int4v c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

struct GemmArgs {
    const int8_t* q;
    const float* qs;
    const int8_t* wq;
    const float* ws;
    const float* b;          // null: none
    const half_t* residual;  // null: none
    half_t* out;
    int M, N, Kp;
    int mtiles, ntiles;
    FastDiv mdiv;
};

template <typename P>
__device__ __forceinline__ auto rsrc_of(const P* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<P*>(p), 0, bytes, 0x00020000);
}
template <typename Rsrc>
__device__ __forceinline__ int4v load16(Rsrc r, uint32_t off) {
    return __builtin_bit_cast(int4v, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// A sum with its scales and bias (0: none), in one order of roundings for every kernel, so that a row's
// results do not depend on how many rows a call has
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float b) { return __builtin_fmaf((float)sum * sx, sw, b); }

// Four consecutive channels n .. n + 3 of row m, of which those below N exist
template <bool BF>
__device__ __forceinline__ void store4(const GemmArgs& a, int m, int n, int4v acc) {
    if (m >= a.M || n >= a.N) return;
    const float sx = a.qs[m];
    const int64_t at = (int64_t)m * a.N + n;
    if (n + 4 <= a.N) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = scaled(acc[i], sx, a.ws[n + i], a.b != nullptr ? a.b[n + i] : 0.f);
        if (a.residual != nullptr) {
            const half4 h = *reinterpret_cast<const half4u*>(a.residual + at);
            const half8 r = half8{h[0], h[1], h[2], h[3], 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += act_get<BF>(r, i);
        }
        *reinterpret_cast<half4u*>(a.out + at) = half4{act_cvt<BF>(v[0]), act_cvt<BF>(v[1]), act_cvt<BF>(v[2]), act_cvt<BF>(v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n + i >= a.N) break;
            float v = scaled(acc[i], sx, a.ws[n + i], a.b != nullptr ? a.b[n + i] : 0.f);
            if (a.residual != nullptr) v += act_get<BF>(half8{a.residual[at + i]}, 0);
            a.out[at + i] = act_cvt<BF>(v);
        }
    }
}

// A workgroup computes 64 rows by 64 channels; its four waves split k and join their sums through LDS.
// Operands go from memory straight to registers.
template <bool BF>
__global__ __launch_bounds__(256) void q8_gemm_kernel(GemmArgs a) {
    __shared__ __attribute__((aligned(16))) int4v part[4][16][kWave];
    const int item = xcd_item(blockIdx.x, gridDim.x);
    const int nt = fdiv(item, a.mdiv), mt = item - nt * a.mtiles;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4;
    const int m0 = 64 * mt, rows = min(64, a.M - m0), kbs = a.Kp / 64;
    const auto rw = rsrc_of(a.wq + (int64_t)nt * 64 * a.Kp, (uint32_t)(64 * a.Kp));
    const auto rx = rsrc_of(a.q + (int64_t)m0 * a.Kp, (uint32_t)(rows * a.Kp));
    int4v acc[4][4];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) acc[b][mb] = int4v{0, 0, 0, 0};
    for (int kb = wave; kb < kbs; kb += 4) {
        int4v w[4], x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) w[b] = load16(rw, (uint32_t)(4096 * kb + 1024 * b + 16 * lane));
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) x[mb] = load16(rx, (uint32_t)((16 * mb + r16) * a.Kp + 64 * kb + 16 * g));
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int mb = 0; mb < 4; ++mb) acc[b][mb] = mfma_i8(w[b], x[mb], acc[b][mb]);
    }
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int mb = 0; mb < 4; ++mb) part[wave][4 * b + mb][lane] = acc[b][mb];
    __syncthreads();
#pragma unroll
    for (int b = 0; b < 4; ++b) {  // wave w finishes rows 16 w .. + 15
        int4v s = part[0][4 * b + wave][lane];
#pragma unroll
        for (int v = 1; v < 4; ++v) s += part[v][4 * b + wave][lane];
        store4<BF>(a, m0 + 16 * wave + r16, 64 * nt + 16 * g + 4 * b, s);
    }
}

// Large products. A workgroup computes BM = 16 MF WM rows by BN = 64 NB WN channels; wave (wm, wn) of WM x WN
// has MF operands of 16 rows and NB weight blocks of 64 channels. Both operands go through LDS, 128 inputs
// (two MFMA steps) a stage, two stages: the loads of the next stage are in flight while one is computed.
//   weights  by 1024-byte direct-to-LDS loads, in memory order: an operand read is 64 lanes' consecutive 16
//            bytes
//   rows     eight rows of 128 bytes a load, position p of row r holding its 16-byte chunk p ^ (r / 2 % 8): a
//            16-lane group reads one chunk of 16 rows from 16 different bank quadruples
template <bool BF, int MF, int NB, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void q8_tile_kernel(GemmArgs a) {
    constexpr int WAVES = WM * WN, BM = 16 * MF * WM, NBLK = NB * WN;
    constexpr int XS = BM * 128, WS = NBLK * 8192;
    __shared__ __attribute__((aligned(1024))) char lds[2 * (XS + WS)];
    const int item = xcd_item(blockIdx.x, gridDim.x);
    // groups of four row tiles, in a group row tiles fastest: what an XCD runs at a time is a patch of the
    // result, whose operands its L2 holds
    const int per = 4 * a.ntiles, grp = item / per, in = item - grp * per;
    const int gm = min(4, a.mtiles - 4 * grp), nt = in / gm, mt = 4 * grp + in - nt * gm;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4, wm = wave % WM, wn = wave / WM;
    const int m0 = BM * mt, rows = min(BM, a.M - m0), Kp = a.Kp, kbs = Kp / 64;
    const int nb0 = NBLK * nt, nblks = min(NBLK, (a.N + 63) / 64 - nb0);
    const auto rx = rsrc_of(a.q + (int64_t)m0 * Kp, (uint32_t)(rows * Kp));
    const auto rw = rsrc_of(a.wq + (int64_t)nb0 * 64 * Kp, (uint32_t)(nblks * 64 * Kp));

    constexpr int XL = BM / 8 / WAVES, WL = NBLK * 8 / WAVES;  // loads a wave a stage
    uint32_t xoff[XL], woff[WL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = 8 * (XL * wave + i) + (lane >> 3);
        xoff[i] = (uint32_t)(r * Kp + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int u = WL * wave + i;  // block u / 8, its step u / 4 % 2, operand u % 4
        woff[i] = (uint32_t)((u >> 3) * 64 * Kp + (u & 7) * 1024 + 16 * lane);
    }
    const auto fetch = [&](int st, int buf) __attribute__((always_inline)) {
        char* base = lds + buf * (XS + WS);
#pragma unroll
        for (int i = 0; i < XL; ++i) dma_lds<16>(rx, base + 1024 * (XL * wave + i), xoff[i] + 128u * st);
#pragma unroll
        for (int i = 0; i < WL; ++i) dma_lds<16>(rw, base + XS + 1024 * (WL * wave + i), woff[i] + 8192u * st);
    };
    int4v acc[NB][4][MF];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int mf = 0; mf < MF; ++mf) acc[nb][b][mf] = int4v{0, 0, 0, 0};

    const int xrow = 16 * MF * wm + r16;  // operand mf of this lane: row xrow + 16 mf
    struct Operands {
        int4v x[MF], w[NB][4];
    };
    const auto read = [&](int kb, int buf, Operands& o) __attribute__((always_inline)) {
        const char* X = lds + buf * (XS + WS);
        const char* W = X + XS;
#pragma unroll
        for (int mf = 0; mf < MF; ++mf) {
            o.x[mf] = *reinterpret_cast<const int4v*>(X + (xrow + 16 * mf) * 128 + 16 * ((4 * kb + g) ^ ((r16 >> 1) & 7)));
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                o.w[nb][b] = *reinterpret_cast<const int4v*>(W + (((wn * NB + nb) * 2 + kb) * 4 + b) * 1024 + 16 * lane);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](const Operands& o) __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int mf = 0; mf < MF; ++mf) acc[nb][b][mf] = mfma_i8(o.w[nb][b], o.x[mf], acc[nb][b][mf]);
        __builtin_amdgcn_sched_barrier(0);
    };
    // The operands of a step are read while the step before it is multiplied, and the barrier stands between the
    // two steps of a stage: past it every wave holds its second step's operands, so the stage's buffer takes
    // the loads of the stage after next, and the next stage's loads have landed.
    const int stages = (kbs + 1) / 2;
    Operands even, odd;
    fetch(0, 0);
    if (stages > 1) {
        fetch(1, 1);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(XL + WL) : "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
    read(0, 0, even);
    for (int st = 0; st + 1 < stages; ++st) {
        read(1, st & 1, odd);
        multiply(even);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (st + 2 < stages) fetch(st + 2, st & 1);
        read(0, (st + 1) & 1, even);
        multiply(odd);
    }
    if (kbs % 2 == 0) read(1, (stages - 1) & 1, odd);
    multiply(even);
    if (kbs % 2 == 0) multiply(odd);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int n = 64 * (nb0 + wn * NB + nb) + 16 * g;
        float sw[16], bv[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sw[i] = n + i < a.N ? a.ws[n + i] : 0.f;
            bv[i] = a.b != nullptr && n + i < a.N ? a.b[n + i] : 0.f;
        }
#pragma unroll
        for (int mf = 0; mf < MF; ++mf) {
            const int m = m0 + xrow + 16 * mf;
            if (m >= a.M) continue;
            const float sx = a.qs[m];
            const int64_t at = (int64_t)m * a.N + n;
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = scaled(acc[nb][i >> 2][mf][i & 3], sx, sw[i], bv[i]);
            if (n + 16 <= a.N) {
                if (a.residual != nullptr) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const half8 r = *reinterpret_cast<const half8u*>(a.residual + at + 8 * h);
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[8 * h + i] += act_get<BF>(r, i);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    half8 o;
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = act_cvt<BF>(v[8 * h + i]);
                    *reinterpret_cast<half8u*>(a.out + at + 8 * h) = o;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (n + i >= a.N) break;
                    if (a.residual != nullptr) v[i] += act_get<BF>(half8{a.residual[at + i]}, 0);
                    a.out[at + i] = act_cvt<BF>(v[i]);
                }
            }
        }
    }
}

// |sum| <= 128^2 Kp has to stay below 2^31
constexpr int64_t kMaxKp = 131008;

}  // namespace

}  // namespace clk

using namespace clk;

extern "C" int clk_q8_projection(clk_stream stream, const clk_buffer* q, const clk_buffer* q_scale,
                                 const clk_buffer* wq, const clk_buffer* w_scale, const clk_buffer* b,
                                 const clk_buffer* residual, const clk_buffer* out, int32_t has_b,
                                 int32_t has_residual) {
    const int act = out != nullptr && out->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {q, q_scale, wq, w_scale, b, residual, out};
    const int types[] = {CLK_S8, CLK_F32, CLK_S8, CLK_F32, CLK_F32, act, act};
    if (int st = check_types("q8_projection", bufs, types, 7)) return st;
    if (q->rank != 2 || out->rank != 2) return invalid("q8_projection: q must be [M,Kp] and out [M,N]");
    const int64_t M = q->dims[0], Kp = q->dims[1], N = out->dims[1];
    if (out->dims[0] != M || M < 0 || N < 0) return invalid("q8_projection: q must be [M,Kp] and out [M,N]");
    if (Kp < 64 || Kp % 64 != 0 || Kp > kMaxKp) {
        return invalid("q8_projection: Kp must be a multiple of 64 from 64 to " + std::to_string(kMaxKp));
    }
    const int64_t nt = (N + 63) / 64;
    if (wq->rank != 6 || wq->dims[0] != nt || wq->dims[1] != Kp / 64 || wq->dims[2] != 4 || wq->dims[3] != 4 ||
        wq->dims[4] != 16 || wq->dims[5] != 16) {
        return invalid("q8_projection: wq must be [ceil(N/64), Kp/64, 4, 4, 16, 16]");
    }
    if (elements(q_scale) != M) return invalid("q8_projection: q_scale must be [M]");
    if (elements(w_scale) != N || (has_b && elements(b) != N)) return invalid("q8_projection: w_scale and b must be [N]");
    if (has_residual && !same_shape(residual, out)) return invalid("q8_projection: residual must be like out");
    if (M == 0 || N == 0) return ok();
    const int64_t mt = (M + 63) / 64;
    if (M > INT32_MAX || N > INT32_MAX - 64 || mt * nt > INT32_MAX / 256) return invalid("q8_projection: too large");
    if (!aligned16(q->data) || !aligned16(wq->data)) return invalid("q8_projection: q and wq must be 16-byte aligned");
    GemmArgs a{static_cast<const int8_t*>(q->data), static_cast<const float*>(q_scale->data),
               static_cast<const int8_t*>(wq->data), static_cast<const float*>(w_scale->data),
               has_b ? static_cast<const float*>(b->data) : nullptr,
               has_residual ? static_cast<const half_t*>(residual->data) : nullptr, static_cast<half_t*>(out->data),
               (int)M, (int)N, (int)Kp, (int)mt, (int)nt, fast_div(mt)};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    if (M >= 256 && N >= 256) {
        a.mtiles = (int)((M + 255) / 256);
        a.ntiles = (int)((N + 255) / 256);
        const dim3 grid((unsigned)(a.mtiles * a.ntiles)), block(512);
        if (act == CLK_BF16) hipLaunchKernelGGL((q8_tile_kernel<true, 4, 2, 4, 2>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((q8_tile_kernel<false, 4, 2, 4, 2>), grid, block, 0, s, a);
        stage_mark(s, 1);
        return launch_status("q8_projection");
    }
    if (act == CLK_BF16) hipLaunchKernelGGL(q8_gemm_kernel<true>, dim3((unsigned)(mt * nt)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(q8_gemm_kernel<false>, dim3((unsigned)(mt * nt)), dim3(256), 0, s, a);
    stage_mark(s, 1);
    return launch_status("q8_projection");
}
