// RMS norm and 8-bit rows for gfx950 (CDNA4). No counterpart in the reference; they stand beside its
// LayerNorm and feed the 8-bit matrix product (q8_gemm.hip).
//
//   rms_norm        s = round16(x + residual), y = round16(s r w), r = 1 / sqrt(mean(s^2) + eps)
//   rms_norm_q8     t = s w, a = max |t|; q = 127 t / a to the nearest, scale = a r / 127: r cancels in q, so
//                   the integers depend on s and w alone
//   rms_norm_bwd    g = dy w, xh = s r: ds = r (g - xh mean(g xh)) + dsum, dw = sum over rows of dy xh
//   quantize_rows   h = x, relu(x) or swish(x[:, :K]) x[:, K:]; q = 127 h / a to the nearest, scale = a / 127
//   dequantize_rows out = q scale
//
// All of them are bound by memory: each value is read once and written once, statistics and products
// are fp32, and results are rounded once.
#include "rows8_dev.h"

#include <algorithm>
#include <type_traits>

namespace clk {

namespace {

typedef half8 half8u __attribute__((aligned(2)));
typedef half_t half_u __attribute__((aligned(2)));
typedef float8v float8u __attribute__((aligned(4)));
typedef float4v float4u __attribute__((aligned(4)));

// A row's sum and maxima over its TPR threads: its lane group, or (TPR > 64) the block's waves through LDS. `slots`
// is one of two sets that alternate, so that one barrier a call is enough: a wave that writes a set again
// has passed the barrier of the call between, which every reader of the set reached after its reads.
struct Stats {
    float sum;
    uint32_t max0, max1;
};
template <int TPR>
struct RowShare {
    Stats slots[2][TPR > kWave ? TPR / kWave : 1];
};
template <int TPR>
__device__ __forceinline__ Stats row_all(Stats s, RowShare<TPR>& share, int& turn) {
    constexpr int W = TPR < kWave ? TPR : kWave;
    s.sum = lanes_sum<W>(s.sum);
    s.max0 = lanes_max<W>(s.max0);
    s.max1 = lanes_max<W>(s.max1);
    if constexpr (TPR > kWave) {
        Stats* slot = share.slots[turn];
        turn ^= 1;
        if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = s;
        __syncthreads();
        s = slot[0];
#pragma unroll
        for (int i = 1; i < TPR / kWave; ++i) {
            s.sum += slot[i].sum;
            s.max0 = max(s.max0, slot[i].max0);
            s.max1 = max(s.max1, slot[i].max1);
        }
    }
    return s;
}

// Rows are split in chunks of 8 values. Widths and addresses are any, so a chunk is one 16-byte access of 2-byte
// alignment: the hardware takes any, and only rows on odd multiples of 2 bytes lose by it (norm of [8192, 8191] in
// bf16 with the residual 124 us, of [8192, 8190] 99, of [8192, 8192] 96). Accesses by pairs or single values,
// which need no alignment, were slower.
//
// A chunk that the width cuts, and one past it, is loaded from the row's last 8 values and shifted down in its
// registers, so that every lane's loads are issued without a branch before any is waited for (a branch
// of its own for the cut chunk made its wave, and at the barrier the row, wait for it: gradients of [8192,
// 8190] 177 us against 108). Rows of less than 8 values are read one by one.
__device__ __forceinline__ half8 load8(const half_t* row, int col, int C) {
    if (C >= 8) return *reinterpret_cast<const half8u*>(row + min(col, C - 8));
    half8 v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < C) v[e] = row[col + e];
    return v;
}
// what load8 gave as the values col .. col + 7, zeros past C
__device__ __forceinline__ half8 cut8(half8 v, int col, int C) {
    const int over = col + 8 - C;  // values past the end
    if (C >= 8 && over > 0) {
        typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
        u64x2 w = __builtin_bit_cast(u64x2, v);
        if (over & 4) w = u64x2{w[1], 0};
        const int bits = 16 * (over & 3);
        if (bits > 0) w = u64x2{w[0] >> bits | w[1] << (64 - bits), w[1] >> bits};
        v = over >= 8 ? half8{} : __builtin_bit_cast(half8, w);
    }
    return v;
}
// a + b, each rounded: as a whole vector, since bf16 values past 2^121 came out times 16 where the sums were put into a half
// vector one by one
template <bool BF>
__device__ __forceinline__ half8 sum8(half8 a, half8 b) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = act_get<BF>(a, e) + act_get<BF>(b, e);
    return __builtin_bit_cast(half8, act_cvt8<BF>(f));
}
template <bool NT = false>
__device__ __forceinline__ void store8(half_t* row, int col, int C, half8 v) {
    if (col + 8 <= C) {
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<half8u*>(row + col));
        else *reinterpret_cast<half8u*>(row + col) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < C) row[col + e] = v[e];
    }
}
__device__ __forceinline__ float8v load8f(const float* row, int col, int C) {
    if (col + 8 <= C) return *reinterpret_cast<const float8u*>(row + col);
    float8v v = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + e < C) v[e] = row[col + e];
    return v;
}
template <bool NT>
__device__ __forceinline__ void store4f(float* to, int n, float4v v) {
    if (n >= 4) {
        if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<float4u*>(to));
        else *reinterpret_cast<float4u*>(to) = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < n) to[e] = v[e];
    }
}
// Sum and maximum over the threads of a block, for the kernels that take a row of any length.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* slot) {
    v = lanes_sum<kWave>(v);
    if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) s += slot[i];
    __syncthreads();
    return s;
}
template <int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slot) {
    v = lanes_max<kWave>(v);
    if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
    __syncthreads();
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) s = max(s, slot[i]);
    __syncthreads();
    return s;
}

// ---- RMS norm -----------------------------------------------------------------------------

struct RmsArgs {
    const half_t* x;
    const half_t* residual;
    const float* w;
    half_t* sum;
    half_t* out;     // 16-bit results
    int8_t* q;       // or 8-bit rows
    float* stat;     // rstd (may be null), or the 8-bit rows' scales
    int64_t M, C, Kp;
    float inv_c, eps;
};

constexpr int kAny = 1024;  // threads of the kernels for rows of any length

// Rows of any length (past 16384 values): a block a row, two passes over it (the second from cache where it fits).
// [1024, 40000] bf16 with the residual 73 us (328 MB, 4.5 TB/s), as 8-bit rows 70; [4096, 20000] 149 and 155, where
// 1024 threads with 4 chunks of a row in registers take 222 and 536 (they spill).
template <bool BF, bool RES, bool Q8>
__global__ __launch_bounds__(kAny) void rms_norm_any_kernel(RmsArgs a) {
    __shared__ float fslot[kAny / kWave];
    __shared__ uint32_t uslot[kAny / kWave];
    const int C = (int)a.C, Kp = (int)a.Kp, first = 8 * threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const half_t* xr = a.x + row * a.C;
        const half_t* rr = a.residual + row * a.C;
        half_t* sr = a.sum + row * a.C;
        const half_t* vr = RES ? sr : xr;  // each thread reads back only what it wrote
        float ss = 0.f;
        uint32_t m = 0, mt = 0;
        const auto collect = [&](int c, half8 v, float d) __attribute__((always_inline)) {
            float8v w = {};
            if constexpr (Q8) w = load8f(a.w, c, C);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = act_get<BF>(v, e) * d;
                ss += f * f;
                m = max(m, abs_bits(f));
                if constexpr (Q8) mt = max(mt, abs_bits(f * w[e]));
            }
        };
        for (int c = first; c < C; c += 8 * kAny) {
            half8 v = cut8(load8(xr, c, C), c, C);
            if constexpr (RES) {
                const half8 r = cut8(load8(rr, c, C), c, C);
                v = sum8<BF>(v, r);
                store8(sr, c, C, v);
            }
            collect(c, v, 1.f);
        }
        ss = block_sum<kAny>(ss, fslot);
        m = block_max<kAny>(m, uslot);
        const float d = BF ? row_shift(m, a.eps) : 1.f;
        const uint32_t plain = mt;
        if (d != 1.f) {
            ss = 0.f;
            mt = 0;
            for (int c = first; c < C; c += 8 * kAny) collect(c, cut8(load8(vr, c, C), c, C), d);
            ss = block_sum<kAny>(ss, fslot);
        }
        const float r = inv_rms(ss, a.inv_c, a.eps * d * d);
        if constexpr (Q8) {
            mt = block_max<kAny>(mt, uslot);
            float dt = d, top, inv, scale;
            if (as_they_are(d, mt)) {
                dt = 1.f;
                mt = block_max<kAny>(plain, uslot);
            }
            row_scale(mt, r, top, inv, scale);
            if (threadIdx.x == 0) a.stat[row] = dt == d ? scale : scale * d;
            for (int c = first; c < Kp; c += 8 * kAny) {
                const half8 v = cut8(load8(vr, c, C), c, C);
                const float8v w = load8f(a.w, c, C);
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = act_get<BF>(v, e) * dt * w[e];
                *reinterpret_cast<uint2v*>(a.q + row * a.Kp + c) = quant8<false>(t, top, inv);
            }
        } else {
            if (threadIdx.x == 0 && a.stat != nullptr) a.stat[row] = r * d;
            for (int c = first; c < C; c += 8 * kAny) {
                const half8 v = cut8(load8(vr, c, C), c, C);
                const float8v w = load8f(a.w, c, C);
                act8<BF> o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (act_t<BF>)(act_get<BF>(v, e) * d * r * w[e]);
                store8(a.out + row * a.C, c, C, raw_act(o));
            }
        }
    }
}

// Rows of up to 8 TPR NCH values, held in registers: TPR threads a row, NCH chunks each, one pass over memory,
// which bounds it. [16384, 8192] bf16 with the residual: 176 us (1.07 GB, 6.1 TB/s); [147456, 128] fp16: 13.8 us
// (5.5 TB/s); 8-bit rows of [4099, 5120] bf16 with the residual: 28 us (5.2 TB/s).
constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

template <bool BF, int TPR, int NCH, bool RES, bool Q8>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_kernel(RmsArgs a) {
    constexpr int ROWS = block_of(TPR) / TPR;
    __shared__ RowShare<TPR> share;
    const int part = threadIdx.x % TPR, sub = threadIdx.x / TPR, C = (int)a.C, Kp = (int)a.Kp;
    int turn = 0;
    float8v w[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) w[j] = load8f(a.w, 8 * (part + TPR * j), C);
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + sub;
        const bool in = ROWS == 1 || row < a.M;
        const int64_t from = ROWS == 1 ? row : min(row, a.M - 1);  // a row past M reads the last one and stores nothing
        const int len = in ? C : 0;
        half8 v[NCH], res[NCH];
#pragma unroll
        for (int j = 0; j < NCH; ++j) v[j] = load8(a.x + from * C, 8 * (part + TPR * j), C);
        if constexpr (RES) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) res[j] = load8(a.residual + from * C, 8 * (part + TPR * j), C);
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                v[j] = cut8(v[j], 8 * (part + TPR * j), C);
                res[j] = cut8(res[j], 8 * (part + TPR * j), C);
                v[j] = sum8<BF>(v[j], res[j]);
                store8(a.sum + row * C, 8 * (part + TPR * j), len, v[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NCH; ++j) v[j] = cut8(v[j], 8 * (part + TPR * j), C);
        }
        Stats s{0.f, 0, 0};
        const auto collect = [&](float d) __attribute__((always_inline)) {
            s = Stats{0.f, 0, 0};
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = act_get<BF>(v[j], e) * d;
                    s.sum += f * f;
                    if constexpr (BF) s.max0 = max(s.max0, abs_bits(f));
                    if constexpr (Q8) s.max1 = max(s.max1, abs_bits(f * w[j][e]));
                }
            s = row_all<TPR>(s, share, turn);
        };
        collect(1.f);
        float d = 1.f, dt = 1.f;  // of the squares and results, of the products that go to 8 bits
        if constexpr (BF) {
            d = row_shift(s.max0, a.eps);
            if (d != 1.f) {
                const uint32_t plain = s.max1;
                collect(d);
                dt = d;
                if (Q8 && as_they_are(d, s.max1)) {
                    dt = 1.f;
                    s.max1 = plain;
                }
            }
        }
        const float r = inv_rms(s.sum, a.inv_c, a.eps * d * d);
        if constexpr (Q8) {
            float top, inv, scale;
            row_scale(s.max1, r, top, inv, scale);
            if (part == 0 && in) a.stat[row] = dt == d ? scale : scale * d;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int col = 8 * (part + TPR * j);
                float t[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = act_get<BF>(v[j], e) * dt * w[j][e];
                if (in && col < Kp) *reinterpret_cast<uint2v*>(a.q + row * Kp + col) = quant8<false>(t, top, inv);
            }
        } else {
            if (part == 0 && in && a.stat != nullptr) a.stat[row] = r * d;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                act8<BF> o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (act_t<BF>)(act_get<BF>(v[j], e) * d * r * w[j][e]);
                store8(a.out + row * C, 8 * (part + TPR * j), len, raw_act(o));
            }
        }
    }
}

// ---- its gradients ------------------------------------------------------------------------

struct RmsBwdArgs {
    const half_t* s;
    const half_t* dout;
    const half_t* dsum;  // null: none
    const float* w;
    const float* rstd;
    half_t* ds;
    float* partial;  // [P][ldp]
    float* dw;
    int64_t M, C, ldp;
    int P;
    float inv_c;
};

// Rows of any length (past 16384 values): a block a row for ds; dw by columns in a kernel of its own, which reads s and
// dout again. [1024, 40000] bf16 with dsum: 107 us (492 MB read and written, 4.6 TB/s).
template <bool BF>
__global__ __launch_bounds__(kAny) void rms_norm_bwd_any_kernel(RmsBwdArgs a) {
    __shared__ float slot[kAny / kWave];
    const int C = (int)a.C, first = 8 * threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const float r = a.rstd[row];
        const half_t* sr = a.s + row * a.C;
        const half_t* dr = a.dout + row * a.C;
        float dot = 0.f;
        for (int c = first; c < C; c += 8 * kAny) {
            const half8 s = cut8(load8(sr, c, C), c, C), dy = cut8(load8(dr, c, C), c, C);
            const float8v w = load8f(a.w, c, C);
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += act_get<BF>(dy, e) * w[e] * (act_get<BF>(s, e) * r);
        }
        dot = block_sum<kAny>(dot, slot) * a.inv_c;
        for (int c = first; c < C; c += 8 * kAny) {
            const half8 s = cut8(load8(sr, c, C), c, C), dy = cut8(load8(dr, c, C), c, C);
            const float8v w = load8f(a.w, c, C);
            half8 dz = {};
            if (a.dsum != nullptr) dz = cut8(load8(a.dsum + row * a.C, c, C), c, C);
            act8<BF> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float d = r * (act_get<BF>(dy, e) * w[e] - act_get<BF>(s, e) * r * dot);
                if (a.dsum != nullptr) d += act_get<BF>(dz, e);
                o[e] = (act_t<BF>)d;
            }
            store8(a.ds + row * a.C, c, C, raw_act(o));
        }
    }
}
// 2048 columns a block, 8 a thread; rows blockIdx.y, + P, ...
template <bool BF>
__global__ __launch_bounds__(256) void rms_norm_dw_any_kernel(RmsBwdArgs a) {
    const int64_t col = 8 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
    if (col >= a.C) return;
    float8v dw = {};
    for (int64_t row = blockIdx.y; row < a.M; row += a.P) {
        const float r = a.rstd[row];
        const half8 s = cut8(load8(a.s + row * a.C, (int)col, (int)a.C), (int)col, (int)a.C);
        const half8 dy = cut8(load8(a.dout + row * a.C, (int)col, (int)a.C), (int)col, (int)a.C);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[e] += act_get<BF>(dy, e) * (act_get<BF>(s, e) * r);
    }
    *reinterpret_cast<float8v*>(a.partial + (int64_t)blockIdx.y * a.ldp + col) = dw;
}

// Rows of up to 8 TPR NCH values in registers, a block's share of dw in registers too, until its rows are done:
// one pass over s, dout and dsum, bound by memory. [16384, 8192] bf16 with dsum: 199 us (1.07 GB, 5.4 TB/s).
template <bool BF, int TPR, int NCH, bool DSUM>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_bwd_kernel(RmsBwdArgs a) {
    constexpr int ROWS = block_of(TPR) / TPR;
    __shared__ RowShare<TPR> share;
    __shared__ float8v groups[ROWS > 1 ? (ROWS - 1) * TPR * NCH : 1];
    const int part = threadIdx.x % TPR, sub = threadIdx.x / TPR, C = (int)a.C;
    int turn = 0;
    float8v w[NCH], dw[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        w[j] = load8f(a.w, 8 * (part + TPR * j), C);
        dw[j] = float8v{};
    }
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)a.P * ROWS) {
        const int64_t row = r0 + sub;
        const bool in = ROWS == 1 || row < a.M;
        const int64_t from = ROWS == 1 ? row : min(row, a.M - 1);  // a row past M reads the last one and counts as zeros
        const int len = in ? C : 0;
        const float r = a.rstd[from];
        half8 s[NCH], dy[NCH], dz[NCH];
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            s[j] = load8(a.s + from * C, 8 * (part + TPR * j), C);
            dy[j] = load8(a.dout + from * C, 8 * (part + TPR * j), C);
            if constexpr (DSUM) dz[j] = load8(a.dsum + from * C, 8 * (part + TPR * j), C);
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            s[j] = cut8(s[j], 8 * (part + TPR * j), C);
            dy[j] = cut8(dy[j], 8 * (part + TPR * j), C);
            if constexpr (DSUM) dz[j] = cut8(dz[j], 8 * (part + TPR * j), C);
            if (!in) s[j] = dy[j] = half8{};
        }
        Stats t{0.f, 0, 0};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float g = act_get<BF>(dy[j], e), xh = act_get<BF>(s[j], e) * r;
                t.sum += g * w[j][e] * xh;
                dw[j][e] += g * xh;
            }
        const float dot = row_all<TPR>(t, share, turn).sum * a.inv_c;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            act8<BF> o;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float xh = act_get<BF>(s[j], e) * r;
                float d = r * (act_get<BF>(dy[j], e) * w[j][e] - xh * dot);
                if constexpr (DSUM) d += act_get<BF>(dz[j], e);
                o[e] = (act_t<BF>)d;
            }
            store8(a.ds + row * C, 8 * (part + TPR * j), len, raw_act(o));
        }
    }
    if constexpr (ROWS > 1) {  // the block's row groups, in order
#pragma unroll
        for (int j = 0; j < NCH; ++j)
            if (sub > 0) groups[((sub - 1) * NCH + j) * TPR + part] = dw[j];
        __syncthreads();
        if (sub > 0) return;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
            for (int i = 0; i < ROWS - 1; ++i) dw[j] += groups[(i * NCH + j) * TPR + part];
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const int col = 8 * (part + TPR * j);
        if (col < a.ldp) *reinterpret_cast<float8v*>(a.partial + (int64_t)blockIdx.x * a.ldp + col) = dw[j];
    }
}

// dw[c] = the sum of the P partial rows: 16 interleaved groups of them, each in order, then the groups. 512 rows
// of 8192: 7 us, that is latency: eight loads in flight a thread.
__global__ __launch_bounds__(256) void rms_norm_dw_kernel(RmsBwdArgs a) {
    __shared__ float sums[16][16];
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + col;
    float v = 0.f;
    if (c < a.C) {
        const float* p = a.partial + c;
        int i = grp;
        for (; i + 7 * 16 < a.P; i += 8 * 16) {
            float u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = p[(int64_t)(i + 16 * k) * a.ldp];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += u[k];
        }
        for (; i < a.P; i += 16) v += p[(int64_t)i * a.ldp];
    }
    sums[grp][col] = v;
    __syncthreads();
    if (grp == 0 && c < a.C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sums[i][col];
        a.dw[c] = t;
    }
}

// Threads a row and 8-value chunks a thread for rows of Kp values (0: the kernels for rows of any length).
struct Route {
    int tpr, nch;
};
Route route_of(int64_t Kp) {
    if (Kp <= 64) return {8, 1};
    if (Kp <= 128) return {16, 1};
    if (Kp <= 256) return {32, 1};
    if (Kp <= 512) return {64, 1};
    if (Kp <= 1024) return {64, 2};
    if (Kp <= 2048) return {256, 1};
    if (Kp <= 4096) return {256, 2};
    if (Kp <= 6144) return {256, 3};
    if (Kp <= 8192) return {512, 2};
    if (Kp <= 12288) return {512, 3};
    if (Kp <= 16384) return {1024, 2};
    return {0, 0};
}
#define CLK_ROUTES(X_) X_(8, 1) X_(16, 1) X_(32, 1) X_(64, 1) X_(64, 2) X_(256, 1) X_(256, 2) X_(256, 3) X_(512, 2) X_(512, 3) X_(1024, 2)

int64_t padded64(int64_t k) { return (k + 63) / 64 * 64; }

// The gradients hold twice the registers: for [4096, 12000] 512 threads with 3 chunks take 100 us, 1024 with 2 88 us.
Route bwd_route(int64_t C) {
    const Route rt = route_of(padded64(C));
    return rt.nch == 3 && rt.tpr == 512 ? Route{1024, 2} : rt;
}

// The workgroups of the backward's first kernel: a rule on the shape alone, so that results do not
// depend on the device. One round of what 256 CUs hold, but where rows are few, about 8 steps each: a
// workgroup costs its row of partial sums, written and read.
int bwd_parts(int64_t M, int64_t C) {
    const Route rt = bwd_route(C);
    if (rt.tpr == 0) return (int)std::min<int64_t>(M, 64);
    const int rows = block_of(rt.tpr) / rt.tpr, threads = block_of(rt.tpr);
    const int64_t steps = (M + rows - 1) / rows, most = 256 * 1024 / threads;
    return (int)std::min(steps, std::min<int64_t>(most, std::max<int64_t>(256, steps / 8)));
}
// 16 threads a column, and a launch takes fewer than 2^32 threads
constexpr int64_t kMostBwd = 1 << 27;
int64_t bwd_ldp(int64_t C) { return (C + 63) / 64 * 64; }

// ---- rows to 8 bits and back --------------------------------------------------------------

struct QuantArgs {
    const void* x;
    int8_t* q;
    float* scale;
    int64_t M, K, Kp;
};

enum { kF16, kBf16, kF32 };
enum { kActNone, kActRelu, kActSwish };

// relu keeps a NaN (a row that holds one is NaN as a whole)
__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }

// 8 values from column col of a row of h: read, and made of what was read
template <int T>
struct Raw8 {
    half8 v;
};
template <>
struct Raw8<kF32> {
    float8v v;
};
template <int T>
__device__ __forceinline__ void read8(const void* x, int64_t at, int col, int K, Raw8<T>& r) {
    if constexpr (T == kF32) r.v = load8f(static_cast<const float*>(x) + at, col, K);
    else r.v = load8(static_cast<const half_t*>(x) + at, col, K);
}
template <int T>
__device__ __forceinline__ void floats8(const Raw8<T>& r, int col, int K, float (&f)[8]) {
    if constexpr (T == kF32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = r.v[e];
    } else {
        const half8 v = cut8(r.v, col, K);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = act_get<T == kBf16>(v, e);
    }
}

// h's 8 values from column c of the row that starts at x[at]
template <int T, int ACT>
__device__ __forceinline__ void hidden8(const void* x, int64_t at, int c, int K, float (&h)[8]) {
    Raw8<T> raw, up;
    read8(x, at, c, K, raw);
    if constexpr (ACT == kActSwish) read8(x, at + K, c, K, up);
    floats8(raw, c, K, h);
    float u[8];
    if constexpr (ACT == kActSwish) floats8(up, c, K, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (ACT == kActSwish) h[e] = h[e] * sigmoid_fast(h[e]) * u[e];
        if constexpr (ACT == kActRelu) h[e] = relu(h[e]);
    }
}

// Rows of any length, read twice. [1024, 40000] bf16: 28 us (123 MB, 4.4 TB/s).
template <int T, int ACT>
__global__ __launch_bounds__(kAny) void quantize_any_kernel(QuantArgs a) {
    __shared__ uint32_t slot[kAny / kWave];
    const int K = (int)a.K, Kp = (int)a.Kp, first = 8 * threadIdx.x;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const int64_t at = row * (ACT == kActSwish ? 2 * a.K : a.K);
        uint32_t m = 0;
        float h[8];
        for (int c = first; c < K; c += 8 * kAny) {
            hidden8<T, ACT>(a.x, at, c, K, h);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, abs_bits(h[e]));
        }
        float top, inv, scale;
        row_scale(block_max<kAny>(m, slot), 1.f, top, inv, scale);
        if (threadIdx.x == 0) a.scale[row] = scale;
        for (int c = first; c < Kp; c += 8 * kAny) {
            hidden8<T, ACT>(a.x, at, c, K, h);
            *reinterpret_cast<uint2v*>(a.q + row * a.Kp + c) = quant8<T != kF32 && ACT != kActSwish>(h, top, inv);
        }
    }
}

// As the norm: a row in registers, bound by memory. relu of [147456, 512] fp16: 45 to 54 us (227 MB, 4.2 to 5.0 TB/s;
// the less of it is left in the far cache by what ran before, the more); swish gate of [147456, 2 x 512] fp16 67 us (378
// MB, 5.6 TB/s), [147456, 512] fp32 64 us (378 MB, 5.9 TB/s).
template <int T, int ACT, int TPR, int NCH>
__global__ __launch_bounds__(block_of(TPR)) void quantize_kernel(QuantArgs a) {
    constexpr int ROWS = block_of(TPR) / TPR;
    constexpr bool GATE = ACT == kActSwish;
    __shared__ RowShare<TPR> share;
    const int part = threadIdx.x % TPR, sub = threadIdx.x / TPR, K = (int)a.K, Kp = (int)a.Kp;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.M; r0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = r0 + sub;
        const bool in = ROWS == 1 || row < a.M;
        const int64_t at = (ROWS == 1 ? row : min(row, a.M - 1)) * (GATE ? 2 * (int64_t)K : K);  // past M: the last row, unused
        Raw8<T> raw[NCH], up[GATE ? NCH : 1];
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            read8(a.x, at, 8 * (part + TPR * j), K, raw[j]);
            if constexpr (GATE) read8(a.x, at + K, 8 * (part + TPR * j), K, up[j]);
        }
        float h[NCH][8];
        Stats s{0.f, 0, 0};
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            float u[8];
            floats8(raw[j], 8 * (part + TPR * j), K, h[j]);
            if constexpr (GATE) floats8(up[j], 8 * (part + TPR * j), K, u);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (GATE) h[j][e] = h[j][e] * sigmoid_fast(h[j][e]) * u[e];
                if constexpr (ACT == kActRelu) h[j][e] = relu(h[j][e]);
                s.max0 = max(s.max0, abs_bits(h[j][e]));
            }
        }
        s = row_all<TPR>(s, share, turn);
        float top, inv, scale;
        row_scale(s.max0, 1.f, top, inv, scale);
        if (part == 0 && in) a.scale[row] = scale;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int col = 8 * (part + TPR * j);
            if (in && col < Kp) *reinterpret_cast<uint2v*>(a.q + row * Kp + col) = quant8<T != kF32 && !GATE>(h[j], top, inv);
        }
    }
}

struct DequantArgs {
    const int8_t* q;
    const float* scale;
    void* out;
    int64_t M, K, Kp;
};

// 2^shift threads a row, 16 bytes of results each at a time, so that a wave's store is a kilobyte in one piece ([16384,
// 8192] to fp32: 121 us, 172 with 32 bytes a thread). Results past half of the 256 MB far cache (NT) go by it:
// whoever reads them next finds little of them there, and the other arrays stay in it. [40000, 2048] quantised,
// dequantised to fp16 and added to another array takes 168 us, 179 without; 12000 rows 58, 57 without. [147456,
// 512] to fp16: 34 us (227 MB, 6.7 TB/s, part of it from the far cache).
template <int T>
constexpr int kDequant = T == kF32 ? 4 : 8;
template <int T, bool NT>
__global__ __launch_bounds__(256) void dequantize_kernel(DequantArgs a, int shift) {
    constexpr int E = kDequant<T>;
    typedef uint32_t words __attribute__((ext_vector_type(E / 4)));
    const int part = threadIdx.x & ((1 << shift) - 1), rows = 256 >> shift;
    for (int64_t row = (int64_t)blockIdx.x * rows + (threadIdx.x >> shift); row < a.M; row += (int64_t)gridDim.x * rows) {
        const float sc = a.scale[row];
        for (int64_t c = E * part; c < a.K; c += E << shift) {
            const words q = *reinterpret_cast<const words*>(a.q + row * a.Kp + c);
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = (float)(int8_t)(q[e >> 2] >> 8 * (e & 3)) * sc;
            const int left = (int)min<int64_t>(a.K - c, E);
            if constexpr (T == kF32) {
                store4f<NT>(static_cast<float*>(a.out) + row * a.K + c, left, float4v{v[0], v[1], v[2], v[3]});
            } else {
                act8<T == kBf16> h;
#pragma unroll
                for (int e = 0; e < E; ++e) h[e] = (act_t<T == kBf16>)v[e];
                store8<NT>(static_cast<half_t*>(a.out) + row * a.K + c, 0, left, raw_act(h));
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------

// M [rows] and C of an activation; the checks shared by the norm's entry points
int check_rows(const char* what, const clk_buffer* x) {
    if (x->rank != 2) return invalid(std::string(what) + ": x must be [M,C]");
    if (x->dims[0] < 0 || x->dims[1] < 1) return invalid(std::string(what) + ": C must be at least 1");
    if (x->dims[0] > INT32_MAX || x->dims[1] > INT32_MAX / 2) return invalid(std::string(what) + ": too large");
    return CLK_OK;
}

bool is_matrix(const clk_buffer* b, int64_t r, int64_t c) { return b->rank == 2 && b->dims[0] == r && b->dims[1] == c; }

unsigned any_blocks(int64_t M) { return (unsigned)std::min<int64_t>(M, 1 << 20); }

// Workgroups for M rows of tpr threads each
unsigned row_blocks(int64_t M, int tpr) {
    const int rows = block_of(tpr) / tpr;
    return (unsigned)std::min<int64_t>((M + rows - 1) / rows, 1 << 20);
}

int rms_forward(const char* what, clk_stream stream, const clk_buffer* x, const clk_buffer* residual,
                const clk_buffer* scale, const clk_buffer* sum, const clk_buffer* out, const clk_buffer* stat,
                float eps, int32_t has_residual, bool want_stat, bool q8) {
    const int act = x != nullptr && x->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {x, residual, scale, sum, out, stat};
    const int types[] = {act, act, CLK_F32, act, q8 ? CLK_S8 : act, CLK_F32};
    if (int st = check_types(what, bufs, types, 6)) return st;
    if (int st = check_rows(what, x)) return st;
    const int64_t M = x->dims[0], C = x->dims[1], Kp = padded64(C);
    if (elements(scale) != C) return invalid(std::string(what) + ": scale must be [C]");
    if (has_residual && (!same_shape(residual, x) || !same_shape(sum, x))) {
        return invalid(std::string(what) + ": residual and sum must be like x");
    }
    if (q8 ? !is_matrix(out, M, Kp) : !same_shape(out, x)) {
        return invalid(std::string(what) + (q8 ? ": q must be [M,Kp], Kp = C rounded up to a multiple of 64" : ": out must be like x"));
    }
    if (want_stat && elements(stat) != M) return invalid(std::string(what) + (q8 ? ": q_scale must be [M]" : ": rstd must be [M]"));
    if (!(eps >= 0.f)) return invalid(std::string(what) + ": eps must not be negative");
    if (M == 0) return ok();
    if (!q8 && has_residual && out->data == sum->data) return invalid(std::string(what) + ": out and sum must not be the same buffer");
    if (q8 && !aligned16(out->data)) return invalid(std::string(what) + ": q must be 16-byte aligned");
    RmsArgs a{static_cast<const half_t*>(x->data), static_cast<const half_t*>(residual->data),
              static_cast<const float*>(scale->data), static_cast<half_t*>(sum->data),
              q8 ? nullptr : static_cast<half_t*>(out->data), q8 ? static_cast<int8_t*>(out->data) : nullptr,
              want_stat ? static_cast<float*>(stat->data) : nullptr, M, C, Kp, 1.f / (float)C, eps};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const bool bf = act == CLK_BF16;
    stage_mark(s, 0);
    const Route rt = route_of(Kp);
#define CLK_RMS_RT(TPR_, NCH_)                                                                                        \
    if (rt.tpr == TPR_ && rt.nch == NCH_) {                                                                           \
        if (has_residual) hipLaunchKernelGGL((rms_norm_kernel<BF, TPR_, NCH_, true, Q8>), grid, block, 0, s, a);      \
        else hipLaunchKernelGGL((rms_norm_kernel<BF, TPR_, NCH_, false, Q8>), grid, block, 0, s, a);                  \
    }
    const auto launch = [&](auto bf_, auto q8_) {
        constexpr bool BF = decltype(bf_)::value, Q8 = decltype(q8_)::value;
        if (rt.tpr == 0) {
            const dim3 grid(any_blocks(M)), block(kAny);
            if (has_residual) hipLaunchKernelGGL((rms_norm_any_kernel<BF, true, Q8>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((rms_norm_any_kernel<BF, false, Q8>), grid, block, 0, s, a);
            return;
        }
        const dim3 grid(row_blocks(M, rt.tpr)), block(block_of(rt.tpr));
        CLK_ROUTES(CLK_RMS_RT)
    };
    if (bf) q8 ? launch(std::true_type(), std::true_type()) : launch(std::true_type(), std::false_type());
    else q8 ? launch(std::false_type(), std::true_type()) : launch(std::false_type(), std::false_type());
#undef CLK_RMS_RT
    stage_mark(s, 1);
    return launch_status(what);
}

}  // namespace

}  // namespace clk

using namespace clk;

extern "C" int clk_rms_norm(clk_stream stream, const clk_buffer* x, const clk_buffer* residual,
                            const clk_buffer* scale, const clk_buffer* sum, const clk_buffer* out,
                            const clk_buffer* rstd, float eps, int32_t has_residual, int32_t want_rstd) {
    return rms_forward("rms_norm", stream, x, residual, scale, sum, out, rstd, eps, has_residual, want_rstd != 0, false);
}

extern "C" int clk_rms_norm_q8(clk_stream stream, const clk_buffer* x, const clk_buffer* residual,
                               const clk_buffer* scale, const clk_buffer* sum, const clk_buffer* q,
                               const clk_buffer* q_scale, float eps, int32_t has_residual) {
    return rms_forward("rms_norm_q8", stream, x, residual, scale, sum, q, q_scale, eps, has_residual, true, true);
}

extern "C" size_t clk_rms_norm_bwd_workspace_size(const clk_buffer* s) {
    if (s == nullptr || s->rank != 2 || s->dims == nullptr || s->dims[0] < 1 || s->dims[1] < 1 ||
        s->dims[0] > INT32_MAX || s->dims[1] > kMostBwd) {
        return 0;
    }
    return (size_t)bwd_parts(s->dims[0], s->dims[1]) * bwd_ldp(s->dims[1]) * 4;
}

extern "C" int clk_rms_norm_bwd(clk_stream stream, const clk_buffer* s, const clk_buffer* scale,
                                const clk_buffer* rstd, const clk_buffer* dout, const clk_buffer* dsum,
                                const clk_buffer* ds, const clk_buffer* dscale, int32_t has_dsum,
                                void* workspace, size_t workspace_bytes) {
    const int act = s != nullptr && s->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {s, scale, rstd, dout, dsum, ds, dscale};
    const int types[] = {act, CLK_F32, CLK_F32, act, act, act, CLK_F32};
    if (int st = check_types("rms_norm_bwd", bufs, types, 7)) return st;
    if (int st = check_rows("rms_norm_bwd", s)) return st;
    if (s->dims[1] > kMostBwd) return invalid("rms_norm_bwd: too large");
    const int64_t M = s->dims[0], C = s->dims[1];
    if (elements(scale) != C || elements(dscale) != C) return invalid("rms_norm_bwd: scale and dscale must be [C]");
    if (elements(rstd) != M) return invalid("rms_norm_bwd: rstd must be [M]");
    if (!same_shape(dout, s) || !same_shape(ds, s) || (has_dsum && !same_shape(dsum, s))) {
        return invalid("rms_norm_bwd: dout, dsum and ds must be like s");
    }
    const size_t need = clk_rms_norm_bwd_workspace_size(s);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
        return invalid("rms_norm_bwd: workspace of " + std::to_string(workspace_bytes) + " bytes, needs " + std::to_string(need));
    }
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return invalid("rms_norm_bwd: workspace must be 256-byte aligned");
    RmsBwdArgs a{static_cast<const half_t*>(s->data), static_cast<const half_t*>(dout->data),
                 has_dsum ? static_cast<const half_t*>(dsum->data) : nullptr, static_cast<const float*>(scale->data),
                 static_cast<const float*>(rstd->data), static_cast<half_t*>(ds->data), static_cast<float*>(workspace),
                 static_cast<float*>(dscale->data), M, C, bwd_ldp(C), M > 0 ? bwd_parts(M, C) : 0, 1.f / (float)C};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int stage = 0;
    stage_mark(st, stage);
    if (M > 0) {
        const Route rt = bwd_route(C);
#define CLK_BWD_RT(TPR_, NCH_)                                                                                        \
    if (rt.tpr == TPR_ && rt.nch == NCH_) {                                                               \
        if (has_dsum) hipLaunchKernelGGL((rms_norm_bwd_kernel<BF, TPR_, NCH_, true>), grid, block, 0, st, a);         \
        else hipLaunchKernelGGL((rms_norm_bwd_kernel<BF, TPR_, NCH_, false>), grid, block, 0, st, a);                 \
    }
        const auto launch = [&](auto bf_) {
            constexpr bool BF = decltype(bf_)::value;
            if (rt.tpr == 0) {
                // dw first: ds may overwrite dout
                hipLaunchKernelGGL(rms_norm_dw_any_kernel<BF>, dim3((unsigned)((C + 2047) / 2048), a.P), dim3(256), 0, st, a);
                stage_mark(st, ++stage);
                hipLaunchKernelGGL(rms_norm_bwd_any_kernel<BF>, dim3(any_blocks(M)), dim3(kAny), 0, st, a);
                return;
            }
            const dim3 grid(a.P), block(block_of(rt.tpr));
            CLK_ROUTES(CLK_BWD_RT)
        };
        act == CLK_BF16 ? launch(std::true_type()) : launch(std::false_type());
        stage_mark(st, ++stage);
#undef CLK_BWD_RT
    }
    hipLaunchKernelGGL(rms_norm_dw_kernel, dim3((unsigned)((C + 15) / 16)), dim3(256), 0, st, a);
    stage_mark(st, ++stage);
    return launch_status("rms_norm_bwd");
}

extern "C" int clk_quantize_rows(clk_stream stream, const clk_buffer* x, const clk_buffer* q,
                                 const clk_buffer* q_scale, int64_t activation) {
    const int xt = x != nullptr && (x->dtype == CLK_BF16 || x->dtype == CLK_F32) ? x->dtype : CLK_F16;
    const clk_buffer* bufs[] = {x, q, q_scale};
    const int types[] = {xt, CLK_S8, CLK_F32};
    if (int st = check_types("quantize_rows", bufs, types, 3)) return st;
    if (activation < 0 || activation > 2) {
        return invalid("quantize_rows: activation is 0 (none), 1 (relu) or 2 (swish gate), got " + std::to_string(activation));
    }
    if (int st = check_rows("quantize_rows", x)) return st;
    const int64_t M = x->dims[0];
    if (activation == kActSwish && x->dims[1] % 2) return invalid("quantize_rows: a gated x must be [M,2K]");
    const int64_t K = activation == kActSwish ? x->dims[1] / 2 : x->dims[1], Kp = padded64(K);
    if (!is_matrix(q, M, Kp)) return invalid("quantize_rows: q must be [M,Kp], Kp = K rounded up to a multiple of 64");
    if (elements(q_scale) != M) return invalid("quantize_rows: q_scale must be [M]");
    if (M == 0) return ok();
    if (!aligned16(q->data)) return invalid("quantize_rows: q must be 16-byte aligned");
    QuantArgs a{x->data, static_cast<int8_t*>(q->data), static_cast<float*>(q_scale->data), M, K, Kp};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    const Route rt = route_of(Kp);
#define CLK_QR_RT(TPR_, NCH_) \
    if (rt.tpr == TPR_ && rt.nch == NCH_) hipLaunchKernelGGL((quantize_kernel<T, A, TPR_, NCH_>), grid, block, 0, s, a);
    const auto launch = [&](auto t_, auto a_) {
        constexpr int T = decltype(t_)::value, A = decltype(a_)::value;
        const dim3 grid(rt.tpr == 0 ? any_blocks(M) : row_blocks(M, rt.tpr)), block(rt.tpr == 0 ? kAny : block_of(rt.tpr));
        if (rt.tpr == 0) hipLaunchKernelGGL((quantize_any_kernel<T, A>), grid, block, 0, s, a);
        CLK_ROUTES(CLK_QR_RT)
    };
    const auto by_act = [&](auto t_) {
        if (activation == kActNone) launch(t_, std::integral_constant<int, kActNone>());
        else if (activation == kActRelu) launch(t_, std::integral_constant<int, kActRelu>());
        else launch(t_, std::integral_constant<int, kActSwish>());
    };
    if (xt == CLK_F32) by_act(std::integral_constant<int, kF32>());
    else if (xt == CLK_BF16) by_act(std::integral_constant<int, kBf16>());
    else by_act(std::integral_constant<int, kF16>());
#undef CLK_QR_RT
    stage_mark(s, 1);
    return launch_status("quantize_rows");
}

extern "C" int clk_dequantize_rows(clk_stream stream, const clk_buffer* q, const clk_buffer* q_scale,
                                   const clk_buffer* out) {
    const int ot = out != nullptr && (out->dtype == CLK_BF16 || out->dtype == CLK_F32) ? out->dtype : CLK_F16;
    const clk_buffer* bufs[] = {q, q_scale, out};
    const int types[] = {CLK_S8, CLK_F32, ot};
    if (int st = check_types("dequantize_rows", bufs, types, 3)) return st;
    if (int st = check_rows("dequantize_rows", out)) return st;
    const int64_t M = out->dims[0], K = out->dims[1], Kp = padded64(K);
    if (!is_matrix(q, M, Kp)) return invalid("dequantize_rows: q must be [M,Kp], Kp = K rounded up to a multiple of 64");
    if (elements(q_scale) != M) return invalid("dequantize_rows: q_scale must be [M]");
    if (M == 0) return ok();
    if (!aligned16(q->data)) return invalid("dequantize_rows: q must be 16-byte aligned");
    DequantArgs a{static_cast<const int8_t*>(q->data), static_cast<const float*>(q_scale->data), out->data, M, K, Kp};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    int shift = 3;
    while (shift < 8 && ((ot == CLK_F32 ? kDequant<kF32> : kDequant<kF16>) << shift) < K) ++shift;
    const dim3 grid(row_blocks(M, 1 << shift)), block(256);
    const auto launch = [&](auto t_) {
        constexpr int T = decltype(t_)::value;
        if (M * K >= (int64_t)(1 << 27) / (T == kF32 ? 4 : 2)) hipLaunchKernelGGL((dequantize_kernel<T, true>), grid, block, 0, s, a, shift);
        else hipLaunchKernelGGL((dequantize_kernel<T, false>), grid, block, 0, s, a, shift);
    };
    if (ot == CLK_F32) launch(std::integral_constant<int, kF32>());
    else if (ot == CLK_BF16) launch(std::integral_constant<int, kBf16>());
    else launch(std::integral_constant<int, kF16>());
    stage_mark(s, 1);
    return launch_status("dequantize_rows");
}
