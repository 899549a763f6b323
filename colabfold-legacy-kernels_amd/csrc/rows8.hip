// RMS norm and 8-bit rows for gfx950 (CDNA4). No counterpart in the reference; they stand beside its
// LayerNorm and feed the 8-bit matrix product (q8_gemm.hip).
//
//   rms_norm        s = round16(x + residual), y = round16(s r w), r = 1 / sqrt(mean(s^2) + eps)
//   rms_norm_q8     t = s w, a = max |t|; q = rint(t (127 / a)), scale = a r / 127: r cancels in q, so
//                   the integers depend on s and w alone
//   rms_norm_bwd    g = dy w, xh = s r: ds = r (g - xh mean(g xh)) + dsum, dw = sum over rows of dy xh
//   quantize_rows   h = x, relu(x) or swish(x[:, :K]) x[:, K:]; q = rint(h (127 / a)), scale = a / 127
//   dequantize_rows out = q scale
//
// All of them are bound by memory: each value is read once and written once, statistics and products
// are fp32, and results are rounded once.
#include "clk_common.h"

#include <algorithm>

namespace clk {

namespace {

typedef half8 half8u __attribute__((aligned(2)));
typedef half_t half_u __attribute__((aligned(2)));
typedef float8v float8u __attribute__((aligned(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

// Rows whose scale a / 127 would leave fp32's normal range count as zeros (then 127 / a is finite too).
constexpr float kTiny = 0x1p-119f;
constexpr uint32_t kInfBits = 0x7f800000u;

// |t| as an integer that orders like it, with infinities and NaN on top: a maximum that keeps them,
// where a float maximum drops NaN
__device__ __forceinline__ uint32_t abs_bits(float t) { return __builtin_bit_cast(uint32_t, t) & 0x7fffffffu; }

// What a row of largest magnitude `bits` is multiplied by before the rounding, and its scale times r.
// A row with an infinity or NaN is zeros with scale NaN, so everything computed from it is NaN.
__device__ __forceinline__ void row_scale(uint32_t bits, float r, float& inv, float& scale) {
    const float a = __builtin_bit_cast(float, bits);
    if (bits >= kInfBits) {
        inv = 0.f;
        scale = __builtin_nanf("");
    } else if (a < kTiny) {
        inv = 0.f;
        scale = 0.f;
    } else {
        inv = 127.f / a;
        scale = a * r / 127.f;
    }
}

// rint(t inv) as an integer, ties to even; |t| <= a bounds it by 127, and inv = 0 (a row of zeros)
// gives 0 also for a t that is not finite
__device__ __forceinline__ int quant(float t, float inv) { return inv == 0.f ? 0 : (int)__builtin_rintf(t * inv); }

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// 1 / sqrt(ss / C + eps) from a row's sum of squares
__device__ __forceinline__ float inv_rms(float ss, float inv_c, float eps) { return 1.f / sqrtf(ss * inv_c + eps); }

// A bf16 row with values past kBig has sums of squares, or products with w, past fp32's range: it is
// taken with its values scaled by kDown (a power of two, so every product stays what it was), where eps
// is nothing.
constexpr float kBig = 0x1p40f, kDown = 0x1p-90f;
__device__ __forceinline__ bool is_big(uint32_t bits) { return bits >= __builtin_bit_cast(uint32_t, kBig) && bits < kInfBits; }

// Sum and maximum over the threads of a block, in every thread; `slot` alternates between calls that no
// barrier separates otherwise.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* slot) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o);
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
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    if ((threadIdx.x & (kWave - 1)) == 0) slot[threadIdx.x / kWave] = v;
    __syncthreads();
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) s = max(s, slot[i]);
    __syncthreads();
    return s;
}

template <bool BF>
__device__ __forceinline__ float get16(const half_t* p) {
    const half_t h = *p;
    if constexpr (BF) {
        return (float)__builtin_bit_cast(__bf16, h);
    } else {
        return (float)h;
    }
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

// Rows of any length: a block a row, two passes over it (the second from cache where it fits).
template <bool BF, bool RES, bool Q8>
__global__ __launch_bounds__(256) void rms_norm_any_kernel(RmsArgs a) {
    __shared__ float fslot[4];
    __shared__ uint32_t uslot[4];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const half_t* xr = a.x + row * a.C;
        const half_t* rr = a.residual + row * a.C;
        half_t* sr = a.sum + row * a.C;
        float ss = 0.f;
        uint32_t m = 0, mt = 0;
        for (int64_t c = threadIdx.x; c < a.C; c += 256) {
            float v = get16<BF>(xr + c);
            if constexpr (RES) {
                const half_t h = act_cvt<BF>(v + get16<BF>(rr + c));
                sr[c] = h;
                v = get16<BF>(&h);
            }
            ss += v * v;
            m = max(m, abs_bits(v));
            if constexpr (Q8) mt = max(mt, abs_bits(v * a.w[c]));
        }
        const half_t* vr = RES ? sr : xr;  // each thread reads back only what it wrote
        ss = block_sum<256>(ss, fslot);
        m = block_max<256>(m, uslot);
        float d = 1.f;
        if (BF && is_big(m)) {
            d = kDown;
            ss = 0.f;
            mt = 0;
            for (int64_t c = threadIdx.x; c < a.C; c += 256) {
                const float v = get16<BF>(vr + c) * d;
                ss += v * v;
                if constexpr (Q8) mt = max(mt, abs_bits(v * a.w[c]));
            }
            ss = block_sum<256>(ss, fslot);
        }
        const float r = inv_rms(ss, a.inv_c, d == 1.f ? a.eps : 0.f);
        if constexpr (Q8) {
            mt = block_max<256>(max(mt, m >= kInfBits ? m : 0u), uslot);
            float inv, scale;
            row_scale(mt, r, inv, scale);
            if (threadIdx.x == 0) a.stat[row] = scale;
            int8_t* qr = a.q + row * a.Kp;
            for (int64_t c = threadIdx.x; c < a.Kp; c += 256) {
                qr[c] = c < a.C ? (int8_t)quant(get16<BF>(vr + c) * d * a.w[c], inv) : (int8_t)0;
            }
        } else {
            if (threadIdx.x == 0 && a.stat != nullptr) a.stat[row] = r * d;
            half_t* orow = a.out + row * a.C;
            for (int64_t c = threadIdx.x; c < a.C; c += 256) {
                orow[c] = act_cvt<BF>(get16<BF>(vr + c) * d * r * a.w[c]);
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

// Workgroup p takes rows p, p + P, ...; its share of dw goes to row p of the workspace, where each thread
// adds to columns of its own.
template <bool BF>
__global__ __launch_bounds__(256) void rms_norm_bwd_any_kernel(RmsBwdArgs a) {
    __shared__ float slot[4];
    float* part = a.partial + (int64_t)blockIdx.x * a.ldp;
    for (int64_t row = blockIdx.x; row < a.M; row += a.P) {
        const float r = a.rstd[row];
        const half_t* sr = a.s + row * a.C;
        const half_t* dr = a.dout + row * a.C;
        float dot = 0.f;
        for (int64_t c = threadIdx.x; c < a.C; c += 256) {
            dot += get16<BF>(dr + c) * a.w[c] * (get16<BF>(sr + c) * r);
        }
        dot = block_sum<256>(dot, slot) * a.inv_c;
        for (int64_t c = threadIdx.x; c < a.C; c += 256) {
            const float dy = get16<BF>(dr + c), xh = get16<BF>(sr + c) * r;
            float d = r * (dy * a.w[c] - xh * dot);
            if (a.dsum != nullptr) d += get16<BF>(a.dsum + row * a.C + c);
            a.ds[row * a.C + c] = act_cvt<BF>(d);
            part[c] = (row == blockIdx.x ? 0.f : part[c]) + dy * xh;
        }
    }
}

// dw[c] = the sum of the P partial rows, in their order within each of 8 interleaved groups
__global__ __launch_bounds__(256) void rms_norm_dw_kernel(RmsBwdArgs a) {
    __shared__ float sums[8][32];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    float v = 0.f;
    if (c < a.C) {
        for (int p = grp; p < a.P; p += 8) v += a.partial[(int64_t)p * a.ldp + c];
    }
    sums[grp][col] = v;
    __syncthreads();
    if (grp == 0 && c < a.C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += sums[i][col];
        a.dw[c] = t;
    }
}

// The workgroups of the backward's first kernel: a rule on the shape alone, so that results do not
// depend on the device.
int bwd_parts(int64_t M, int64_t C) {
    (void)C;
    return (int)std::min<int64_t>(M, 512);
}
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

template <int T>
__device__ __forceinline__ float get_any(const void* p, int64_t i) {
    if constexpr (T == kF32) {
        return static_cast<const float*>(p)[i];
    } else {
        return get16<T == kBf16>(static_cast<const half_t*>(p) + i);
    }
}

// relu keeps a NaN (a row that holds one is NaN as a whole)
__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }

template <int T, int ACT>
__device__ __forceinline__ float hidden(const void* x, int64_t row, int64_t k, int64_t K) {
    if constexpr (ACT == kActSwish) {
        const float g = get_any<T>(x, row * 2 * K + k), u = get_any<T>(x, row * 2 * K + K + k);
        return g * sigmoid_fast(g) * u;
    } else {
        const float v = get_any<T>(x, row * K + k);
        return ACT == kActRelu ? relu(v) : v;
    }
}

template <int T, int ACT>
__global__ __launch_bounds__(256) void quantize_any_kernel(QuantArgs a) {
    __shared__ uint32_t slot[4];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        uint32_t m = 0;
        for (int64_t k = threadIdx.x; k < a.K; k += 256) m = max(m, abs_bits(hidden<T, ACT>(a.x, row, k, a.K)));
        float inv, scale;
        row_scale(block_max<256>(m, slot), 1.f, inv, scale);
        if (threadIdx.x == 0) a.scale[row] = scale;
        for (int64_t k = threadIdx.x; k < a.Kp; k += 256) {
            a.q[row * a.Kp + k] = k < a.K ? (int8_t)quant(hidden<T, ACT>(a.x, row, k, a.K), inv) : (int8_t)0;
        }
    }
}

struct DequantArgs {
    const int8_t* q;
    const float* scale;
    void* out;
    int64_t M, K, Kp;
};

template <int T>
__global__ __launch_bounds__(256) void dequantize_any_kernel(DequantArgs a) {
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const float sc = a.scale[row];
        for (int64_t k = threadIdx.x; k < a.K; k += 256) {
            const float v = (float)a.q[row * a.Kp + k] * sc;
            if constexpr (T == kF32) {
                static_cast<float*>(a.out)[row * a.K + k] = v;
            } else {
                static_cast<half_t*>(a.out)[row * a.K + k] = act_cvt<T == kBf16>(v);
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------

int64_t padded64(int64_t k) { return (k + 63) / 64 * 64; }

bool is_act(int t) { return t == CLK_F16 || t == CLK_BF16; }

// M [rows] and C of an activation; the checks shared by the norm's entry points
int check_rows(const char* what, const clk_buffer* x) {
    if (x->rank != 2) return invalid(std::string(what) + ": x must be [M,C]");
    if (x->dims[0] < 0 || x->dims[1] < 1) return invalid(std::string(what) + ": C must be at least 1");
    if (x->dims[0] > INT32_MAX || x->dims[1] > INT32_MAX / 2) return invalid(std::string(what) + ": too large");
    return CLK_OK;
}

bool is_matrix(const clk_buffer* b, int64_t r, int64_t c) { return b->rank == 2 && b->dims[0] == r && b->dims[1] == c; }

unsigned row_blocks(int64_t M) { return (unsigned)std::min<int64_t>(M, 1 << 20); }

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
#define CLK_RMS(BF_, RES_, Q8_)                                                                      \
    if (bf == BF_ && (has_residual != 0) == RES_ && q8 == Q8_)                                       \
        hipLaunchKernelGGL((rms_norm_any_kernel<BF_, RES_, Q8_>), dim3(row_blocks(M)), dim3(256), 0, s, a);
    CLK_RMS(false, false, false) CLK_RMS(false, false, true) CLK_RMS(false, true, false) CLK_RMS(false, true, true)
    CLK_RMS(true, false, false) CLK_RMS(true, false, true) CLK_RMS(true, true, false) CLK_RMS(true, true, true)
#undef CLK_RMS
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
        s->dims[0] > INT32_MAX || s->dims[1] > INT32_MAX / 2) {
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
    stage_mark(st, 0);
    if (M > 0) {
        if (act == CLK_BF16) hipLaunchKernelGGL(rms_norm_bwd_any_kernel<true>, dim3(a.P), dim3(256), 0, st, a);
        else hipLaunchKernelGGL(rms_norm_bwd_any_kernel<false>, dim3(a.P), dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL(rms_norm_dw_kernel, dim3((unsigned)((C + 31) / 32)), dim3(256), 0, st, a);
    stage_mark(st, 1);
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
    const int t = xt == CLK_F32 ? kF32 : xt == CLK_BF16 ? kBf16 : kF16;
    stage_mark(s, 0);
#define CLK_QR(T_, A_) \
    if (t == T_ && activation == A_) hipLaunchKernelGGL((quantize_any_kernel<T_, A_>), dim3(row_blocks(M)), dim3(256), 0, s, a);
    CLK_QR(kF16, 0) CLK_QR(kF16, 1) CLK_QR(kF16, 2) CLK_QR(kBf16, 0) CLK_QR(kBf16, 1) CLK_QR(kBf16, 2)
    CLK_QR(kF32, 0) CLK_QR(kF32, 1) CLK_QR(kF32, 2)
#undef CLK_QR
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
    if (ot == CLK_F32) hipLaunchKernelGGL(dequantize_any_kernel<kF32>, dim3(row_blocks(M)), dim3(256), 0, s, a);
    else if (ot == CLK_BF16) hipLaunchKernelGGL(dequantize_any_kernel<kBf16>, dim3(row_blocks(M)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(dequantize_any_kernel<kF16>, dim3(row_blocks(M)), dim3(256), 0, s, a);
    stage_mark(s, 1);
    return launch_status("dequantize_rows");
}
