// Attention of one new token a sequence over a paged key-value cache, for gfx950 (CDNA4). No counterpart in the reference.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j), over the length[b] tokens that the sequence's
//   pages hold for the head of keys h / (Hq / Hkv);  lse = log2(sum_j p_j), in the log2 domain
//
// Every cached byte is needed once, which bounds it: 4 Hq / Hkv operations a cached value are far under the matrix
// cores' rate up to some hundred query heads a head of keys.
//
// A wave takes 32 tokens at a time, two blocks of the cache (kv_cache.h), for 16 query heads of one head of keys
// (rows past the group's last are zeros and cost nothing: the cache's bytes are what takes the time):
//   S^T = K Q^T        K's operands are the cache's bytes as they lie; a lane gets tokens 4 g .. + 3 of each block for
//                      query l % 16
//   O^T += V^T P^T     P^T's operand is what the lane holds; V's operand for it is again the cache's bytes
// with the running maximum and sum of a softmax. Both operands come from memory to registers with nothing between.
#include "kv_cache.h"

#include <algorithm>
#include <type_traits>

namespace clk {

namespace {

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 32;  // tokens a wave takes at a time

struct AttnArgs {
    const half_t* q;  // [B, Hq, D]
    const char* kc;
    const char* vc;
    const float* ks;
    const float* vs;
    const int32_t* table;  // [B, per]
    const int32_t* len;    // [B]
    half_t* out;
    float* lse;  // may be null
    int B, Hkv, G, blocks;  // G query heads a head of keys, in blocks of 16
    int per, pages, page;
    FastDiv by_page, by_blocks, by_hkv;
    float scale2;  // scale log2 e
};

template <bool BF>
__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) {
    if constexpr (BF) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return mfma16x16x32(a, b, c);
    }
}

// Four 8-bit integers as bf16, which holds them exactly: by fp32, whose low halves are then zeros
__device__ __forceinline__ uint2v bf16_of_bytes(uint32_t w) {
    uint32_t f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __builtin_bit_cast(uint32_t, (float)(int8_t)(w >> 8 * e));
    return uint2v{__builtin_amdgcn_perm(f[1], f[0], 0x07060302u), __builtin_amdgcn_perm(f[3], f[2], 0x07060302u)};
}
__device__ __forceinline__ half8 join(uint2v a, uint2v b) { return __builtin_bit_cast(half8, uint4v{a[0], a[1], b[0], b[1]}); }

// Eight weights in two 16-bit parts each, 2^-16 (bf16) or 2^-22 of them at most away from their sum: one would make a
// result's error half a step larger than its own rounding. The matrix cores have time for both.
// ABOVE: the first part is a step below the weight cut off, so that the second is positive too and an infinity among
// the values stays one (a second part of zero or below would make it NaN).
template <bool BF, bool ABOVE>
__device__ __forceinline__ void two_parts(const float (&f)[8], half8& hi, half8& lo) {
    float rest[8];
    if constexpr (ABOVE) {
        raw8 cut;
        if constexpr (BF) {
#pragma unroll
            for (int e = 0; e < 8; ++e) cut[e] = (uint16_t)(__builtin_bit_cast(uint32_t, f[e]) >> 16);
        } else {
            uint4v w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f[2 * e], f[2 * e + 1]));
            cut = __builtin_bit_cast(raw8, w);
        }
        hi = __builtin_bit_cast(half8, __builtin_elementwise_sub_sat(cut, raw8{1, 1, 1, 1, 1, 1, 1, 1}));
    } else {
        hi = __builtin_bit_cast(half8, act_cvt8<BF>(f));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = f[e] - act_get<BF>(hi, e);
    lo = __builtin_bit_cast(half8, act_cvt8<BF>(rest));
}

// A tile's cached bytes as they were loaded: keys as operands, values as cells of four tokens a channel block
template <bool Q8, int D>
struct Tile {
    static constexpr int NK = Q8 ? (D + 63) / 64 : D / 32;  // key loads a block
    static constexpr int C = value_group(Q8, D);            // channel blocks a value load
    static constexpr int NV = D / 16 / C;
    uint4v k[2][NK];
    uint4v v[2][NV];  // 8-byte loads (Q8, D no multiple of 64) in the low half
    float4v ks[2], vs[2];
};

template <bool BF, bool Q8, int D>
__global__ __launch_bounds__(kWaves * kWave) void paged_attn_kernel(AttnArgs a) {
    typedef Tile<Q8, D> T;
    constexpr int KS = D / 32, DB = D / 16, SIZE = Q8 ? 1 : 2;
    constexpr bool MBF = BF || Q8;       // the products' operands are bf16
    constexpr bool QLO = Q8 && !BF;      // fp16 queries in two bf16 parts, which is exact
    constexpr float kBias = MBF ? -24.f : 15.f;
    __shared__ float stat[kWaves][2][16];
    __shared__ float acc[2][16][D + 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, i16 = lane & 15, g = lane >> 4;
    int item = blockIdx.x;
    const int seq_head = fdiv(item, a.by_blocks), rb = item - seq_head * a.blocks;
    const int b = fdiv(seq_head, a.by_hkv), h = seq_head - b * a.Hkv;
    const int rows = min(16, a.G - 16 * rb);
    const int64_t qrow = ((int64_t)b * a.Hkv + h) * a.G + 16 * rb;
    const int len = max(a.len[b], 0);
    const int32_t* table = a.table + (int64_t)b * a.per;
    bool bad = (int64_t)len > (int64_t)a.per * a.page;
    const int keys = bad ? 0 : len;

    // the queries' operands; channels in the order of the keys'
    half8 q[KS], qlo[QLO ? KS : 1];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const bool pair = Q8 && (s / 2 * 64 + 64 <= D);
        const int d = pair ? s / 2 * 64 + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
        uint4v raw{};
        if (i16 < rows) raw = *reinterpret_cast<const uint4v*>(a.q + (qrow + i16) * D + d);
        q[s] = __builtin_bit_cast(half8, raw);
        if constexpr (QLO) {
            bf16x8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = (float)q[s][e];
                hi[e] = (__bf16)f;
                lo[e] = (__bf16)(f - (float)hi[e]);
            }
            q[s] = __builtin_bit_cast(half8, hi);
            qlo[s] = __builtin_bit_cast(half8, lo);
        }
    }

    float4v o[DB];
#pragma unroll
    for (int e = 0; e < DB; ++e) o[e] = float4v{};
    float m = -__builtin_inff(), l = 0.f;

    for (int k0 = wave * kTile; k0 < keys; k0 += kWaves * kTile) {
        T t;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int at = k0 + 16 * n < keys ? k0 + 16 * n : k0;
            const int p = fdiv(at, a.by_page);
            int page = table[p];  // one that the cache does not have: page 0, and NaN in the end
            if ((uint32_t)page >= (uint32_t)a.pages) {
                bad = true;
                page = 0;
            }
            const int64_t row = ((int64_t)page * a.Hkv + h) * a.page + (at - p * a.page);
            const char* kb = a.kc + row * (D * SIZE);
            const char* vb = a.vc + row * (D * SIZE);
#pragma unroll
            for (int s = 0; s < T::NK; ++s) {
                if constexpr (!Q8) {
                    t.k[n][s] = *reinterpret_cast<const uint4v*>(kb + s * 1024 + lane * 16);
                } else if (s * 64 + 64 <= D) {
                    t.k[n][s] = *reinterpret_cast<const uint4v*>(kb + s * 1024 + lane * 16);
                } else {
                    const uint2v w = *reinterpret_cast<const uint2v*>(kb + s * 1024 + (g >> 1) * 256 + i16 * 16 + (g & 1) * 8);
                    t.k[n][s] = uint4v{w[0], w[1], 0, 0};
                }
            }
#pragma unroll
            for (int s = 0; s < T::NV; ++s) {
                if constexpr (T::C * SIZE == 4) {
                    t.v[n][s] = *reinterpret_cast<const uint4v*>(vb + s * 1024 + lane * 16);
                } else {
                    const uint2v w = *reinterpret_cast<const uint2v*>(vb + s * 512 + lane * 8);
                    t.v[n][s] = uint4v{w[0], w[1], 0, 0};
                }
            }
            if constexpr (Q8) {
                t.ks[n] = *reinterpret_cast<const float4v*>(a.ks + row + 4 * g);
                t.vs[n] = *reinterpret_cast<const float4v*>(a.vs + row + 4 * g);
            }
        }
        float s2[2][4], top = -__builtin_inff();
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float4v s{};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                half8 op;
                if constexpr (!Q8) {
                    op = __builtin_bit_cast(half8, t.k[n][c]);
                } else {
                    const uint4v w = t.k[n][c / 2];
                    const int part = (c / 2 * 64 + 64 <= D) ? c & 1 : 0;
                    op = join(bf16_of_bytes(w[2 * part]), bf16_of_bytes(w[2 * part + 1]));
                }
                s = mfma<MBF>(op, q[c], s);
                if constexpr (QLO) s = mfma<MBF>(op, qlo[c], s);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = s[i] * a.scale2;
                if constexpr (Q8) x *= t.ks[n][i];
                s2[n][i] = k0 + 16 * n + 4 * g + i < keys ? x : -__builtin_inff();
                top = fmaxf(top, s2[n][i]);
            }
        }
        top = wave_xor_max4(top);
        const float m_new = fmaxf(m, top);
        const float base = (m_new == -__builtin_inff() ? 0.f : m_new) - kBias;
        const float alpha = exp2_fast(m - kBias - base);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < DB; ++e) o[e] *= alpha;
        m = m_new;
        float pf[8];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = exp2_fast(s2[n][i] - base);
                l += x;
                if constexpr (Q8) x = k0 + 16 * n + 4 * g + i < keys ? x * t.vs[n][i] : 0.f;
                pf[4 * n + i] = x;
            }
        half8 p, plo;
        two_parts<MBF, !Q8>(pf, p, plo);
        if (!Q8 && k0 + kTile > keys) {  // values behind the last token may be anything: zeros
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int s = 0; s < T::NV; ++s)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int key = k0 + 16 * n + 4 * g + 2 * (w & 1);
                        uint32_t keep = key + 1 < keys ? 0xffffffffu : key < keys ? 0xffffu : 0u;
                        t.v[n][s][w] &= keep;
                    }
        }
#pragma unroll
        for (int e = 0; e < DB; ++e) {
            half8 op;
            const int s = e / T::C, c = e % T::C;
            if constexpr (!Q8) {
                op = join(uint2v{t.v[0][s][2 * c], t.v[0][s][2 * c + 1]}, uint2v{t.v[1][s][2 * c], t.v[1][s][2 * c + 1]});
            } else {
                op = join(bf16_of_bytes(t.v[0][s][c]), bf16_of_bytes(t.v[1][s][c]));
            }
            o[e] = mfma<MBF>(op, p, o[e]);
            o[e] = mfma<MBF>(op, plo, o[e]);
        }
    }

    // the waves' parts, joined in LDS
    l = wave_xor_sum4(l);
    if (g == 0) {
        stat[wave][0][i16] = m;
        stat[wave][1][i16] = bad ? __builtin_nanf("") : l;
    }
    __syncthreads();
    float m_all = -__builtin_inff(), l_all = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m_all = fmaxf(m_all, stat[w][0][i16]);
    const float m_ref = m_all == -__builtin_inff() ? 0.f : m_all;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) l_all += stat[w][1][i16] * exp2_fast(stat[w][0][i16] - m_ref);
    const float mine = exp2_fast(m - m_ref);
#pragma unroll
    for (int e = 0; e < DB; ++e) o[e] *= mine;
#pragma unroll
    for (int half = 2; half >= 1; half /= 2) {
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int e = 0; e < DB; ++e) *reinterpret_cast<float4v*>(&acc[wave - half][i16][16 * e + 4 * g]) = o[e];
        }
        __syncthreads();
        if (wave < half) {
#pragma unroll
            for (int e = 0; e < DB; ++e) o[e] += *reinterpret_cast<const float4v*>(&acc[wave][i16][16 * e + 4 * g]);
        }
        __syncthreads();
    }
    if (wave != 0 || i16 >= rows) return;
    const bool none = len == 0;
    const float inv = 1.f / l_all;
#pragma unroll
    for (int e = 0; e < DB; ++e) {
        float4v r = o[e] * inv;
        if (none) r = float4v{};
        *reinterpret_cast<raw4*>(a.out + (qrow + i16) * D + 16 * e + 4 * g) = act_cvt4<BF>(r);
    }
    if (a.lse != nullptr && g == 0) a.lse[qrow + i16] = none ? -__builtin_inff() : m_all + (__builtin_amdgcn_logf(l_all) - kBias);
}

}  // namespace

}  // namespace clk

using namespace clk;

extern "C" size_t clk_paged_attention_workspace_size(const clk_buffer* q, const clk_buffer* k_cache, const clk_buffer* page_table) {
    return 0;
}

extern "C" int clk_paged_attention(clk_stream stream, const clk_buffer* q, const clk_buffer* k_cache, const clk_buffer* v_cache,
                                   const clk_buffer* k_scale, const clk_buffer* v_scale, const clk_buffer* page_table,
                                   const clk_buffer* lengths, const clk_buffer* out, const clk_buffer* lse, float scale,
                                   int32_t want_lse, void* workspace, size_t workspace_bytes) {
    const char* what = "paged_attention";
    const int act = q != nullptr && q->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {q, page_table, lengths, out, lse};
    const int types[] = {act, CLK_S32, CLK_S32, act, CLK_F32};
    if (int st = check_types(what, bufs, types, 5)) return st;
    CacheShape c;
    if (int st = check_cache(what, k_cache, v_cache, k_scale, v_scale, act, c)) return st;
    if (q->rank != 3 || q->dims[2] != c.D || q->dims[1] < 1 || q->dims[1] % c.heads) {
        return invalid("paged_attention: q must be [B,Hq,D], Hq a multiple of the cache's heads and D its D");
    }
    const int64_t B = q->dims[0], Hq = q->dims[1];
    if (page_table->rank != 2 || page_table->dims[0] != B || page_table->dims[1] < 1) {
        return invalid("paged_attention: page_table must be [B,pages of a sequence]");
    }
    if (lengths->rank != 1 || lengths->dims[0] != B) return invalid("paged_attention: lengths must be [B]");
    if (!same_shape(out, q)) return invalid("paged_attention: out must be like q");
    if (want_lse && (lse->rank != 2 || lse->dims[0] != B || lse->dims[1] != Hq)) return invalid("paged_attention: lse must be [B,Hq]");
    if (!(scale == scale) || scale - scale != 0.f) return invalid("paged_attention: scale must be finite");
    const int64_t G = Hq / c.heads, blocks = (G + 15) / 16;
    if (B > INT32_MAX / (c.heads * blocks) || B * c.heads * blocks >= (1 << 24) || page_table->dims[1] > (1 << 30) / c.page) {
        return invalid("paged_attention: too large");
    }
    if (B > 0 && (!aligned16(q->data) || !aligned16(out->data))) return invalid("paged_attention: q and out must be 16-byte aligned");
    if (B == 0) return ok();
    AttnArgs a{};
    a.q = static_cast<const half_t*>(q->data);
    a.kc = static_cast<const char*>(k_cache->data);
    a.vc = static_cast<const char*>(v_cache->data);
    a.ks = static_cast<const float*>(k_scale->data);
    a.vs = static_cast<const float*>(v_scale->data);
    a.table = static_cast<const int32_t*>(page_table->data);
    a.len = static_cast<const int32_t*>(lengths->data);
    a.out = static_cast<half_t*>(out->data);
    a.lse = want_lse ? static_cast<float*>(lse->data) : nullptr;
    a.B = (int)B;
    a.Hkv = (int)c.heads;
    a.G = (int)G;
    a.blocks = (int)blocks;
    a.per = (int)page_table->dims[1];
    a.pages = (int)c.pages;
    a.page = (int)c.page;
    a.by_page = fast_div(c.page);
    a.by_blocks = fast_div(blocks);
    a.by_hkv = fast_div(c.heads);
    a.scale2 = scale * kLog2e;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    const dim3 grid((unsigned)(B * c.heads * blocks)), block(kWaves * kWave);
    const auto launch = [&](auto d_) {
        constexpr int D = decltype(d_)::value;
        if (act == CLK_BF16) {
            if (c.q8) hipLaunchKernelGGL((paged_attn_kernel<true, true, D>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((paged_attn_kernel<true, false, D>), grid, block, 0, s, a);
        } else {
            if (c.q8) hipLaunchKernelGGL((paged_attn_kernel<false, true, D>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((paged_attn_kernel<false, false, D>), grid, block, 0, s, a);
        }
    };
    switch (c.D) {
    case 32: launch(std::integral_constant<int, 32>()); break;
    case 64: launch(std::integral_constant<int, 64>()); break;
    case 96: launch(std::integral_constant<int, 96>()); break;
    case 128: launch(std::integral_constant<int, 128>()); break;
    case 160: launch(std::integral_constant<int, 160>()); break;
    case 192: launch(std::integral_constant<int, 192>()); break;
    case 224: launch(std::integral_constant<int, 224>()); break;
    default: launch(std::integral_constant<int, 256>()); break;
    }
    stage_mark(s, 1);
    return launch_status(what);
}
