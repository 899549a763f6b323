// Attention of one new token a sequence over a paged key-value cache, for gfx950 (CDNA4). No counterpart in the reference.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[b, h] . k_j), over the length[b] tokens that the sequence's
//   pages hold for the head of keys h / (Hq / Hkv);  lse = log2(sum_j p_j), in the log2 domain
//
// Every cached byte is needed once, which bounds it: 4 Hq / Hkv operations a cached value are far under the matrix
// cores' rate up to some hundred query heads a head of keys.
//
// A wave takes two or four blocks of 16 tokens of the cache (kv_cache.h) at a time, for 16 query heads of one head of keys
// (rows past the group's last are zeros and cost nothing: the cache's bytes are what takes the time):
//   S^T = K Q^T        K's operands are the cache's bytes as they lie; a lane gets tokens 4 g .. + 3 of each block for
//                      query l % 16
//   O^T += V^T P^T     P^T's operand is what the lane holds; V's operand for it is again the cache's bytes
// with the running maximum and sum of a softmax. Both operands come from memory to registers with nothing between.
//
// 256 sequences of 4096 on 8 heads of 128 in bf16 (4.2 GB) take 627 us, 6.7 TB/s, where reading alone reaches 6.9; one of 131071
// (537 MB) 84 + 5, 6.4 TB/s; 61 ragged ones of up to 8192 on 4 heads in 8 bits (167 MB) 36 + 5, 4.7 TB/s: some 3 us
// before the first keys arrive, and the longest parts have 1024 tokens where even shares would have 841; one of 77
// tokens 4.2 us, a launch's time.
#include "kv_cache.h"

#include <algorithm>
#include <type_traits>

namespace clk {

namespace {

typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef int int4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
// Tokens of room for which a workgroup takes an item whole, with nothing to plan or join: one sequence of 512 tokens on 8 heads
// of 128 in bf16 6.4 us, 8.6 in parts; 64 of 512 26.2 and 34.4; but one of 1024 9.6 and 8.6 in parts, of 2048 18.0 and
// 9.6; 64 of 1024 48.3 and 51.5, 256 of 512 94.5 and 91.6. The host knows the table's room, not the lengths: 77
// tokens take 4.0 us with room for 512 and 6.3 with more, whose join has nothing to do.
constexpr int kDirect = 512;

// Blocks of 16 tokens a wave takes at a time, and the tokens of a workgroup's step. (Four blocks, where the registers hold
// them, were slower with 8 bits and the same with 16.)
constexpr int kBlocks = 2;
constexpr int kChunk = kWaves * 16 * kBlocks;

// Workgroups a CU that the kernels' registers are kept for
constexpr int occupancy(int64_t D) { return D <= 64 ? 4 : D <= 128 ? 3 : 2; }
// Sequences, one a lane, up to which each workgroup works out by itself which part of which item it takes
constexpr int kPlanned = 64;
constexpr int kPlanThreads = 256;
constexpr int kMostSplit = 256 * 4 * 3;

// Weights are taken times 2^bias, which their sum has too and which cancels: fp16 ones so that small ones keep their bits (a
// weight of 2^-25 of the largest, of which a long sequence may have millions, would be 0), bf16 ones so that
// sums of values near the type's largest stay in fp32's range: all weights of a sequence are less than 1 together. (A
// factor for the longest would take the bits of values under 2^-100 from short ones.)
template <bool MBF>
__device__ __forceinline__ float bias_of(int len) {
    return MBF ? -(float)(32 - __builtin_clz((uint32_t)max(len, 1))) : 15.f;
}

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
    int B, Hkv, G, blocks, heads;  // G query heads a head of keys, in blocks of 16; heads = Hkv blocks: a sequence's items
    int per, pages, page;
    FastDiv by_page, by_blocks, by_heads;
    float scale2;  // scale log2 e
    // of a split call
    int W;          // workgroups that fill the chip
    float* part_o;  // [2 W][16][D]
    float* part_s;  // [2 W][2][16]: running maximum, sum
    int4v* split;   // [W]: an item in parts, its first part, how many it has, the sequence's length
    int4v* plan;    // of each workgroup: sequence, item of the sequence, part << 16 | parts, place; null: it works that out
    int* meta;      // the items in parts; planned workgroups
};

// A wave-uniform value on the scalar unit, and a scalar load from an array that the kernel does not write: a page's number
// by a vector load would be waited for behind all keys and values in flight.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int scalar_load(const int32_t* p, int64_t i) {
    return reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p))[i];
}

// Sum over the wave, and inclusive sums, by DPP (a shuffle waits for LDS at each of its six steps)
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);   // row_shr 1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) { return lane_value(wave_scan(v), kWave - 1); }

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

// Eight weights in two 16-bit parts each, 2^-17 of them at most away from their sum (bf16): one would make a result's error
// half a step larger than its own rounding. The matrix cores have time for both.
// ABOVE: the first part is a step below the weight cut off, so that the second is positive too and an infinity among
// the values stays one (a second part of zero or below would make it NaN). The parts are then 2^-15 (bf16) or 2^-21
// away at most. An fp16 weight under kLeastAbove has a first part of zero: attend takes infinities apart there.
constexpr float kLeastAbove = 0x1p-23f;
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

// The infinities among two fp16 values, with a zero for another value
__device__ __forceinline__ uint32_t infinities(uint32_t w) {
    return ((w & 0x7fffu) == 0x7c00u ? w & 0xffffu : 0u) | ((w & 0x7fff0000u) == 0x7c000000u ? w & 0xffff0000u : 0u);
}

// A tile's cached bytes as they were loaded: keys as operands, values as cells of four tokens a channel block
template <bool Q8, int D, int NB>
struct Tile {
    static constexpr int NK = Q8 ? (D + 63) / 64 : D / 32;  // key loads a block
    static constexpr int C = value_group(Q8, D);            // channel blocks a value load
    static constexpr int NV = D / 16 / C;
    uint4v k[NB][NK];
    uint4v v[NB][NV];  // 8-byte loads (Q8, D no multiple of 64) in the low half
    float4v ks[NB], vs[NB];
};

// One item, the query heads 16 rb .. + 15 of head of keys h of sequence b, and tokens of it
struct Span {
    int b, h, rb, rows, from, to, len;  // len: of the sequence
    int64_t qrow;
};
__device__ __forceinline__ Span span_of(const AttnArgs& a, int b, int hr, int from, int to, int len) {
    Span s;
    s.b = b;
    s.h = fdiv(hr, a.by_blocks);
    s.rb = hr - s.h * a.blocks;
    s.rows = min(16, a.G - 16 * s.rb);
    s.qrow = ((int64_t)b * a.Hkv + s.h) * a.G + 16 * s.rb;
    s.from = from;
    s.to = to;
    s.len = len;
    return s;
}

// A wave's running maximum, sum and results: for query l % 16, o[e] channels 16 e + 4 g .. + 3
template <int D>
struct State {
    float4v o[D / 16];
    float m, l;
    bool bad;  // a page that the cache does not have
};

// Where a tile's blocks lie in the cache, in tokens x heads, and whether they hold tokens of the span: a block past it (or on
// a page that the cache does not have, which sets bad) is loaded as zeros, by a buffer of no bytes. The pages' numbers
// are loaded first, all at once.
template <int NB>
struct Pages {
    int page[NB];
};
template <int NB>
__device__ __forceinline__ Pages<NB> pages_of(const AttnArgs& a, const Span& sp, const int32_t* table, int k0) {
    Pages<NB> p;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int at = k0 + 16 * n;
        p.page[n] = scalar_load(table, fdiv(at < sp.to ? at : sp.from, a.by_page));
    }
    return p;
}
struct Where {
    int64_t row;
    bool in;
};
__device__ __forceinline__ Where where_of(const AttnArgs& a, const Span& sp, int at, int page, bool& bad) {
    Where w;
    const bool have = (uint32_t)page < (uint32_t)a.pages;
    bad |= at < sp.to && !have;
    w.in = at < sp.to && have;
    const int in_page = at - fdiv(at, a.by_page) * a.page;
    w.row = w.in ? ((int64_t)page * a.Hkv + sp.h) * a.page + in_page : 0;
    return w;
}
template <typename P>
__device__ __forceinline__ auto rsrc_of(const P* p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<P*>(p), 0, bytes, 0x00020000);
}
template <bool NT, typename Rsrc>
__device__ __forceinline__ uint4v load16(Rsrc r, uint32_t off) {
    return __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, NT ? 2 : 0));
}
template <bool NT, typename Rsrc>
__device__ __forceinline__ uint4v load8(Rsrc r, uint32_t off) {
    const uint2v w = __builtin_bit_cast(uint2v, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, NT ? 2 : 0));
    return uint4v{w[0], w[1], 0, 0};
}
template <bool NT, bool Q8, int D, int NB>
__device__ __forceinline__ void load_keys(const AttnArgs& a, const Where (&at)[NB], int lane, Tile<Q8, D, NB>& t) {
    constexpr int SIZE = Q8 ? 1 : 2;
    const int i16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const auto r = rsrc_of(a.kc + at[n].row * (D * SIZE), at[n].in ? 16 * D * SIZE : 0);
#pragma unroll
        for (int s = 0; s < t.NK; ++s) {
            if (!Q8 || s * 64 + 64 <= D) t.k[n][s] = load16<NT>(r, lane * 16 + s * 1024);
            else t.k[n][s] = load8<NT>(r, (g >> 1) * 256 + i16 * 16 + (g & 1) * 8 + s * 1024);
        }
        if constexpr (Q8) t.ks[n] = __builtin_bit_cast(float4v, load16<NT>(rsrc_of(a.ks + at[n].row, at[n].in ? 64 : 0), g * 16));
    }
}
template <bool NT, bool Q8, int D, int NB>
__device__ __forceinline__ void load_values(const AttnArgs& a, const Where (&at)[NB], int lane, Tile<Q8, D, NB>& t) {
    constexpr int SIZE = Q8 ? 1 : 2;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const auto r = rsrc_of(a.vc + at[n].row * (D * SIZE), at[n].in ? 16 * D * SIZE : 0);
#pragma unroll
        for (int s = 0; s < t.NV; ++s) {
            if constexpr (Tile<Q8, D, NB>::C * SIZE == 4) t.v[n][s] = load16<NT>(r, lane * 16 + s * 1024);
            else t.v[n][s] = load8<NT>(r, lane * 8 + s * 512);
        }
        if constexpr (Q8) t.vs[n] = __builtin_bit_cast(float4v, load16<NT>(rsrc_of(a.vs + at[n].row, at[n].in ? 64 : 0), (lane >> 4) * 16));
    }
}

// The wave's tiles of a span: every kWaves-th. The next tile's keys are loaded as soon as this one's scores have been
// computed, into the same registers, and its values as soon as the results have: each load has half a tile's work to arrive in.
template <bool BF, bool Q8, bool NT, int D>
__device__ __forceinline__ void attend(const AttnArgs& a, const Span& sp, int wave, State<D>& st) {
    constexpr int NB = kBlocks;
    typedef Tile<Q8, D, NB> T;
    constexpr int KS = D / 32, DB = D / 16, TILE = 16 * NB, STEP = kWaves * TILE;
    constexpr bool MBF = BF || Q8;   // the products' operands are bf16
    constexpr bool QLO = Q8 && !BF;  // fp16 queries in two bf16 parts, which is exact
    const int lane = threadIdx.x % kWave, i16 = lane & 15, g = lane >> 4, keys = sp.to;
    const float bias = bias_of<MBF>(sp.len);
    const int32_t* table = a.table + (int64_t)sp.b * a.per;

    // the queries' operands; channels in the order of the keys'
    half8 q[KS], qlo[QLO ? KS : 1];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const bool pair = Q8 && (s / 2 * 64 + 64 <= D);
        const int d = pair ? s / 2 * 64 + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
        uint4v raw{};
        if (i16 < sp.rows) raw = *reinterpret_cast<const uint4v*>(a.q + (sp.qrow + i16) * D + d);
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

#pragma unroll
    for (int e = 0; e < DB; ++e) st.o[e] = float4v{};
    st.m = -__builtin_inff();
    st.l = 0.f;
    st.bad = false;

    int k0 = sp.from + wave * TILE;
    if (k0 >= keys) return;
    T t;
    Where at[NB];
    Pages<NB> pages = pages_of<NB>(a, sp, table, k0);
#pragma unroll
    for (int n = 0; n < NB; ++n) at[n] = where_of(a, sp, k0 + 16 * n, pages.page[n], st.bad);
    load_keys<NT, Q8, D, NB>(a, at, lane, t);
    load_values<NT, Q8, D, NB>(a, at, lane, t);
    for (;;) {
        pages = pages_of<NB>(a, sp, table, k0 + STEP);
        float s2[NB][4], top = -__builtin_inff();
#pragma unroll
        for (int n = 0; n < NB; ++n) {
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
#pragma unroll
        for (int n = 0; n < NB; ++n) at[n] = where_of(a, sp, k0 + STEP + 16 * n, pages.page[n], st.bad);
        load_keys<NT, Q8, D, NB>(a, at, lane, t);
        top = wave_xor_max4(top);
        if (__any(top > st.m)) {
            const float m_new = fmaxf(st.m, top);
            const float alpha = m_new == st.m ? 1.f : exp2_fast(st.m - m_new);
            st.l *= alpha;
#pragma unroll
            for (int e = 0; e < DB; ++e) st.o[e] *= alpha;
            st.m = m_new;
        }
        const float base = (st.m == -__builtin_inff() ? 0.f : st.m) - bias;
        if (!Q8 && k0 + TILE > keys) {  // values behind the last token may be anything: zeros
#pragma unroll
            for (int n = 0; n < NB; ++n)
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
        for (int n = 0; n < NB; n += 2) {
            float pf[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = exp2_fast(s2[n + i / 4][i % 4] - base);
                st.l += x;
                if constexpr (Q8) x = k0 + 16 * (n + i / 4) + 4 * g + i % 4 < keys ? x * t.vs[n + i / 4][i % 4] : 0.f;
                pf[i] = x;
            }
            half8 p, plo;
            two_parts<MBF, !Q8>(pf, p, plo);
            if constexpr (!MBF) {
                // Where a first part is zero an infinity would become NaN: infinities are then multiplied by a weight of 1,
                // by themselves. (Bits less one put zeros, and what no token has, on top.)
                uint32_t least = ~0u;
#pragma unroll
                for (int i = 0; i < 8; ++i) least = min(least, __builtin_bit_cast(uint32_t, pf[i]) - 1);
                if (__any(least < __builtin_bit_cast(uint32_t, kLeastAbove) - 1)) {
                    half8 one;
#pragma unroll
                    for (int i = 0; i < 8; ++i) one[i] = pf[i] == 0.f ? (half_t)0.f : (half_t)1.f;
#pragma unroll
                    for (int e = 0; e < DB; ++e) {
                        uint4v inf;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            auto& v = t.v[n + w / 2][e / T::C];
                            const int at = 2 * (e % T::C) + w % 2;
                            inf[w] = infinities(v[at]);
                            v[at] ^= inf[w];
                        }
                        st.o[e] = mfma<MBF>(__builtin_bit_cast(half8, inf), one, st.o[e]);
                        __builtin_amdgcn_sched_barrier(0);  // (one after another, which takes no further registers)
                    }
                }
                // (Without this the compiler, ROCm 7.2's, joins the operands below of registers that it has used again.)
#pragma unroll
                for (int b = n; b < n + 2; ++b)
#pragma unroll
                    for (int s = 0; s < T::NV; ++s) asm volatile("" : "+v"(t.v[b][s]));
            }
#pragma unroll
            for (int e = 0; e < DB; ++e) {
                half8 op;
                const int s = e / T::C, c = e % T::C;
                if constexpr (!Q8) {
                    op = join(uint2v{t.v[n][s][2 * c], t.v[n][s][2 * c + 1]}, uint2v{t.v[n + 1][s][2 * c], t.v[n + 1][s][2 * c + 1]});
                } else {
                    op = join(bf16_of_bytes(t.v[n][s][c]), bf16_of_bytes(t.v[n + 1][s][c]));
                }
                st.o[e] = mfma<MBF>(op, p, st.o[e]);
                st.o[e] = mfma<MBF>(op, plo, st.o[e]);
            }
        }
        k0 += STEP;
        if (k0 >= keys) return;
        load_values<NT, Q8, D, NB>(a, at, lane, t);
    }
}

// What the workgroup's waves have of a span, summed: each of the rows' channels by one thread, four at a time, as results
// (part_o null) or as a part for paged_attn_join_kernel. One barrier.
template <int D>
struct WaveShare {
    float stat[kWaves][2][16];
    float acc[kWaves][16][D + 4];
};
template <bool BF, bool MBF, int D>
__device__ __forceinline__ void join_waves(const AttnArgs& a, const Span& sp, const State<D>& st, int wave, WaveShare<D>& share,
                                           float* part_o, float* part_s) {
    const int lane = threadIdx.x % kWave, i16 = lane & 15, g = lane >> 4;
    const float l = wave_xor_sum4(st.l);
    if (i16 < sp.rows) {
        if (g == 0) {
            share.stat[wave][0][i16] = st.m;
            share.stat[wave][1][i16] = st.bad ? __builtin_nanf("") : l;
        }
#pragma unroll
        for (int e = 0; e < D / 16; ++e) *reinterpret_cast<float4v*>(&share.acc[wave][i16][16 * e + 4 * g]) = st.o[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < sp.rows * (D / 4); i += kWaves * kWave) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4));
        float m = share.stat[0][0][r], sum = 0.f;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, share.stat[w][0][r]);
        const float ref = m == -__builtin_inff() ? 0.f : m;
        float4v o{};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = exp2_fast(share.stat[w][0][r] - ref);
            sum += f * share.stat[w][1][r];
            o += f * *reinterpret_cast<const float4v*>(&share.acc[w][r][d]);
        }
        if (part_o != nullptr) {
            *reinterpret_cast<float4v*>(part_o + r * D + d) = o;
            if (d == 0) {
                part_s[r] = m;
                part_s[16 + r] = sum;
            }
        } else {
            *reinterpret_cast<raw4*>(a.out + (sp.qrow + r) * D + d) = act_cvt4<BF>(o * (1.f / sum));
            if (a.lse != nullptr && d == 0) a.lse[sp.qrow + r] = m + (__builtin_amdgcn_logf(sum) - bias_of<MBF>(sp.len));
        }
    }
}

// Results of a sequence of no tokens (zeros), or of one with more than its pages hold (NaN)
template <bool BF, int D>
__device__ __forceinline__ void finish_empty(const AttnArgs& a, const Span& sp, bool bad) {
    const float v = bad ? __builtin_nanf("") : 0.f;
    const raw4 r = act_cvt4<BF>(float4v{v, v, v, v});
    for (int i = threadIdx.x; i < sp.rows * (D / 4); i += kWaves * kWave) *reinterpret_cast<raw4*>(a.out + sp.qrow * D + 4 * i) = r;
    if (a.lse != nullptr && (int)threadIdx.x < sp.rows) a.lse[sp.qrow + threadIdx.x] = bad ? v : -__builtin_inff();
}

// A workgroup an item: for caches that no sequence can have more than kDirect tokens in
template <bool BF, bool Q8, int D>
__global__ __launch_bounds__(kWaves* kWave, occupancy(D)) void paged_attn_kernel(AttnArgs a) {
    __shared__ WaveShare<D> share;
    const int wave = uniform((int)(threadIdx.x / kWave));
    const int b = fdiv(blockIdx.x, a.by_heads);
    const int len = scalar_load(a.len, b);
    const bool bad = (int64_t)len > (int64_t)a.per * a.page;
    const Span sp = span_of(a, b, blockIdx.x - b * a.heads, 0, len, len);
    if (bad || len <= 0) {
        finish_empty<BF, D>(a, sp, bad);
        return;
    }
    State<D> st;
    attend<BF, Q8, false, D>(a, sp, wave, st);
    join_waves<BF, BF || Q8, D>(a, sp, st, wave, share, nullptr, nullptr);
}

// Chunks of a sequence
__device__ __forceinline__ int chunks_in(const AttnArgs& a, int len) {
    return len <= 0 || (int64_t)len > (int64_t)a.per * a.page ? 0 : (len + kChunk - 1) / kChunk;
}
// Parts of a sequence's items, c chunks each at most; a sequence of no tokens has one, which writes its results
__device__ __forceinline__ int parts_in(int chunks, int c) { return chunks <= c ? 1 : (chunks - 1) / c + 1; }

// Items in parts of about as many chunks, however the lengths differ, one a workgroup. c, the most chunks of a part, is the
// least with which W workgroups, all at once on the chip, are enough, but at most what room = W - min(items, W / 2)
// workgroups would need if parts were as long as that to the last (with so many items that theirs do not fit on the
// chip at once anyway). Items of one part are finished at once; parts of the others are numbered through and left for
// paged_attn_join_kernel.
// (All chunks in W equal runs, one a workgroup, where a run could end one item and begin the next, was more even but a
// workgroup had two short spans as often as one, each with its chain of loads: 61 sequences of up to 8192 over 8 bits
// took 43 us.)
//
// over(f) calls f for the caller's share of the lengths, sum adds up what the callers have.
template <typename Over, typename Sum>
__device__ __forceinline__ int chunks_of_parts(const AttnArgs& a, Over over, Sum sum) {
    int64_t mine = 0;
    over([&](int len) { mine += chunks_in(a, len); });
    const int64_t items = (int64_t)a.B * a.heads, room = a.W - min<int64_t>(items, a.W / 2);
    const int64_t U = (((int64_t)sum((uint32_t)(mine >> 24)) << 24) + sum((uint32_t)mine & 0xffffffu)) * a.heads;
    const auto most = [&](int64_t groups) {
        if (U < 1 << 30) return max(1, (int)(((uint32_t)U + (uint32_t)groups - 1) / (uint32_t)groups));
        return (int)min<int64_t>(1 << 30, (U + groups - 1) / groups);
    };
    int c = most(room);
    if (items > a.W) return c;  // which has as many parts at least
    for (int low = most(a.W); low < c;) {  // the least c, or this one, with at most W parts
        const int mid = low + (c - low) / 2;
        int64_t parts = 0;
        over([&](int len) { parts += parts_in(chunks_in(a, len), mid); });
        if ((int64_t)sum((uint32_t)min<int64_t>(parts, 1 << 24)) * a.heads <= a.W) c = mid;  // (a lane's 2^24 are too many)
        else low = mid + 1;
    }
    return c;
}
// A sequence's workgroups, and below them its parts (16 bits) and items in parts
struct Count {
    uint32_t groups, parts;
};
__device__ __forceinline__ Count count_of(const AttnArgs& a, int len, int c) {
    const uint32_t k = (uint32_t)parts_in(chunks_in(a, len), c), groups = k * (uint32_t)a.heads;
    return Count{groups, k > 1 ? groups << 16 | (uint32_t)a.heads : 0};
}

// What a workgroup does: part j of the k of an item, and the place of its results where k > 1
struct Work {
    int b, hr, j, k, slot, len;
};

// The work of paged_attn_split_kernel's workgroups where there are so many sequences that it would take each of them long
// to go through: 256 sequences a workgroup, which counts those before by itself.
__global__ __launch_bounds__(kPlanThreads) void paged_attn_plan_kernel(AttnArgs a) {
    constexpr int WAVES = kPlanThreads / kWave;
    __shared__ uint32_t red[2][WAVES];
    const int tid = threadIdx.x, wave = uniform((int)(tid / kWave)), first = blockIdx.x * kPlanThreads;
    int turn = 0;
    const auto waves = [&](uint32_t v, uint32_t& below) {  // sum of v over all threads, and over the waves below
        v = wave_sum(v);
        if (tid % kWave == 0) red[turn][wave] = v;
        __syncthreads();
        uint32_t all = 0;
        below = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w == wave) below = all;
            all += red[turn][w];
        }
        turn ^= 1;  // one barrier a sum: the next goes through the other half
        return all;
    };
    uint32_t below;
    const auto sum = [&](uint32_t v) { return waves(v, below); };
    const int c = chunks_of_parts(a, [&](auto f) {
        for (int b = tid; b < a.B; b += kPlanThreads) f(a.len[b]);
    }, sum);
    Count before{0, 0};
    for (int b = tid; b < first; b += kPlanThreads) {
        const Count n = count_of(a, a.len[b], c);
        before.groups += n.groups;
        before.parts += n.parts;
    }
    before.groups = sum(before.groups);
    before.parts = sum(before.parts);
    const int b = first + tid, len = b < a.B ? a.len[b] : 0;
    const Count n = b < a.B ? count_of(a, len, c) : Count{0, 0};
    uint32_t groups_below, parts_below;
    const uint32_t groups = before.groups + waves(n.groups, groups_below), parts = before.parts + waves(n.parts, parts_below);
    if (blockIdx.x == gridDim.x - 1 && tid == 0) {
        a.meta[0] = (int)(parts & 0xffffu);
        a.meta[1] = (int)groups;
    }
    const int at = (int)(before.groups + groups_below + wave_scan(n.groups) - n.groups);
    const uint32_t p = before.parts + parts_below + wave_scan(n.parts) - n.parts;
    if (b >= a.B) return;
    const int k = (int)n.groups / a.heads, slot = (int)(p >> 16);
    for (int hr = 0, i = 0; hr < a.heads; ++hr) {
        if (k > 1) a.split[(p & 0xffffu) + hr] = int4v{b * a.heads + hr, slot + i, k, len};
        for (int j = 0; j < k; ++j, ++i) a.plan[at + i] = int4v{b, hr, j << 16 | k, slot + i};
    }
}

// The workgroup's work as each works it out for itself; false: it has none
__device__ __forceinline__ bool work_of(const AttnArgs& a, Work& work) {
    const int tid = threadIdx.x, lane = tid % kWave;
    // each wave looks at all lengths by itself: lane's are b0 .. b1 - 1, and the first is kept
    const int per = (a.B + kWave - 1) / kWave, b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B);
    const int len0 = b0 < b1 ? a.len[b0] : -1;
    const auto over = [&](auto f) {  // f of the lane's lengths, in order
        for (int b = b0; b < b1; ++b) f(b == b0 ? len0 : a.len[b]);
    };
    const int c = chunks_of_parts(a, over, [](uint32_t v) { return wave_sum(v); });
    uint32_t groups = 0, parts = 0;
    over([&](int len) {
        const Count n = count_of(a, len, c);
        groups += n.groups;
        parts += n.parts;
    });
    const uint32_t id = blockIdx.x, groups_to = wave_scan(groups), parts_to = wave_scan(parts);
    if (id == 0 && tid == kWave - 1) a.meta[0] = (int)(parts_to & 0xffffu);
    const uint64_t has = __ballot(groups_to > id);
    if (has == 0) return false;
    const int from = __builtin_ctzll(has);
    uint32_t before = lane_value(groups_to - groups, from), parts_before = lane_value(parts_to - parts, from);
    int b = from * per, len = (int)lane_value((uint32_t)len0, from);
    Count n = count_of(a, len, c);
    while (before + n.groups <= id) {
        before += n.groups;
        parts_before += n.parts;
        len = scalar_load(a.len, ++b);
        n = count_of(a, len, c);
    }
    const int at = (int)(id - before);
    work.b = b;
    work.len = len;
    work.k = parts_in(chunks_in(a, len), c);
    work.hr = at / work.k;
    work.j = at - work.hr * work.k;
    work.slot = (int)(parts_before >> 16) + at;
    if (work.k > 1 && tid == 0 && work.j == 0) a.split[(parts_before & 0xffffu) + work.hr] = int4v{b * a.heads + work.hr, work.slot, work.k, len};
    return true;
}

template <bool BF, bool Q8, bool NT, int D>
__global__ __launch_bounds__(kWaves* kWave, occupancy(D)) void paged_attn_split_kernel(AttnArgs a) {
    __shared__ WaveShare<D> share;
    const int wave = uniform((int)(threadIdx.x / kWave));
    Work work;
    if (a.plan != nullptr) {
        if ((int)blockIdx.x >= scalar_load(a.meta, 1)) return;
        const int32_t* p = reinterpret_cast<const int32_t*>(a.plan);
        const int64_t at = 4 * (int64_t)blockIdx.x;
        const int jk = scalar_load(p, at + 2);
        work = Work{scalar_load(p, at), scalar_load(p, at + 1), jk >> 16, jk & 0xffff, scalar_load(p, at + 3), 0};
        work.len = scalar_load(a.len, work.b);
    } else if (!work_of(a, work)) {
        return;
    }
    // (which the compiler does not see to be one value a wave: it would load through loops over the lanes)
    work = Work{uniform(work.b), uniform(work.hr), uniform(work.j), uniform(work.k), uniform(work.slot), uniform(work.len)};
    const int len = work.len, chunks = chunks_in(a, len), each = (chunks - 1) / work.k + 1;
    const Span sp = span_of(a, work.b, work.hr, work.j * each * kChunk, min(len, (work.j + 1) * each * kChunk), len);
    if (chunks == 0) {
        finish_empty<BF, D>(a, sp, len > 0);
        return;
    }
    float *part_o = nullptr, *part_s = nullptr;
    if (work.k > 1) {
        part_o = a.part_o + (int64_t)work.slot * 16 * D;
        part_s = a.part_s + work.slot * 32;
    }
    State<D> st;
    attend<BF, Q8, NT, D>(a, sp, wave, st);
    join_waves<BF, BF || Q8, D>(a, sp, st, wave, share, part_o, part_s);
}

// An item's parts, in their order: one of its rows (blockIdx.y) a workgroup, its parts dealt to four or eight waves. What it
// waits for is a chain of loads, so the first parts' results are on their way before the weights are known, and eight
// a wave from then on.
template <bool BF, bool MBF, int D, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void paged_attn_join_kernel(AttnArgs a) {
    constexpr int COLS = D <= 128 ? 2 : 4, EARLY = 4, AT_ONCE = 8;  // channels a lane; parts a wave
    typedef float cols __attribute__((ext_vector_type(COLS)));
    __shared__ float weight[kMostSplit + 1];
    __shared__ float red[2][WAVES];
    __shared__ float parts[WAVES][D];
    const int4v item = a.split[blockIdx.x];
    if ((int)blockIdx.x >= a.meta[0]) return;
    const int first = item[1], n = item[2], r = blockIdx.y, b = fdiv(item[0], a.by_heads);
    const Span sp = span_of(a, b, item[0] - b * a.heads, 0, 0, item[3]);
    if (r >= sp.rows) return;
    const int tid = threadIdx.x, wave = uniform((int)(tid / kWave)), lane = tid % kWave;
    const auto slot = [&](int p) { return (int64_t)first + p; };
    const int col = min(lane * COLS, D - COLS);
    const auto part = [&](int p) { return *reinterpret_cast<const cols*>(a.part_o + (slot(p) * 16 + r) * D + col); };
    cols early[EARLY];
#pragma unroll
    for (int k = 0; k < EARLY; ++k) early[k] = part(min(wave + WAVES * k, n - 1));
    float m = -__builtin_inff(), l = 0.f;
    for (int p = tid; p < n; p += WAVES * kWave) {
        weight[p] = a.part_s[slot(p) * 32 + r];
        m = fmaxf(m, weight[p]);
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) m = fmaxf(m, red[0][w]);
    const float ref = m == -__builtin_inff() ? 0.f : m;
    for (int p = tid; p < n; p += WAVES * kWave) {
        const float w = exp2_fast(weight[p] - ref);
        weight[p] = w;
        l += w * a.part_s[slot(p) * 32 + 16 + r];
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) l += __shfl_xor(l, d);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) l += red[1][w];
    cols o{};
#pragma unroll
    for (int k = 0; k < EARLY; ++k) {
        const int p = wave + WAVES * k;
        if (p < n) o += early[k] * weight[p];
    }
    for (int p = wave + WAVES * EARLY; p < n; p += WAVES * AT_ONCE) {
        cols v[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) v[k] = part(min(p + WAVES * k, n - 1));
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (p + WAVES * k < n) o += v[k] * weight[p + WAVES * k];
        }
    }
    *reinterpret_cast<cols*>(&parts[wave][col]) = o;
    __syncthreads();
    if (tid < D / 4) {
        float4v v{};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += *reinterpret_cast<const float4v*>(&parts[w][4 * tid]);
        *reinterpret_cast<raw4*>(a.out + (sp.qrow + r) * D + 4 * tid) = act_cvt4<BF>(v * (1.f / l));
    }
    if (a.lse != nullptr && tid == 0) a.lse[sp.qrow + r] = m + (__builtin_amdgcn_logf(l) - bias_of<MBF>(sp.len));
}

// ---- host -----------------------------------------------------------------------------------

// How a call is run: a rule on the shapes alone, so that results do not depend on the device
struct Plan {
    int64_t items = 0;  // 0: a shape that the entry point rejects
    int W = 0;          // of a split call, 0: a workgroup an item
    int64_t grid = 0;
    size_t o = 0, s = 0, split = 0, meta = 0, plan = 0;
    size_t bytes() const { return o + s + split + meta + plan; }
};
Plan plan_of(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t per, int64_t page) {
    Plan p;
    if (B < 0 || Hq < 1 || Hkv < 1 || Hq % Hkv || per < 1 || page < 16 || page % 16 || D < 32 || D > 256 || D % 32) return p;
    const int64_t blocks = (Hq / Hkv + 15) / 16;
    if (Hkv > 16384 || blocks > 16384 || Hkv * blocks > 16384 || B > (1 << 23) / (Hkv * blocks) || per > (1 << 30) / page) return p;
    p.items = p.grid = B * Hkv * blocks;
    if (per * page > kDirect && B > 0) {
        // One round of workgroups, but where the items nearly make one already, three, so that the long among them are cut
        // finely enough to fill the last round: 256 ragged sequences of up to 4096 on 8 heads of 128 in bf16 232 us, 236 with two
        // and 241 with one; but 61 of up to 8192 on 4 heads in 8 bits 43 with one, 45.5 with two and 47 with three.
        p.W = 256 * occupancy(D) * (p.items > 128 * occupancy(D) ? 3 : 1);
        // With c as the kernel takes it, all chunks / c <= room = W - min(items, W / 2), and an item has under its chunks / c + 1
        // parts: under room + items workgroups; items of two parts and more have over c chunks: under room such items
        // and 2 room parts.
        p.grid = p.W - std::min<int64_t>(p.items, p.W / 2) + p.items;
        p.o = (size_t)2 * p.W * 16 * D * 4;
        p.s = (size_t)2 * p.W * 32 * 4;
        p.split = (size_t)p.W * 16;
        p.meta = 256;
        // Many items of many sequences are dealt out by a launch before (2.5 to 7 us and a gap), of 128 channels in bf16: 1024
        // sequences of 1024 on 8 heads 661 us, 672 without; 4096 ragged ones 906, 2411 without; 256 of 1024 171 with it and
        // without; but 50 ragged ones of up to 4096 61.8, 54.6 without, and 128 of 1024 on one head 21.3, 19.4 without.
        if (B > kPlanned && p.items > 128 * occupancy(D)) p.plan = (size_t)p.grid * 16;
    }
    return p;
}

}  // namespace

}  // namespace clk

using namespace clk;

extern "C" size_t clk_paged_attention_workspace_size(const clk_buffer* q, const clk_buffer* k_cache, const clk_buffer* page_table) {
    for (const clk_buffer* b : {q, k_cache, page_table}) {
        if (b == nullptr || b->dims == nullptr) return 0;
    }
    if (q->rank != 3 || k_cache->rank != 4 || page_table->rank != 2) return 0;
    return plan_of(q->dims[0], q->dims[1], k_cache->dims[1], k_cache->dims[3], page_table->dims[1], k_cache->dims[2]).bytes();
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
    const float scale2 = scale * kLog2e;
    if (!(scale2 - scale2 == 0.f)) return invalid("paged_attention: scale must be finite, times log2(e) too");
    const int64_t G = Hq / c.heads, blocks = (G + 15) / 16;
    const Plan plan = plan_of(B, Hq, c.heads, c.D, page_table->dims[1], c.page);
    if (B > 0 && plan.items == 0) return invalid("paged_attention: too large");
    if (B > 0 && (!aligned16(q->data) || !aligned16(out->data))) return invalid("paged_attention: q and out must be 16-byte aligned");
    if (B == 0) return ok();
    const size_t need = plan.bytes();
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
        return invalid("paged_attention: workspace of " + std::to_string(workspace_bytes) + " bytes, needs " + std::to_string(need));
    }
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return invalid("paged_attention: workspace must be 256-byte aligned");
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
    a.heads = (int)(c.heads * blocks);
    a.by_heads = fast_div(a.heads);
    a.scale2 = scale2;
    a.W = plan.W;
    char* ws = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_s = reinterpret_cast<float*>(ws + plan.o);
    a.split = reinterpret_cast<int4v*>(ws + plan.o + plan.s);
    a.meta = reinterpret_cast<int*>(ws + plan.o + plan.s + plan.split);
    a.plan = plan.plan ? reinterpret_cast<int4v*>(ws + plan.o + plan.s + plan.split + plan.meta) : nullptr;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int stage = 0;
    stage_mark(s, stage);
    const dim3 block(kWaves * kWave);
    // Keys and values of a cache past half of the 256 MB far cache are loaded past the caches, unless more than one workgroup
    // reads them: 61 sequences of 2600 on 4 heads in 8 bits (164 MB) 41.1 us, 44.3 through the caches; 256 of 4096 (4.2 GB)
    // 634 and 704; but 61 of 650 (41 MB, of which a next call finds some) 19.8 and 18.9. The host knows the cache, not how
    // much of it the sequences hold, nor what they share: 8 of 512 in one of 670 MB 10.3 and 11.1, but 61 of 650 in one of
    // 330 MB 19.7 and 19.0, and 64 of 1088 in bf16 that share their first 1024 28.9 and 25.2.
    const bool past = blocks == 1 && 2 * elements(k_cache) * (c.q8 ? 1 : 2) >= (int64_t)1 << 27;
    const auto kernels = [&](auto bf_, auto q8_, auto d_) {
        constexpr bool BF = decltype(bf_)::value, Q8 = decltype(q8_)::value;
        constexpr int D = decltype(d_)::value;
        if (plan.W == 0) {
            hipLaunchKernelGGL((paged_attn_kernel<BF, Q8, D>), dim3((unsigned)plan.grid), block, 0, s, a);
            return;
        }
        if (a.plan != nullptr) {
            hipLaunchKernelGGL(paged_attn_plan_kernel, dim3((unsigned)((B + kPlanThreads - 1) / kPlanThreads)), dim3(kPlanThreads), 0, s, a);
            stage_mark(s, ++stage);
        }
        if (past) hipLaunchKernelGGL((paged_attn_split_kernel<BF, Q8, true, D>), dim3((unsigned)plan.grid), block, 0, s, a);
        else hipLaunchKernelGGL((paged_attn_split_kernel<BF, Q8, false, D>), dim3((unsigned)plan.grid), block, 0, s, a);
        stage_mark(s, ++stage);
        // Eight waves where items have sixteen parts and more: one sequence of 16384 on one head 13.3 -> 11.8 us, of 131071 on eight
        // 90.6 -> 89.7; but 16 ragged ones of up to 4097 on one head (twelve parts) 14.4 -> 15.3.
        const dim3 items((unsigned)std::min<int64_t>(plan.items, plan.W), (unsigned)std::min<int64_t>(G, 16));
        if (16 * plan.items <= plan.W) hipLaunchKernelGGL((paged_attn_join_kernel<BF, BF || Q8, D, 8>), items, dim3(8 * kWave), 0, s, a);
        else hipLaunchKernelGGL((paged_attn_join_kernel<BF, BF || Q8, D, 4>), items, dim3(4 * kWave), 0, s, a);
    };
    const auto launch = [&](auto d_) {
        if (act == CLK_BF16) c.q8 ? kernels(std::true_type(), std::true_type(), d_) : kernels(std::true_type(), std::false_type(), d_);
        else c.q8 ? kernels(std::false_type(), std::true_type(), d_) : kernels(std::false_type(), std::false_type(), d_);
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
    stage_mark(s, ++stage);
    return launch_status(what);
}
