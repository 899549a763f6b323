// Queries, keys and values on their way from a projection to attention, for gfx950 (CDNA4). No counterpart in the
// reference.
//
//   qk_norm_rope        x [T, Hq + 2 Hkv, D]: each query and key head n = x r w, r = 1 / sqrt(mean(x^2) + eps), then its
//                       first R channels rotated in pairs (a, b) -> (a cos - b sin, a sin + b cos) by the angles of
//                       the token's position; values as they are; q, k and v apart
//   qk_norm_rope_bwd    g' = the gradient rotated back, xh = x r, g = g' w: dx = r (g - xh mean(g xh)), dw = sum over tokens
//                       and heads of g' xh
//   qk_norm_rope_cache  the forward with keys and values written into the cache, in 16 bits or as 8-bit rows of a
//                       token's head (each value rounded once, from fp32)
//   kv_cache_write, kv_cache_read  keys and values into the cache as they are, and back
//
// All of them are bound by memory: each value is read once and written once, statistics and products are fp32. At 16384 tokens
// of 48 + 6 + 6 heads of 128 in bf16 the forward takes 100 us (5.0 TB/s of its 503 MB, the rate of a large copy; a
// plain copy in the same pattern 109) and the gradients 151 + 6 (5.0 TB/s of 755 MB); 32771 tokens of 8 heads of 128 take
// 55 us into a 16-bit cache and 48 back (4.9 and 5.6 TB/s of 268 MB each); a prompt of 4099 tokens of 32 + 8 + 8 heads of
// 128 takes 27 us into an 8-bit cache (3.4 TB/s of 92 MB, 4.3 at 32768 tokens); one token 3.7 us.
//
// A head is a group of LG lanes (the power of two at or past D / 8) with 8 channels each, the two halves of its pairs: a
// lane whose channels are rotated by halves holds channels 4 j .. + 3 and R / 2 + 4 j .. + 3, so that pairs never
// cross lanes; all others hold 8 j .. + 7. A workgroup takes 256 / LG tokens of up to HPG heads of one kind, and
// reads a token's cosines and sines once for them. Workgroups go through a token's heads first.
#include "kv_cache.h"
#include "rows8_dev.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(off)  // every kernel rounds alike, whichever of them a call's size picks

namespace clk {

namespace {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
enum { kQuery, kKey, kValue };

struct HeadsArgs {
    const half_t* x;  // [T, Hq + 2 Hkv, D]
    const float* qn;
    const float* kn;
    const float* rope;  // [P, R]
    const int32_t* pos;
    const int32_t* slots;
    half_t* q;
    half_t* k;
    half_t* v;
    void* kc;  // the cache
    void* vc;
    float* ks;
    float* vs;
    const half_t* dq;
    const half_t* dk;
    const half_t* dv;
    half_t* dx;
    float* partial;
    float* dqn;
    float* dkn;
    int64_t T;
    int Hq, Hkv, D, R, P;
    int cq, ck;          // chunks of heads: queries', keys' (values' as keys')
    int parts;           // workgroups a chunk
    int windows;         // workgroups a group of cached heads
    int cached_heads;    // of a step: heads of a group
    FastDiv by_chunks, by_groups;
    int page, slots_end;  // the cache's page, and its tokens
    FastDiv by_page;
    float inv_d, eps;
    bool interleaved;
};

// A lane's 8 channels of its head: two runs of four
struct Lane {
    int c0, c1;
    bool in, turned;
};
__device__ __forceinline__ Lane lane_of(int j, int D, int R, bool interleaved) {
    Lane l;
    l.in = 8 * j < D;
    l.turned = 8 * j < R;
    const bool halves = l.turned && !interleaved;
    l.c0 = !l.in ? 0 : halves ? 4 * j : 8 * j;
    l.c1 = !l.in ? 4 : halves ? R / 2 + 4 * j : 8 * j + 4;
    return l;
}

__device__ __forceinline__ raw8 load_head(const half_t* row, const Lane& l) {
    const raw4 a = *reinterpret_cast<const raw4*>(row + l.c0), b = *reinterpret_cast<const raw4*>(row + l.c1);
    const raw8 v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return l.in ? v : raw8{};
}
__device__ __forceinline__ raw8 load_once(const half_t* row, const Lane& l) {  // 8 channels in a row
    const raw8 v = __builtin_nontemporal_load(reinterpret_cast<const raw8*>(row + l.c0));
    return l.in ? v : raw8{};
}
__device__ __forceinline__ void store_head(half_t* row, const Lane& l, raw8 v) {
    *reinterpret_cast<raw4*>(row + l.c0) = raw4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<raw4*>(row + l.c1) = raw4{v[4], v[5], v[6], v[7]};
}
// Loads and stores through a buffer over a block of tokens: heads past its tokens, lanes past a head and heads past a chunk are
// offsets past the buffer, which read zeros and are not written. (A store in a branch would make the compiler wait for
// all loads and stores in flight at the next use of a load.)
__device__ __forceinline__ auto tokens_buffer(const half_t* first, int64_t tokens, int64_t row_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<half_t*>(first), 0, (uint32_t)(tokens * row_bytes), 0x00020000);
}
constexpr uint32_t kDropped = 0x40000000u;  // a buffer has 256 / LG tokens of 2^13 heads of 16 LG bytes at most; twice this is past it too
struct At {
    uint32_t c0, c1;
};
__device__ __forceinline__ At at_of(const Lane& l, int64_t head, int D) {  // a lane's channels of a head of the buffer
    const uint32_t base = (uint32_t)head * D * 2;
    return At{l.in ? base + 2 * l.c0 : kDropped, l.in ? base + 2 * l.c1 : kDropped};
}
template <typename Rsrc>
__device__ __forceinline__ raw8 load_head(Rsrc r, const At& at, uint32_t more) {
    const auto a = __builtin_amdgcn_raw_buffer_load_b64(r, at.c0 + more, 0, 0), b = __builtin_amdgcn_raw_buffer_load_b64(r, at.c1 + more, 0, 0);
    return __builtin_bit_cast(raw8, uint4v{a[0], a[1], b[0], b[1]});
}
template <typename Rsrc>
__device__ __forceinline__ void store_head(Rsrc r, const At& at, uint32_t more, raw8 v) {
    const uint4v w = __builtin_bit_cast(uint4v, v);
    __builtin_amdgcn_raw_buffer_store_b64(uint2v{w[0], w[1]}, r, at.c0 + more, 0, 0);
    __builtin_amdgcn_raw_buffer_store_b64(uint2v{w[2], w[3]}, r, at.c1 + more, 0, 0);
}
template <bool BF>
__device__ __forceinline__ void floats(raw8 v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = act_get<BF>(__builtin_bit_cast(half8, v), e);
}
__device__ __forceinline__ void load_weight(const float* w, const Lane& l, float (&f)[8]) {
    typedef float4v float4u __attribute__((aligned(4)));
    const float4v a = *reinterpret_cast<const float4u*>(w + l.c0), b = *reinterpret_cast<const float4u*>(w + l.c1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[e] = l.in ? a[e] : 0.f;
        f[4 + e] = l.in ? b[e] : 0.f;
    }
}

// The angles of lane j's four pairs at a position, (1, 0) where it has none; false at a position that the table does not have
struct Angles {
    float4v cos, sin;
};
__device__ __forceinline__ bool load_angles(const HeadsArgs& a, int pos, int j, bool turned, Angles& t) {
    const bool ok = (uint32_t)pos < (uint32_t)a.P;
    const float* row = a.rope + (int64_t)(ok ? pos : 0) * a.R;
    const int at = turned ? 4 * j : 0;
    t.cos = *reinterpret_cast<const float4v*>(row + at);
    t.sin = *reinterpret_cast<const float4v*>(row + a.R / 2 + at);
    return ok;
}

// A lane's pairs by the angles' (cos, sin), or back by (cos, -sin)
template <bool BACK, bool interleaved>
__device__ __forceinline__ void turn_pairs(float (&f)[8], const Angles& t, const Lane& l) {
    float a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = interleaved ? f[2 * e] : f[e];
        b[e] = interleaved ? f[2 * e + 1] : f[4 + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float s = BACK ? -t.sin[e] : t.sin[e];
        const float x = __builtin_fmaf(a[e], t.cos[e], -(b[e] * s)), y = __builtin_fmaf(a[e], s, b[e] * t.cos[e]);
        a[e] = x;
        b[e] = y;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float& x = f[interleaved ? 2 * e : e];
        float& y = f[interleaved ? 2 * e + 1 : 4 + e];
        x = l.turned ? a[e] : x;
        y = l.turned ? b[e] : y;
    }
}

template <bool BACK>
__device__ __forceinline__ void turn(float (&f)[8], const Angles& t, const Lane& l, bool interleaved) {
    if (interleaved) turn_pairs<BACK, true>(f, t, l);
    else turn_pairs<BACK, false>(f, t, l);
}

// f times r = 1 / sqrt(mean(f^2) + eps), and r; NaN where the token has no position. bf16 heads whose squares leave fp32's
// range are taken times a power of two, as rows are (row_shift), which their sum shows: values past 2^46, or none
// past 2^-35 and an eps of next to nothing.
//
// A head has some hundred instructions for its 16 bytes a lane, which at 5 TB/s is about what the vector units have time for:
// the square root's reciprocal is the hardware's with one Newton step (a division and a square root took thirty more).
template <bool BF, int LG>
__device__ __forceinline__ float normalise(float (&f)[8], float inv_d, float eps, bool ok, float otherwise = __builtin_nanf("")) {
    const auto squares = [&] {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(f[e], f[e], s);
        return lanes_sum<LG>(s);
    };
    float ss = squares(), d = 1.f;
    if constexpr (BF) {
        const bool far = !(ss < 0x1p100f) || (ss < 0x1p-70f && eps < 0x1p-100f);
        if (__any(far)) {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[e]));
            m = lanes_max<LG>(m);
            d = far ? row_shift(m, eps) : 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= d;
            ss = squares();
        }
    }
    const float v = __builtin_fmaf(ss, inv_d, eps * d * d), y = __builtin_amdgcn_rsqf(v), e = __builtin_fmaf(-v * y, y, 1.f);
    float r = e == e ? __builtin_fmaf(0.5f * y, e, y) : y;  // (an infinite v has y = 0)
    r = ok ? r : otherwise;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= r;
    return r * d;
}

// The heads of workgroup row `chunk`: their kind, the first of them among their kind, and how many
struct Heads {
    int kind, first, count;
};
template <int HPG>
__device__ __forceinline__ Heads heads_of(const HeadsArgs& a, int chunk) {
    Heads h;
    h.kind = chunk < a.cq ? kQuery : chunk < a.cq + a.ck ? kKey : kValue;
    const int i = h.kind == kQuery ? chunk : h.kind == kKey ? chunk - a.cq : chunk - a.cq - a.ck;
    h.first = i * HPG;
    h.count = min(HPG, (h.kind == kQuery ? a.Hq : a.Hkv) - h.first);
    return h;
}
__device__ __forceinline__ int head_at(const HeadsArgs& a, int kind) {
    return kind == kQuery ? 0 : kind == kKey ? a.Hq : a.Hq + a.Hkv;
}

// ---- the cache ------------------------------------------------------------------------------

// Where a token's head lies: its block, and its row in it
struct Place {
    int64_t block;  // in values
    int64_t scale;
    int t;
};
__device__ __forceinline__ Place place_of(const HeadsArgs& a, int slot, int head) {
    const int page = fdiv(slot, a.by_page), in = slot - page * a.page;
    const int64_t row = (int64_t)page * a.Hkv + head;
    return Place{(row * a.page + (in & ~15)) * a.D, row * a.page + in, in & 15};
}

// A lane's 8 channels of a key (l) or value (8 j ..) into the cache, in 16 bits
__device__ __forceinline__ void cache_key16(void* kc, const Place& p, const Lane& l, raw8 v) {
    uint16_t* at = static_cast<uint16_t*>(kc) + p.block;
    *reinterpret_cast<raw4*>(at + key_place(false, p.t, l.c0)) = raw4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<raw4*>(at + key_place(false, p.t, l.c1)) = raw4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void cache_value16(void* vc, const Place& p, int c, raw8 v) {
    uint16_t* at = static_cast<uint16_t*>(vc) + p.block + value_place(2, p.t, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) at[8 * e] = v[e];
}
// and as 8-bit rows: f in fp32, of 16-bit values where IN16. Every lane of the group comes here.
template <int LG, bool IN16>
__device__ __forceinline__ uint2v to_row8(const float (&f)[8], float& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[e]));
    float top, inv;
    row_scale(lanes_max<LG>(m), 1.f, top, inv, scale);
    return quant8<IN16>(f, top, inv);
}
__device__ __forceinline__ void cache_key8(void* kc, const Place& p, const Lane& l, uint2v w) {
    int8_t* at = static_cast<int8_t*>(kc) + p.block;
    *reinterpret_cast<uint32_t*>(at + key_place(true, p.t, l.c0)) = w[0];
    *reinterpret_cast<uint32_t*>(at + key_place(true, p.t, l.c1)) = w[1];
}
__device__ __forceinline__ void cache_value8(void* vc, const Place& p, int group, int c, uint2v w) {
    int8_t* at = static_cast<int8_t*>(vc) + p.block + value_place(group, p.t, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) at[4 * group * e] = (int8_t)(w[e >> 2] >> 8 * (e & 3));
}

// ---- forward --------------------------------------------------------------------------------

// A query's or key's 8 channels (f) normed, weighted and rotated; NaN where the token has no position
template <bool BF, int LG>
__device__ __forceinline__ void norm_rope(const HeadsArgs& a, float (&f)[8], const float (&w)[8], const Angles& angles, bool ok, const Lane& l) {
    normalise<BF, LG>(f, a.inv_d, a.eps, ok);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= w[e];
    turn<false>(f, angles, l, a.interleaved);
}

// Heads apart: up to HPG of them (h), normed and rotated, or values copied, for the tokens from block 256 / LG on and
// every a.parts-th such block
template <bool BF, int LG, int HPG, bool NORM>
__device__ __forceinline__ void heads_apart(const HeadsArgs& a, int block, const Heads& h) {
    constexpr int TOKENS = kThreads / LG;
    const int j = threadIdx.x % LG, sub = threadIdx.x / LG;
    const Lane l = lane_of(j, a.D, NORM ? a.R : 0, a.interleaved);
    const int H = a.Hq + 2 * a.Hkv, mine = h.kind == kQuery ? a.Hq : a.Hkv;
    half_t* out = h.kind == kQuery ? a.q : h.kind == kKey ? a.k : a.v;
    const At from = at_of(l, (int64_t)sub * H + head_at(a, h.kind) + h.first, a.D), to = at_of(l, (int64_t)sub * mine + h.first, a.D);
    const auto more = [&](int i) { return i < h.count ? (uint32_t)(i * a.D * 2) : kDropped; };
    float w[8];
    if constexpr (NORM) load_weight(h.kind == kQuery ? a.qn : a.kn, l, w);
    for (int64_t t0 = (int64_t)block * TOKENS; t0 < a.T; t0 += (int64_t)a.parts * TOKENS) {
        const int64_t tokens = min<int64_t>(TOKENS, a.T - t0);
        const auto x = tokens_buffer(a.x + t0 * H * a.D, tokens, (int64_t)H * a.D * 2);
        const auto y = tokens_buffer(out + t0 * mine * a.D, tokens, (int64_t)mine * a.D * 2);
        raw8 raw[HPG];
#pragma unroll
        for (int i = 0; i < HPG; ++i) raw[i] = load_head(x, from, more(i));
        Angles angles;
        bool ok = true;
        if constexpr (NORM) ok = load_angles(a, a.pos[t0 + min<int64_t>(sub, tokens - 1)], j, l.turned, angles);
#pragma unroll
        for (int i = 0; i < HPG; ++i) {
            if constexpr (NORM) {
                float f[8];
                floats<BF>(raw[i], f);
                norm_rope<BF, LG>(a, f, w, angles, ok, l);
                raw[i] = act_cvt8<BF>(f);
            }
            store_head(y, to, more(i), raw[i]);
        }
    }
}

template <bool BF, int LG, int HPG>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(HeadsArgs a) {
    const int block = fdiv(blockIdx.x, a.by_chunks);
    const Heads h = heads_of<HPG>(a, blockIdx.x - block * a.by_chunks.d);
    if (h.kind == kValue) heads_apart<BF, LG, HPG, false>(a, block, h);
    else heads_apart<BF, LG, HPG, true>(a, block, h);
}

// ---- backward -------------------------------------------------------------------------------

// Heads a workgroup row: 151 us at the size above, 168 with two. A workgroup goes on to further tokens, so that the weights'
// gradients have one partial row a workgroup, which are summed in a fixed order, without atomics.
constexpr int kBwdHeads = 4;

template <bool BF, int LG>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_bwd_kernel(HeadsArgs a) {
    constexpr int TOKENS = kThreads / LG, HPG = kBwdHeads;
    __shared__ float sums[TOKENS][LG * 8 + 1];
    const int j = threadIdx.x % LG, sub = threadIdx.x / LG;
    const int block = fdiv(blockIdx.x, a.by_chunks), chunk = blockIdx.x - block * a.by_chunks.d;
    const Heads h = heads_of<HPG>(a, chunk);
    const Lane l = lane_of(j, a.D, h.kind == kValue ? 0 : a.R, a.interleaved);
    const int H = a.Hq + 2 * a.Hkv, mine = h.kind == kQuery ? a.Hq : a.Hkv;
    const half_t* dy = h.kind == kQuery ? a.dq : h.kind == kKey ? a.dk : a.dv;
    const At at = at_of(l, (int64_t)sub * H + head_at(a, h.kind) + h.first, a.D), g_at = at_of(l, (int64_t)sub * mine + h.first, a.D);
    const auto more = [&](int i) { return i < h.count ? (uint32_t)(i * a.D * 2) : kDropped; };
    float w[8], dw[8] = {};
    if (h.kind != kValue) load_weight(h.kind == kQuery ? a.qn : a.kn, l, w);
    for (int64_t t0 = (int64_t)block * TOKENS; t0 < a.T; t0 += (int64_t)a.parts * TOKENS) {
        const int64_t tokens = min<int64_t>(TOKENS, a.T - t0);
        const auto x = tokens_buffer(a.x + t0 * H * a.D, tokens, (int64_t)H * a.D * 2);
        const auto y = tokens_buffer(dy + t0 * mine * a.D, tokens, (int64_t)mine * a.D * 2);
        const auto dx = tokens_buffer(a.dx + t0 * H * a.D, tokens, (int64_t)H * a.D * 2);
        raw8 raw[HPG], graw[HPG];
#pragma unroll
        for (int i = 0; i < HPG; ++i) {
            if (h.kind != kValue) raw[i] = load_head(x, at, more(i));
            graw[i] = load_head(y, g_at, more(i));
        }
        Angles angles;
        bool ok = true;
        if (h.kind != kValue) ok = load_angles(a, a.pos[t0 + min<int64_t>(sub, tokens - 1)], j, l.turned, angles);
#pragma unroll
        for (int i = 0; i < HPG; ++i) {
            raw8 o = graw[i];
            if (h.kind != kValue) {
                float f[8], g[8], dot = 0.f;
                floats<BF>(raw[i], f);
                floats<BF>(graw[i], g);
                const bool real = sub < tokens && i < h.count;  // what is none counts as zeros, whatever eps is
                const float r = normalise<BF, LG>(f, a.inv_d, a.eps, ok && real, real ? __builtin_nanf("") : 0.f);
                turn<true>(g, angles, l, a.interleaved);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    dw[e] = __builtin_fmaf(g[e], f[e], dw[e]);
                    g[e] *= w[e];
                    dot = __builtin_fmaf(g[e], f[e], dot);
                }
                dot = lanes_sum<LG>(dot) * a.inv_d;
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = r * __builtin_fmaf(-f[e], dot, g[e]);
                o = act_cvt8<BF>(g);
            }
            store_head(dx, at, more(i), o);
        }
    }
    if (h.kind == kValue) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (l.in) {
            sums[sub][l.c0 + e] = dw[e];
            sums[sub][l.c1 + e] = dw[4 + e];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.D; c += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) s += sums[i][c];
        a.partial[((int64_t)chunk * a.parts + block) * a.D + c] = s;
    }
}

// dqn and dkn (blockIdx.y): the sums of their partial rows, 64 interleaved groups of them, each in order, then the
// groups in order: 1536 rows of 128 take three loads of eight rows in a row a thread, 6 us.
constexpr int kDwGroups = 64;
__global__ __launch_bounds__(16 * kDwGroups) void qk_norm_dw_kernel(HeadsArgs a) {
    __shared__ float sums[kDwGroups][17];
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
    const int first = blockIdx.y ? a.cq * a.parts : 0, n = (blockIdx.y ? a.ck : a.cq) * a.parts;
    float v = 0.f;
    if (c < a.D) {
        const float* p = a.partial + (int64_t)first * a.D + c;
        int i = grp;
        for (; i + 7 * kDwGroups < n; i += 8 * kDwGroups) {
            float u[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) u[k] = p[(int64_t)(i + kDwGroups * k) * a.D];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += u[k];
        }
        for (; i < n; i += kDwGroups) v += p[(int64_t)i * a.D];
    }
    sums[grp][col] = v;
    __syncthreads();
    if (grp == 0 && c < a.D) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kDwGroups; ++i) t += sums[i][col];
        (blockIdx.y ? a.dkn : a.dqn)[c] = t;
    }
}

// ---- cache in, cache out --------------------------------------------------------------------

// What goes token by token into a block of the cache touches 16 bytes (keys) or 2 (values) here and there: 134 MB of keys and
// values in 16 bits took 227 us in and out again so, and 100 now. Tokens that fill a block move together.
//
// Sixteen tokens of a call from 16 w on, as the cache sees them. Where a block of the cache is filled by sixteen tokens in a
// row, whichever token it begins with, the workgroup that has its first token moves it whole, with stores (or loads) of
// whole lines; the other tokens go one by one.
struct Window {
    int first;      // the token that a whole block begins with, from 16 w on; -1: none does
    uint32_t rest;  // the tokens that go one by one (one bit each, from 16 w on)
};
__device__ __forceinline__ Window window_of(const HeadsArgs& a, int64_t t0) {
    const int64_t t = t0 - 15 + (int)(threadIdx.x % kWave);  // the wave's lanes: 15 tokens before, 16, 15 after
    const auto slot_at = [&](int64_t i) { return i >= 0 && i < a.T ? a.slots[i] : -1; };
    const int slot = slot_at(t), after = slot_at(t + 1);
    const bool live = (uint32_t)slot < (uint32_t)a.slots_end;
    const uint64_t all = __ballot(live), begins = __ballot(live && slot % kCacheBlock == 0);
    uint64_t run = __ballot(live && after == slot + 1);  // the next token follows; then the next 2, 4, 8 and 15 do
    run &= run >> 1;
    run &= run >> 2;
    run &= run >> 4;
    const uint64_t whole = begins & run & run >> 7;
    uint64_t covered = whole | whole << 1;
    covered |= covered << 2;
    covered |= covered << 4;
    covered |= covered << 8;
    const uint32_t mine = (uint32_t)(whole >> 15) & 0xffffu;  // one at most: the other tokens of a block begin none
    return Window{mine ? __builtin_ctz(mine) : -1, (uint32_t)((all & ~covered) >> 15) & 0xffffu};
}

// Heads a workgroup moves for its 16 tokens, and the rounds it needs for them
template <int LG>
constexpr int kHeadsAtOnce = kThreads / LG / 16 > 0 ? kThreads / LG / 16 : 1;
template <int LG>
constexpr int kRounds = LG * 16 > kThreads ? LG * 16 / kThreads : 1;

// A block of 16 tokens as rows in LDS, 16 bytes between rows more than they have
template <int LG, bool Q8>
struct BlockRows {
    static constexpr int ROW = 8 * LG * (Q8 ? 1 : 2) + 16;
    char rows[kHeadsAtOnce<LG>][16][ROW];
};

// Four tokens of C channels of a block's values, from rows or to them: unit u of a head has channels 16 (C b + e) + i of tokens
// 4 g + j, with u = (4 b + g) 16 + i
template <int C, typename F>
__device__ __forceinline__ void value_unit(int u, F f) {
    const int i = u & 15, g = u >> 4 & 3, b = u >> 6;
#pragma unroll
    for (int e = 0; e < C; ++e)
#pragma unroll
        for (int j = 0; j < 4; ++j) f(4 * e + j, 4 * g + j, 16 * (C * b + e) + i);
}

// A lane's 8 channels of a key and a value: as they come, and as the cache holds them
struct Pair {
    raw8 key, value;
};
struct Pair8 {
    uint2v key, value;
    float key_scale, value_scale;
};
struct Turn {  // a token's angles
    Angles angles;
    bool ok;
};
// What a token's heads of keys and values come from: the projection's row (STEP), or k and v
template <bool STEP>
__device__ __forceinline__ Pair fetch(const HeadsArgs& a, int64_t token, int head, const Lane& lk, const Lane& lv) {
    Pair p;
    if constexpr (STEP) {
        const half_t* row = a.x + (token * (a.Hq + 2 * a.Hkv) + a.Hq + head) * a.D;
        p.key = load_head(row, lk);
        p.value = load_head(row + (int64_t)a.Hkv * a.D, lv);
    } else {
        // past the caches, which the cache is left in: 134 MB written and read again 118 us through them, 100 so
        const int64_t at = (token * a.Hkv + head) * a.D;
        p.key = load_once(a.dk + at, lk);
        p.value = load_once(a.dv + at, lv);
    }
    return p;
}
// Norm and rotation of a step's key, and both as 8-bit rows (all lanes of the head come here)
template <bool BF, int LG, bool Q8, bool STEP>
__device__ __forceinline__ Pair8 held(const HeadsArgs& a, Pair& p, const float (&w)[8], const Turn& turn, const Lane& lk) {
    Pair8 h{};
    float f[8];
    if constexpr (STEP || Q8) floats<BF>(p.key, f);
    if constexpr (STEP) {
        norm_rope<BF, LG>(a, f, w, turn.angles, turn.ok, lk);
        p.key = act_cvt8<BF>(f);
    }
    if constexpr (Q8) {
        h.key = to_row8<LG, !STEP>(f, h.key_scale);
        floats<BF>(p.value, f);
        h.value = to_row8<LG, true>(f, h.value_scale);
    }
    return h;
}

// Keys and values of heads h0 .. h1 - 1, kHeadsAtOnce at a time, into the cache, window by window
template <bool BF, int LG, bool Q8, bool STEP>
__device__ __forceinline__ void cache_windows(const HeadsArgs& a, BlockRows<LG, Q8> (&share)[2], int64_t window, int64_t step, int h0, int h1) {
    constexpr int TOKENS = kThreads / LG, HEADS = kHeadsAtOnce<LG>, ROUNDS = kRounds<LG>, SIZE = Q8 ? 1 : 2;
    const int j = threadIdx.x % LG, sub = threadIdx.x / LG, group = value_group(Q8, a.D);
    const Lane lk = lane_of(j, a.D, STEP ? a.R : 0, a.interleaved), lv = lane_of(j, a.D, 0, false);
    float w[8];
    if constexpr (STEP) load_weight(a.kn, lk, w);
    for (int64_t t0 = 16 * window; t0 < a.T; t0 += 16 * step) {
        Pair p[ROUNDS];
        Turn turn[STEP ? ROUNDS : 1];
        const auto load = [&](int64_t from, int h) {  // sixteen tokens
#pragma unroll
            for (int round = 0; round < ROUNDS; ++round) {
                const int n = sub + round * TOKENS;
                p[round] = fetch<STEP>(a, min(from + (n & 15), a.T - 1), min(h + (n >> 4), h1 - 1), lk, lv);
            }
        };
        const auto load_turns = [&](int64_t from) {
            if constexpr (STEP) {
#pragma unroll
                for (int round = 0; round < ROUNDS; ++round) {
                    const int n = sub + round * TOKENS;
                    turn[round].ok = load_angles(a, a.pos[min(from + (n & 15), a.T - 1)], j, lk.turned, turn[round].angles);
                }
            }
        };
        load(t0, h0);  // on their way before it is known which of them go one by one
        load_turns(t0);
        const Window win = window_of(a, t0);
        if (win.first >= 0) {
            const int64_t from = t0 + win.first;
            const int slot = a.slots[from];
            if (win.first > 0) {
                load(from, h0);
                load_turns(from);
            }
            for (int h = h0;;) {
                const int heads = min(HEADS, h1 - h);
#pragma unroll
                for (int round = 0; round < ROUNDS; ++round) {
                    const int n = sub + round * TOKENS, t = n & 15, hs = n >> 4;
                    const Pair8 q = held<BF, LG, Q8, STEP>(a, p[round], w, turn[STEP ? round : 0], lk);
                    char* key = share[0].rows[hs][t];
                    char* value = share[1].rows[hs][t];
                    if (!lk.in) continue;
                    if constexpr (Q8) {
                        *reinterpret_cast<uint32_t*>(key + lk.c0) = q.key[0];
                        *reinterpret_cast<uint32_t*>(key + lk.c1) = q.key[1];
                        *reinterpret_cast<uint2v*>(value + 8 * j) = q.value;
                        if (j == 0 && hs < heads) {
                            const int64_t at = place_of(a, slot + t, h + hs).scale;
                            a.ks[at] = q.key_scale;
                            a.vs[at] = q.value_scale;
                        }
                    } else {
                        store_head(reinterpret_cast<half_t*>(key), lk, p[round].key);
                        *reinterpret_cast<raw8*>(value + 16 * j) = p[round].value;
                    }
                }
                if (h + HEADS < h1) load(from, h + HEADS);
                __syncthreads();
                for (int n = threadIdx.x; n < a.D * SIZE * heads; n += kThreads) {  // 16 D SIZE / 16 units of 16 bytes a head
                    const int hs = n / (a.D * SIZE), u = n - hs * a.D * SIZE;
                    const int64_t at = place_of(a, slot, h + hs).block * SIZE + u * 16;
                    *reinterpret_cast<raw8*>(static_cast<char*>(a.kc) + at) =
                        *reinterpret_cast<const raw8*>(&share[0].rows[hs][u & 15][16 * (u >> 4)]);
                    const auto& rows = share[1].rows[hs];
                    char* to = static_cast<char*>(a.vc) + at;
                    if constexpr (!Q8) {
                        raw8 v;
                        value_unit<2>(u, [&](int k, int t, int c) { v[k] = *reinterpret_cast<const uint16_t*>(&rows[t][2 * c]); });
                        *reinterpret_cast<raw8*>(to) = v;
                    } else {
                        uint32_t v[4] = {};
                        const auto byte = [&](int k, int t, int c) { v[k >> 2] |= (uint32_t)(uint8_t)rows[t][c] << 8 * (k & 3); };
                        if (group == 4) {
                            value_unit<4>(u, byte);
                        } else {
                            value_unit<2>(2 * u, byte);
                            value_unit<2>(2 * u + 1, [&](int k, int t, int c) { byte(k + 8, t, c); });
                        }
                        *reinterpret_cast<uint4v*>(to) = uint4v{v[0], v[1], v[2], v[3]};
                    }
                }
                __syncthreads();
                if ((h += HEADS) >= h1) break;
            }
        }
        if (win.rest == 0) continue;
        if (win.first >= 0) {  // (again, which is rare and spares their registers above)
            load(t0, h0);
            load_turns(t0);
        }
        for (int h = h0;;) {
            const int heads = min(HEADS, h1 - h);
#pragma unroll
            for (int round = 0; round < ROUNDS; ++round) {
                const int n = sub + round * TOKENS, t = n & 15, hs = n >> 4;
                const bool live = hs < heads && (win.rest >> t & 1) && lk.in;
                const Place at = place_of(a, live ? a.slots[t0 + t] : 0, h + min(hs, heads - 1));
                const Pair8 q = held<BF, LG, Q8, STEP>(a, p[round], w, turn[STEP ? round : 0], lk);
                if (!live) continue;
                if constexpr (Q8) {
                    cache_key8(a.kc, at, lk, q.key);
                    cache_value8(a.vc, at, group, lv.c0, q.value);
                    if (j == 0) {
                        a.ks[at.scale] = q.key_scale;
                        a.vs[at.scale] = q.value_scale;
                    }
                } else {
                    cache_key16(a.kc, at, lk, p[round].key);
                    cache_value16(a.vc, at, lv.c0, p[round].value);
                }
            }
            if ((h += HEADS) >= h1) break;
            load(t0, h);
        }
    }
}

// blockIdx.y: heads
template <bool BF, int LG, bool Q8>
__global__ __launch_bounds__(kThreads) void kv_cache_write_kernel(HeadsArgs a) {
    __shared__ __attribute__((aligned(16))) BlockRows<LG, Q8> share[2];
    const int h0 = blockIdx.y * kHeadsAtOnce<LG>;
    cache_windows<BF, LG, Q8, false>(a, share, blockIdx.x, gridDim.x, h0, min(h0 + kHeadsAtOnce<LG>, a.Hkv));
}

// The first workgroups take windows of keys and values, which take longer, the others queries
template <bool BF, int LG, bool Q8, int HPG>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_cache_kernel(HeadsArgs a) {
    __shared__ __attribute__((aligned(16))) BlockRows<LG, Q8> share[2];
    const int cached = a.windows * a.by_groups.d;
    if ((int)blockIdx.x < cached) {
        const int window = fdiv(blockIdx.x, a.by_groups), h0 = (blockIdx.x - window * a.by_groups.d) * a.cached_heads;
        cache_windows<BF, LG, Q8, true>(a, share, window, a.windows, h0, min(h0 + a.cached_heads, a.Hkv));
    } else {
        const int n = blockIdx.x - cached, block = fdiv(n, a.by_chunks);
        heads_apart<BF, LG, HPG, true>(a, block, heads_of<HPG>(a, n - block * a.by_chunks.d));
    }
}

template <bool BF, int LG, bool Q8>
__global__ __launch_bounds__(kThreads) void kv_cache_read_kernel(HeadsArgs a) {
    constexpr int TOKENS = kThreads / LG, HEADS = kHeadsAtOnce<LG>, ROUNDS = kRounds<LG>, SIZE = Q8 ? 1 : 2;
    __shared__ __attribute__((aligned(16))) BlockRows<LG, Q8> share[2];
    const int j = threadIdx.x % LG, sub = threadIdx.x / LG, group = value_group(Q8, a.D);
    const int h0 = blockIdx.y * HEADS, heads = min(HEADS, a.Hkv - h0);
    const Lane l = lane_of(j, a.D, 0, false);
    const auto times = [](uint2v q, float scale) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(q[e >> 2] >> 8 * (e & 3)) * scale;
        return act_cvt8<BF>(f);
    };
    for (int64_t t0 = 16 * (int64_t)blockIdx.x; t0 < a.T; t0 += 16 * (int64_t)gridDim.x) {
        const Window w = window_of(a, t0);
        if (w.first >= 0) {
            const int slot = a.slots[t0 + w.first];
            float scale[2][ROUNDS];
            if constexpr (Q8) {
#pragma unroll
                for (int round = 0; round < ROUNDS; ++round) {
                    const int n = sub + round * TOKENS;
                    const int64_t at = place_of(a, slot + (n & 15), h0 + min(n >> 4, heads - 1)).scale;
                    scale[0][round] = a.ks[at];
                    scale[1][round] = a.vs[at];
                }
            }
            for (int n = threadIdx.x; n < a.D * SIZE * heads; n += kThreads) {
                const int hs = n / (a.D * SIZE), u = n - hs * a.D * SIZE;
                const int64_t at = place_of(a, slot, h0 + hs).block * SIZE + u * 16;
                const raw8 key = *reinterpret_cast<const raw8*>(static_cast<const char*>(a.kc) + at);
                const raw8 value = *reinterpret_cast<const raw8*>(static_cast<const char*>(a.vc) + at);
                *reinterpret_cast<raw8*>(&share[0].rows[hs][u & 15][16 * (u >> 4)]) = key;
                auto& rows = share[1].rows[hs];
                if constexpr (!Q8) {
                    value_unit<2>(u, [&](int k, int t, int c) { *reinterpret_cast<uint16_t*>(&rows[t][2 * c]) = value[k]; });
                } else {
                    const uint4v v = __builtin_bit_cast(uint4v, value);
                    const auto byte = [&](int k, int t, int c) { rows[t][c] = (char)(v[k >> 2] >> 8 * (k & 3)); };
                    if (group == 4) {
                        value_unit<4>(u, byte);
                    } else {
                        value_unit<2>(2 * u, byte);
                        value_unit<2>(2 * u + 1, [&](int k, int t, int c) { byte(k + 8, t, c); });
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int round = 0; round < ROUNDS; ++round) {
                const int n = sub + round * TOKENS, t = n & 15, hs = n >> 4;
                if (hs >= heads || !l.in) continue;
                const int64_t to = ((t0 + w.first + t) * a.Hkv + h0 + hs) * a.D;
#pragma unroll
                for (int values = 0; values < 2; ++values) {
                    const char* row = share[values].rows[hs][t];
                    raw8 v;
                    if constexpr (Q8) v = times(*reinterpret_cast<const uint2v*>(row + 8 * j), scale[values][round]);
                    else v = *reinterpret_cast<const raw8*>(row + 16 * j);
                    store_head((values ? a.v : a.k) + to, l, v);
                }
            }
            __syncthreads();
        }
        // the others, and zeros for tokens that have no slot (those are in no block)
#pragma unroll
        for (int round = 0; round < ROUNDS; ++round) {
            const int n = sub + round * TOKENS, t = n & 15, hs = n >> 4;
            if (hs >= heads || !l.in || t0 + t >= a.T) continue;
            const int slot = a.slots[t0 + t], head = h0 + hs;
            const bool live = (uint32_t)slot < (uint32_t)a.slots_end;
            if (live && !(w.rest >> t & 1)) continue;  // a block's
            raw8 v[2] = {};
            if (live) {
                const Place p = place_of(a, slot, head);
                if constexpr (Q8) {
                    const uint2v key = *reinterpret_cast<const uint2v*>(static_cast<const int8_t*>(a.kc) + p.block + key_place(true, p.t, l.c0));
                    const uint8_t* at = static_cast<const uint8_t*>(a.vc) + p.block + value_place(group, p.t, l.c0);
                    uint2v value{};
#pragma unroll
                    for (int e = 0; e < 8; ++e) value[e >> 2] |= (uint32_t)at[4 * group * e] << 8 * (e & 3);
                    v[0] = times(key, a.ks[p.scale]);
                    v[1] = times(value, a.vs[p.scale]);
                } else {
                    v[0] = *reinterpret_cast<const raw8*>(static_cast<const uint16_t*>(a.kc) + p.block + key_place(false, p.t, l.c0));
                    const uint16_t* at = static_cast<const uint16_t*>(a.vc) + p.block + value_place(2, p.t, l.c0);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[1][e] = at[8 * e];
                }
            }
            const int64_t to = ((t0 + t) * a.Hkv + head) * a.D;
            store_head(a.k + to, l, v[0]);
            store_head(a.v + to, l, v[1]);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------

int lanes_of(int64_t D) {
    int lg = 1;
    while (8 * lg < D) lg *= 2;
    return lg;
}
int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Workgroups for T tokens: a launch takes fewer than 2^32 threads, and the kernels go round
int token_blocks(int64_t T, int lg, int chunks) {
    return (int)std::min<int64_t>((T + kThreads / lg - 1) / (kThreads / lg), std::max(1, (1 << 22) / chunks));
}

#define CLK_LANES(X_) X_(1) X_(2) X_(4) X_(8) X_(16) X_(32)
#define CLK_CACHE_LANES(X_) X_(4) X_(8) X_(16) X_(32)

constexpr int64_t kMostHeads = 8192;

// T, H and D of packed heads, the norms' weights and the angles: the checks of the norm's entry points
int check_heads(const char* what, const clk_buffer* qkv, int64_t hkv, const clk_buffer* qn, const clk_buffer* kn,
                const clk_buffer* rope, const clk_buffer* pos, float eps, HeadsArgs& a) {
    const std::string w(what);
    const int64_t T = qkv->dims[0], H = qkv->dims[1], D = qkv->dims[2];
    if (D < 8 || D > 256 || D % 8) return invalid(w + ": D must be a multiple of 8 up to 256, got " + std::to_string(D));
    if (hkv < 1 || H - 2 * hkv < 1) {
        return invalid(w + ": qkv must be [T,Hq+2*Hkv,D] with at least one query and one key head, got " + std::to_string(H) +
                       " heads and Hkv = " + std::to_string(hkv));
    }
    if (T < 0 || T > INT32_MAX || H > kMostHeads) return invalid(w + ": too large");
    if (elements(qn) != D || elements(kn) != D) return invalid(w + ": q_norm and k_norm must be [D]");
    if (rope->rank != 2 || rope->dims[0] < 1 || rope->dims[0] > INT32_MAX || rope->dims[1] < 8 || rope->dims[1] > D ||
        rope->dims[1] % 8) {
        return invalid(w + ": rope must be [P,R] with a row at least and R a multiple of 8 up to D");
    }
    if (pos->rank != 1 || pos->dims[0] != T) return invalid(w + ": positions must be [T]");
    if (!(eps >= 0.f)) return invalid(w + ": eps must not be negative");
    a.x = static_cast<const half_t*>(qkv->data);
    a.qn = static_cast<const float*>(qn->data);
    a.kn = static_cast<const float*>(kn->data);
    a.rope = static_cast<const float*>(rope->data);
    a.pos = static_cast<const int32_t*>(pos->data);
    a.T = T;
    a.Hq = (int)(H - 2 * hkv);
    a.Hkv = (int)hkv;
    a.D = (int)D;
    a.R = (int)rope->dims[1];
    a.P = (int)rope->dims[0];
    a.inv_d = 1.f / (float)D;
    // The hardware's reciprocal root takes subnormal numbers for zeros. A head of fp16 has them only where all of it is zeros
    // (their squares are past 2^-48), whose results are 0 with any eps but 0, and whose gradients, at least 2^63 2^-24 of a weight,
    // are infinite or 0.
    a.eps = qkv->dtype == CLK_F16 && eps > 0.f ? std::max(eps, 0x1p-126f) : eps;
    return CLK_OK;
}
bool is_heads(const clk_buffer* b, int64_t T, int64_t H, int64_t D) { return b->rank == 3 && dims_are(b, T, H, D); }

int check_aligned(const char* what, std::initializer_list<const clk_buffer*> bufs) {
    for (const clk_buffer* b : bufs) {
        if (elements(b) > 0 && !aligned16(b->data)) return invalid(std::string(what) + ": buffers must be 16-byte aligned");
    }
    return CLK_OK;
}
void set_cache(HeadsArgs& a, const CacheShape& c, const clk_buffer* k, const clk_buffer* v, const clk_buffer* ks,
               const clk_buffer* vs, const clk_buffer* slots) {
    a.kc = k->data;
    a.vc = v->data;
    a.ks = static_cast<float*>(ks->data);
    a.vs = static_cast<float*>(vs->data);
    a.slots = static_cast<const int32_t*>(slots->data);
    a.page = (int)c.page;
    a.slots_end = (int)(c.pages * c.page);
    a.by_page = fast_div(c.page);
}

// Heads a workgroup: more share a token's angles and keep more loads in flight, and take longer pieces of memory in a row, where
// there are workgroups enough without. 16384 tokens of 60 heads of 128: 100 us with eight, 110 with four, 131 with two; of 48
// heads 4099 27.7, 25.7 and 31.8 (42.7 with one), 1500 12.5 with eight, 11.4 with four and 13.4 with one, 128 3.65 with one
// and 4.1 with four. Between, four would be ahead from 256 tokens on (4.5 and 4.6; 1024 8.8 and 10.2).
int heads_at_once(int64_t T, int heads, int lg) {
    const int64_t blocks = (T * lg + kThreads - 1) / kThreads;
    return blocks * ceil_div(heads, 8) >= 2048 ? 8 : blocks * heads >= 4096 ? 4 : 1;
}

#define CLK_L(LG_)                                                                                  \
    if (lg == LG_) {                                                                                \
        if (bf) launch(std::true_type(), std::integral_constant<int, LG_>());                       \
        else launch(std::false_type(), std::integral_constant<int, LG_>());                         \
    }

void launch_forward(HeadsArgs& a, bool bf, hipStream_t s) {
    const int lg = lanes_of(a.D);
    const int hpg = heads_at_once(a.T, a.Hq + 2 * a.Hkv, lg);
    a.cq = ceil_div(a.Hq, hpg);
    a.ck = ceil_div(a.Hkv, hpg);
    const int chunks = a.cq + 2 * a.ck;
    a.by_chunks = fast_div(chunks);
    a.parts = token_blocks(a.T, lg, chunks);
    const dim3 grid(a.parts * chunks), block(kThreads);
    const auto launch = [&](auto bf_, auto lg_) {
        constexpr bool BF = decltype(bf_)::value;
        constexpr int LG = decltype(lg_)::value;
        if (hpg == 8) hipLaunchKernelGGL((qk_norm_rope_kernel<BF, LG, 8>), grid, block, 0, s, a);
        else if (hpg == 4) hipLaunchKernelGGL((qk_norm_rope_kernel<BF, LG, 4>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((qk_norm_rope_kernel<BF, LG, 1>), grid, block, 0, s, a);
    };
    CLK_LANES(CLK_L)
}

// Workgroups for T tokens' windows of 16, and the heads that each takes
int window_blocks(int64_t T, int groups) { return (int)std::min<int64_t>((T + 15) / 16, std::max(1, (1 << 22) / groups)); }
int head_groups(int64_t heads, int lg) { return ceil_div(heads, std::max(1, kThreads / lg / 16)); }

void launch_step(HeadsArgs& a, bool bf, bool q8, hipStream_t s) {
    const int lg = lanes_of(a.D);
    const bool four = heads_at_once(a.T, a.Hq, lg) > 1;
    a.cq = ceil_div(a.Hq, four ? 4 : 1);
    a.by_chunks = fast_div(a.cq);
    a.parts = token_blocks(a.T, lg, a.cq);
    // Heads that a workgroup takes one after another: more share their window's look at the slots and its angles, which are as
    // many bytes as a key and a value, and have the next head's on their way; where that leaves enough workgroups. 4099
    // tokens of 32 + 8 + 8 heads of 128 into 8 bits 27.1 us with four, 28.0 with two, 29.6 with one, into 16 26.6, 28.3 and
    // 29.8; 32768 tokens into 8 176, 185 and 204; 1031 tokens 12.5 with four, 10.4 with two, 11.2 with one; 512 tokens 11.7,
    // 8.5 and 7.2; and eight at 4099 30.1.
    const int once = std::max(1, kThreads / lg / 16);
    const int64_t windows = (a.T + 15) / 16 * head_groups(a.Hkv, lg);
    a.cached_heads = once * (windows >= 1024 ? 4 : windows >= 512 ? 2 : 1);
    const int groups = ceil_div(a.Hkv, a.cached_heads);
    a.by_groups = fast_div(groups);
    a.windows = window_blocks(a.T, groups);
    const dim3 grid(a.parts * a.cq + a.windows * groups), block(kThreads);
    const auto launch = [&](auto bf_, auto lg_) {
        constexpr bool BF = decltype(bf_)::value;
        constexpr int LG = decltype(lg_)::value;
        if (q8) {
            if (four) hipLaunchKernelGGL((qk_norm_rope_cache_kernel<BF, LG, true, 4>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((qk_norm_rope_cache_kernel<BF, LG, true, 1>), grid, block, 0, s, a);
        } else {
            if (four) hipLaunchKernelGGL((qk_norm_rope_cache_kernel<BF, LG, false, 4>), grid, block, 0, s, a);
            else hipLaunchKernelGGL((qk_norm_rope_cache_kernel<BF, LG, false, 1>), grid, block, 0, s, a);
        }
    };
    CLK_CACHE_LANES(CLK_L)
}
#undef CLK_L

// The backward's workgroups a chunk of heads: a rule on the shape alone, so that results do not depend on the device.
// About two rounds of what 256 CUs hold in all.
int bwd_parts(int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
    const int chunks = ceil_div(Hq, kBwdHeads) + 2 * ceil_div(Hkv, kBwdHeads), tokens = kThreads / lanes_of(D);
    return (int)std::min<int64_t>((T + tokens - 1) / tokens, std::max(1, 2048 / chunks));
}

}  // namespace

int check_cache(const char* what, const clk_buffer* k, const clk_buffer* v, const clk_buffer* ks, const clk_buffer* vs, int act,
                CacheShape& c) {
    const std::string w(what);
    const int held = k != nullptr && k->dtype == CLK_S8 ? CLK_S8 : act;
    const clk_buffer* bufs[] = {k, v, ks, vs};
    const int types[] = {held, held, CLK_F32, CLK_F32};
    if (int st = check_types((w + ": cache").c_str(), bufs, types, 4)) return st;
    if (k->rank != 4 || !same_shape(k, v)) return invalid(w + ": k_cache and v_cache must be [pages,heads,page,D], alike");
    c = CacheShape{k->dims[0], k->dims[1], k->dims[2], k->dims[3], held == CLK_S8};
    if (c.D < 32 || c.D > 256 || c.D % 32) return invalid(w + ": a cache's D must be a multiple of 32 up to 256, got " + std::to_string(c.D));
    if (c.page < 16 || c.page % 16) return invalid(w + ": a cache's page must be a multiple of 16, got " + std::to_string(c.page));
    if (c.pages < 1 || c.heads < 1) return invalid(w + ": a cache must have a page and a head at least");
    if (c.heads > 16384 || c.page > (1 << 20) || c.pages > INT32_MAX / c.page) return invalid(w + ": too large");
    if (c.q8) {
        for (const clk_buffer* s : {ks, vs}) {
            if (s->rank != 3 || !dims_are(s, c.pages, c.heads, c.page)) return invalid(w + ": an 8-bit cache's scales must be [pages,heads,page]");
        }
    }
    if (k->data == v->data) return invalid(w + ": k_cache and v_cache must not be the same buffer");
    if (!aligned16(k->data) || !aligned16(v->data) || (c.q8 && (!aligned16(ks->data) || !aligned16(vs->data)))) {
        return invalid(w + ": a cache's buffers must be 16-byte aligned");
    }
    return CLK_OK;
}

}  // namespace clk

using namespace clk;

extern "C" int clk_qk_norm_rope(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm, const clk_buffer* k_norm,
                                const clk_buffer* rope, const clk_buffer* positions, const clk_buffer* q, const clk_buffer* k,
                                const clk_buffer* v, float eps, int32_t interleaved) {
    const int act = qkv != nullptr && qkv->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {qkv, q_norm, k_norm, rope, positions, q, k, v};
    const int types[] = {act, CLK_F32, CLK_F32, CLK_F32, CLK_S32, act, act, act};
    if (int st = check_types("qk_norm_rope", bufs, types, 8)) return st;
    if (qkv->rank != 3 || k->rank != 3) return invalid("qk_norm_rope: qkv must be [T,Hq+2*Hkv,D], k [T,Hkv,D]");
    HeadsArgs a{};
    if (int st = check_heads("qk_norm_rope", qkv, k->dims[1], q_norm, k_norm, rope, positions, eps, a)) return st;
    if (!is_heads(q, a.T, a.Hq, a.D) || !is_heads(k, a.T, a.Hkv, a.D) || !is_heads(v, a.T, a.Hkv, a.D)) {
        return invalid("qk_norm_rope: q must be [T,Hq,D], k and v [T,Hkv,D]");
    }
    if (int st = check_aligned("qk_norm_rope", {qkv, rope, q, k, v})) return st;
    if (a.T == 0) return ok();
    a.q = static_cast<half_t*>(q->data);
    a.k = static_cast<half_t*>(k->data);
    a.v = static_cast<half_t*>(v->data);
    a.interleaved = interleaved != 0;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    launch_forward(a, act == CLK_BF16, s);
    stage_mark(s, 1);
    return launch_status("qk_norm_rope");
}

extern "C" int clk_qk_norm_rope_cache(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm, const clk_buffer* k_norm,
                                      const clk_buffer* rope, const clk_buffer* positions, const clk_buffer* slots,
                                      const clk_buffer* q, const clk_buffer* k_cache, const clk_buffer* v_cache,
                                      const clk_buffer* k_scale, const clk_buffer* v_scale, float eps, int32_t interleaved) {
    const char* what = "qk_norm_rope_cache";
    const int act = qkv != nullptr && qkv->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {qkv, q_norm, k_norm, rope, positions, slots, q};
    const int types[] = {act, CLK_F32, CLK_F32, CLK_F32, CLK_S32, CLK_S32, act};
    if (int st = check_types(what, bufs, types, 7)) return st;
    CacheShape c;
    if (int st = check_cache(what, k_cache, v_cache, k_scale, v_scale, act, c)) return st;
    if (qkv->rank != 3) return invalid("qk_norm_rope_cache: qkv must be [T,Hq+2*Hkv,D]");
    HeadsArgs a{};
    if (int st = check_heads(what, qkv, c.heads, q_norm, k_norm, rope, positions, eps, a)) return st;
    if (c.D != a.D) return invalid("qk_norm_rope_cache: qkv and the cache must have the same D");
    if (!is_heads(q, a.T, a.Hq, a.D)) return invalid("qk_norm_rope_cache: q must be [T,Hq,D]");
    if (slots->rank != 1 || slots->dims[0] != a.T) return invalid("qk_norm_rope_cache: slots must be [T]");
    if (int st = check_aligned(what, {qkv, rope, q})) return st;
    if (a.T == 0) return ok();
    a.q = static_cast<half_t*>(q->data);
    a.interleaved = interleaved != 0;
    set_cache(a, c, k_cache, v_cache, k_scale, v_scale, slots);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    launch_step(a, act == CLK_BF16, c.q8, s);
    stage_mark(s, 1);
    return launch_status(what);
}

extern "C" size_t clk_qk_norm_rope_bwd_workspace_size(const clk_buffer* qkv, const clk_buffer* dk) {
    if (qkv == nullptr || dk == nullptr || qkv->rank != 3 || dk->rank != 3 || qkv->dims == nullptr || dk->dims == nullptr) return 0;
    const int64_t T = qkv->dims[0], H = qkv->dims[1], D = qkv->dims[2], hkv = dk->dims[1], hq = H - 2 * hkv;
    if (T < 1 || T > INT32_MAX || H > kMostHeads || hkv < 1 || hq < 1 || D < 8 || D > 256 || D % 8) return 0;
    const size_t rows = (size_t)bwd_parts(T, hq, hkv, D) * (ceil_div(hq, kBwdHeads) + ceil_div(hkv, kBwdHeads));
    return (rows * D * 4 + 255) / 256 * 256;
}

extern "C" int clk_qk_norm_rope_bwd(clk_stream stream, const clk_buffer* qkv, const clk_buffer* q_norm, const clk_buffer* k_norm,
                                    const clk_buffer* rope, const clk_buffer* positions, const clk_buffer* dq,
                                    const clk_buffer* dk, const clk_buffer* dv, const clk_buffer* dqkv, const clk_buffer* dq_norm,
                                    const clk_buffer* dk_norm, float eps, int32_t interleaved, void* workspace,
                                    size_t workspace_bytes) {
    const char* what = "qk_norm_rope_bwd";
    const int act = qkv != nullptr && qkv->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {qkv, q_norm, k_norm, rope, positions, dq, dk, dv, dqkv, dq_norm, dk_norm};
    const int types[] = {act, CLK_F32, CLK_F32, CLK_F32, CLK_S32, act, act, act, act, CLK_F32, CLK_F32};
    if (int st = check_types(what, bufs, types, 11)) return st;
    if (qkv->rank != 3 || dk->rank != 3) return invalid("qk_norm_rope_bwd: qkv must be [T,Hq+2*Hkv,D], dk [T,Hkv,D]");
    HeadsArgs a{};
    if (int st = check_heads(what, qkv, dk->dims[1], q_norm, k_norm, rope, positions, eps, a)) return st;
    if (!is_heads(dq, a.T, a.Hq, a.D) || !is_heads(dk, a.T, a.Hkv, a.D) || !is_heads(dv, a.T, a.Hkv, a.D)) {
        return invalid("qk_norm_rope_bwd: dq must be [T,Hq,D], dk and dv [T,Hkv,D]");
    }
    if (!same_shape(dqkv, qkv)) return invalid("qk_norm_rope_bwd: dqkv must be like qkv");
    if (elements(dq_norm) != a.D || elements(dk_norm) != a.D) return invalid("qk_norm_rope_bwd: dq_norm and dk_norm must be [D]");
    if (int st = check_aligned(what, {qkv, rope, dq, dk, dv, dqkv})) return st;
    const size_t need = clk_qk_norm_rope_bwd_workspace_size(qkv, dk);
    if (workspace_bytes < need || (need > 0 && workspace == nullptr)) {
        return invalid("qk_norm_rope_bwd: workspace of " + std::to_string(workspace_bytes) + " bytes, needs " + std::to_string(need));
    }
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return invalid("qk_norm_rope_bwd: workspace must be 256-byte aligned");
    a.dq = static_cast<const half_t*>(dq->data);
    a.dk = static_cast<const half_t*>(dk->data);
    a.dv = static_cast<const half_t*>(dv->data);
    a.dx = static_cast<half_t*>(dqkv->data);
    a.dqn = static_cast<float*>(dq_norm->data);
    a.dkn = static_cast<float*>(dk_norm->data);
    a.partial = static_cast<float*>(workspace);
    a.interleaved = interleaved != 0;
    a.cq = ceil_div(a.Hq, kBwdHeads);
    a.ck = ceil_div(a.Hkv, kBwdHeads);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    int stage = 0;
    stage_mark(s, stage);
    if (a.T > 0) {
        a.parts = bwd_parts(a.T, a.Hq, a.Hkv, a.D);
        a.by_chunks = fast_div(a.cq + 2 * a.ck);
        const dim3 grid(a.parts * (a.cq + 2 * a.ck)), block(kThreads);
        const int lg = lanes_of(a.D);
#define CLK_L(LG_)                                                                                                    \
    if (lg == LG_) {                                                                                                  \
        if (act == CLK_BF16) hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<true, LG_>), grid, block, 0, s, a);          \
        else hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<false, LG_>), grid, block, 0, s, a);                         \
    }
        CLK_LANES(CLK_L)
#undef CLK_L
        stage_mark(s, ++stage);
    }
    hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(ceil_div(a.D, 16), 2), dim3(16 * kDwGroups), 0, s, a);
    stage_mark(s, ++stage);
    return launch_status(what);
}

namespace clk {

namespace {

// What kv_cache_write and kv_cache_read share: k, v [T,Hkv,D] beside the cache
int check_moved(const char* what, const clk_buffer* k, const clk_buffer* v, const clk_buffer* slots, const clk_buffer* k_cache,
                const clk_buffer* v_cache, const clk_buffer* k_scale, const clk_buffer* v_scale, HeadsArgs& a, bool& q8, bool& bf) {
    const int act = k != nullptr && k->dtype == CLK_BF16 ? CLK_BF16 : CLK_F16;
    const clk_buffer* bufs[] = {k, v, slots};
    const int types[] = {act, act, CLK_S32};
    if (int st = check_types(what, bufs, types, 3)) return st;
    CacheShape c;
    if (int st = check_cache(what, k_cache, v_cache, k_scale, v_scale, act, c)) return st;
    const int64_t T = k->rank == 3 ? k->dims[0] : -1;
    if (T < 0 || !is_heads(k, T, c.heads, c.D) || !is_heads(v, T, c.heads, c.D)) {
        return invalid(std::string(what) + ": k and v must be [T,heads,D], heads and D the cache's");
    }
    if (T > INT32_MAX) return invalid(std::string(what) + ": too large");
    if (slots->rank != 1 || slots->dims[0] != T) return invalid(std::string(what) + ": slots must be [T]");
    if (int st = check_aligned(what, {k, v})) return st;
    a.T = T;
    a.Hkv = (int)c.heads;
    a.D = (int)c.D;
    set_cache(a, c, k_cache, v_cache, k_scale, v_scale, slots);
    q8 = c.q8;
    bf = act == CLK_BF16;
    return CLK_OK;
}

}  // namespace

}  // namespace clk

#define CLK_MOVE(KERNEL_)                                                                                              \
    const int lg = lanes_of(a.D);                                                                                      \
    const int groups = head_groups(a.Hkv, lg);                                                                         \
    const dim3 grid(window_blocks(a.T, groups), groups), block(kThreads);                                              \
    const auto launch = [&](auto bf_, auto lg_) {                                                                      \
        constexpr bool BF = decltype(bf_)::value;                                                                      \
        constexpr int LG = decltype(lg_)::value;                                                                       \
        if (q8) hipLaunchKernelGGL((KERNEL_<BF, LG, true>), grid, block, 0, s, a);                                     \
        else hipLaunchKernelGGL((KERNEL_<BF, LG, false>), grid, block, 0, s, a);                                       \
    };                                                                                                                 \
    CLK_CACHE_LANES(CLK_L)
#define CLK_L(LG_)                                                                                                     \
    if (lg == LG_) {                                                                                                   \
        if (bf) launch(std::true_type(), std::integral_constant<int, LG_>());                                          \
        else launch(std::false_type(), std::integral_constant<int, LG_>());                                            \
    }

extern "C" int clk_kv_cache_write(clk_stream stream, const clk_buffer* k, const clk_buffer* v, const clk_buffer* slots,
                                  const clk_buffer* k_cache, const clk_buffer* v_cache, const clk_buffer* k_scale,
                                  const clk_buffer* v_scale) {
    HeadsArgs a{};
    bool q8, bf;
    if (int st = check_moved("kv_cache_write", k, v, slots, k_cache, v_cache, k_scale, v_scale, a, q8, bf)) return st;
    if (a.T == 0) return ok();
    a.dk = static_cast<const half_t*>(k->data);
    a.dv = static_cast<const half_t*>(v->data);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    CLK_MOVE(kv_cache_write_kernel)
    stage_mark(s, 1);
    return launch_status("kv_cache_write");
}

extern "C" int clk_kv_cache_read(clk_stream stream, const clk_buffer* k_cache, const clk_buffer* v_cache, const clk_buffer* k_scale,
                                 const clk_buffer* v_scale, const clk_buffer* slots, const clk_buffer* k, const clk_buffer* v) {
    HeadsArgs a{};
    bool q8, bf;
    if (int st = check_moved("kv_cache_read", k, v, slots, k_cache, v_cache, k_scale, v_scale, a, q8, bf)) return st;
    if (a.T == 0) return ok();
    a.k = static_cast<half_t*>(k->data);
    a.v = static_cast<half_t*>(v->data);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    CLK_MOVE(kv_cache_read_kernel)
    stage_mark(s, 1);
    return launch_status("kv_cache_read");
}
