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
#include <type_traits>

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

// The chunk that stands first in row r of an LDS tile of 64-byte rows. A 16-byte LDS read takes its lanes in the sets
// 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 (and the same 32 lanes on), so that in one pass rows 0-3 and 12-15
// of one chunk meet rows 4-11 of its neighbour: these have to lie in different banks. With r / 4 for -r / 4 they
// meet pairwise, and a read takes 8 cycles, not 4 (8192 x 8192 x 8192: 1.7e7 cycles of bank conflicts, so none; LDS
// does not bound it, so that saves power and 2 of 427 us).
__device__ __forceinline__ int swizzle(int r) { return -(r >> 2) & 3; }

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
    bool lines;  // each 64 channels of a row are a whole line of out
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

// RL consecutive channels n .. of row m, of which those below N exist: their scales and biases, and the results
template <int RL>
struct Channels {
    float sw[RL], b[RL];
    __device__ __forceinline__ Channels(const GemmArgs& a, int n) {
#pragma unroll
        for (int i = 0; i < RL; ++i) {
            sw[i] = n + i < a.N ? a.ws[n + i] : 0.f;
            b[i] = a.b != nullptr && n + i < a.N ? a.b[n + i] : 0.f;
        }
    }
};
// a and b: two pieces of row lane % 16. Then a is a piece of row lane % 8, b one of row lane % 8 + 8: the first of the
// pieces in lanes with lane % 16 < 8, the second in the others, so that a store of each fills eight rows' lines. (Writing
// 151 MB by nontemporal stores of half lines takes 41 us, of whole lines 26.)
__device__ __forceinline__ void rows_of_eight(half8& a, half8& b) {
    constexpr int kTurn8 = 0x128;  // each 16 lanes rotated by 8
    const uint4v x = __builtin_bit_cast(uint4v, a), y = __builtin_bit_cast(uint4v, b);
    uint4v u, v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)x[i], (int)y[i], kTurn8, 0xf, 0xc, false);
        v[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)y[i], (int)x[i], kTurn8, 0xf, 0x3, false);
    }
    a = __builtin_bit_cast(half8, u);
    b = __builtin_bit_cast(half8, v);
}

template <int W>
struct Vec16;
template <>
struct Vec16<4> {
    typedef half4 type;
    typedef half4u unaligned;
};
template <>
struct Vec16<8> {
    typedef half8 type;
    typedef half8u unaligned;
};
__device__ __forceinline__ int64_t at_of(const GemmArgs& a, int m, int n) { return (int64_t)m * a.N + n; }
template <bool BF, int RL>
__device__ __forceinline__ void store_run(const GemmArgs& a, int m, int n, const Channels<RL>& ch, const int (&sum)[RL]) {
    constexpr int W = RL < 8 ? RL : 8;  // channels an access
    if (m >= a.M || n >= a.N) return;
    const float sx = a.qs[m];
    const int64_t at = at_of(a, m, n);
    float v[RL];
#pragma unroll
    for (int i = 0; i < RL; ++i) v[i] = scaled(sum[i], sx, ch.sw[i], ch.b[i]);
    if (n + RL <= a.N) {
        if (a.residual != nullptr) {
            typename Vec16<W>::type r[RL / W];
#pragma unroll
            for (int h = 0; h < RL / W; ++h) r[h] = *reinterpret_cast<const typename Vec16<W>::unaligned*>(a.residual + at + W * h);
#pragma unroll
            for (int i = 0; i < RL; ++i) v[i] += act_get<BF>(half8{r[i / W][i % W]}, 0);
        }
#pragma unroll
        for (int h = 0; h < RL / W; ++h) {
            typename Vec16<W>::type o;
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] = act_cvt<BF>(v[W * h + i]);
            *reinterpret_cast<typename Vec16<W>::unaligned*>(a.out + at + W * h) = o;
        }
    } else {
#pragma unroll
        for (int i = 0; i < RL; ++i) {
            if (n + i < a.N) {
                if (a.residual != nullptr) v[i] += act_get<BF>(half8{a.residual[at + i]}, 0);
                a.out[at + i] = act_cvt<BF>(v[i]);
            }
        }
    }
}
// The same for a wave's rows m0 .. m0 + 15 and 64 channels that all exist (16 a lane), with their residual (ADD), by
// stores of whole lines, nontemporal where they are such in memory too (LINES): 20000 x 1024 x 1024 with a residual
// takes 37 us, 38 by nontemporal half lines and 51 by whole lines through the caches; 4096 x 1024 x 4094 26 us
// through the caches and 35 by nontemporal stores.
template <bool BF, bool ADD, bool LINES>
__device__ __forceinline__ void store_lines(const GemmArgs& a, int m0, int n, int r16, const Channels<16>& ch, const int (&sum)[16],
                                            const half8 (&res)[2]) {
    const float sx = a.qs[min(m0 + r16, a.M - 1)];
    half8 o[2];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = scaled(sum[i], sx, ch.sw[i], ch.b[i]);
        if constexpr (ADD) v += act_get<BF>(res[i / 8], i % 8);
        o[i / 8][i % 8] = act_cvt<BF>(v);
    }
    rows_of_eight(o[0], o[1]);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int m = m0 + 8 * p + (r16 & 7);
        if (m >= a.M) continue;
        half8u* to = reinterpret_cast<half8u*>(a.out + at_of(a, m, n + 8 * (r16 >> 3)));
        if constexpr (LINES) __builtin_nontemporal_store(o[p], to);
        else *to = o[p];
    }
}

// Up to four rows: a product is the reading of its weights. A workgroup computes one operand of 16 channels; its
// four waves split k in runs of steps and join their sums through LDS. Operands go from memory straight to
// registers, four steps ahead, so a wave has 4 to 8 KB in flight; the rows' 16-byte pieces come in operand
// order, which is slow for 16 rows (see below) but costs little where most lanes have none. [1, 4096] x
// [4096, 4096]: 3.9 us (16.8 MB: 4.3 TB/s from the far cache), 0.3 us less than the kernel below; with five
// and more rows that one is as fast or faster (7 rows, 8192 to 2048: 5.2 against 6.1 us).
constexpr int kFewRows = 4;

template <bool BF>
__global__ __launch_bounds__(256) void q8_rows_kernel(GemmArgs a) {
    constexpr int KW = 4, U = 4;
    __shared__ __attribute__((aligned(16))) int4v part[KW][kWave];
    const int o = xcd_item(blockIdx.x, gridDim.x);  // operand o % 4 of block o / 4
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4, kbs = a.Kp / 64;
    const auto rw = rsrc_of(a.wq + (int64_t)(o / 4) * 64 * a.Kp, (uint32_t)(64 * a.Kp));
    const auto rx = rsrc_of(a.q, (uint32_t)(a.M * a.Kp));
    const int run = (kbs + KW - 1) / KW, begin = min(kbs, run * wave), end = min(kbs, begin + run);
    int4v acc{0, 0, 0, 0}, x[U], w[U];
    // (a step past the run's end reads past the buffers' range: zeros, no traffic)
    const auto load = [&](int kb, int4v& xs, int4v& ws) __attribute__((always_inline)) {
        const uint32_t past = kb < end ? 0u : 0x80000000u;
        ws = load16(rw, past + (uint32_t)(4096 * kb + 1024 * (o % 4) + 16 * lane));
        xs = load16(rx, past + (uint32_t)(r16 * a.Kp + 64 * kb + 16 * g));
    };
#pragma unroll
    for (int i = 0; i < U; ++i) load(begin + i, x[i], w[i]);
    for (int kb = begin; kb < end; kb += U) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            acc = mfma_i8(w[i], x[i], acc);
            load(kb + U + i, x[i], w[i]);
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int v = 1; v < KW; ++v) acc += part[v][lane];
    const int n = 64 * (o / 4) + 16 * g + 4 * (o % 4);
    store_run<BF, 4>(a, r16, n, Channels<4>(a, n), {acc[0], acc[1], acc[2], acc[3]});
}

// A workgroup computes 16 MF WM rows by 16 NU WN channels. Its waves are KS groups of WM x WN; wave (wm, wn) of a
// group has MF operands of 16 rows and NU of 16 channels, and the groups take every KS-th step of 64 inputs
// (one MFMA step) and join their sums through LDS. Both operands go through LDS, a step at a time, in a
// ring of RING buffers a group: a buffer is filled again as soon as every wave of the group holds its
// operands in registers, so the loads of RING - 1 steps are in flight while one is computed.
//   weights  by 1024-byte direct-to-LDS loads, in memory order: an operand read is 64 lanes' consecutive 16
//            bytes
//   rows     16 rows of 64 bytes a load, position p of row r holding its 16-byte chunk p ^ swizzle(r). (Loaded
//            straight in operand order, 16 bytes of 16 rows after each other, the same kilobyte takes three times
//            as long: 16 bytes a clock and CU against 44.)
// Large products are bound by power: 8192 x 8192 x 8192 with a residual takes 426 to 462 us (2.38 to 2.58 POP/s), machine
// by machine, with the matrix cores busy for 75% of the cycles at 1.64 to 1.77 GHz (2.4 in kernels that memory
// bounds). Few rows are bound by the weights' reading (48 x 4096 x 8192: 8.7 us, 34 MB at 3.9 TB/s), medium ones
// by the fill and tail of one round of workgroups (1531 x 1100 x 2050 with a residual: 10.6 us, 0.65 POP/s).
template <bool BF, int MF, int NU, int WM, int WN, int KS, int RING>
__global__ __launch_bounds__(64 * WM * WN * KS) void q8_tile_kernel(GemmArgs a) {
    constexpr int G = WM * WN, XT = MF * WM, WT = NU * WN, STEP = 1024 * (XT + WT), BM = 16 * XT;
    constexpr int XL = XT / G, WL = WT / G, L = XL + WL;  // loads a wave a step
    static_assert(XL * G == XT && WL * G == WT && RING >= 3 && (RING - 1) * L < 64 && KS * RING * STEP <= 160 * 1024);
    __shared__ __attribute__((aligned(1024))) char lds[KS * RING * STEP];
    const int item = xcd_item(blockIdx.x, gridDim.x);
    // groups of four row tiles, in a group row tiles fastest: what an XCD runs at a time is a patch of the
    // result, whose operands its L2 holds
    const int per = 4 * a.ntiles, grp4 = item / per, in = item - grp4 * per;
    const int gm = min(4, a.mtiles - 4 * grp4), nt = in / gm, mt = 4 * grp4 + in - nt * gm;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4, grp = wave / G, wg = wave % G, wm = wg % WM, wn = wg / WM;
    const int m0 = BM * mt, rows = min(BM, a.M - m0), Kp = a.Kp, kbs = Kp / 64;
    const int o0 = WT * nt, nb0 = o0 / 4;  // the tile's first operand of channels, and its block
    const int nblks = min((o0 % 4 + WT + 3) / 4, (a.N + 63) / 64 - nb0);
    const auto rx = rsrc_of(a.q + (int64_t)m0 * Kp, (uint32_t)(rows * Kp));
    const auto rw = rsrc_of(a.wq + (int64_t)nb0 * 64 * Kp, (uint32_t)(nblks * 64 * Kp));
    char* ring = lds + grp * RING * STEP;

    uint32_t xoff[XL], woff[WL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const int r = 16 * (XL * wg + i) + (lane >> 2);
        xoff[i] = (uint32_t)(r * Kp + 16 * ((lane & 3) ^ swizzle(r)));
    }
#pragma unroll
    for (int i = 0; i < WL; ++i) {
        const int o = o0 % 4 + WL * wg + i;
        woff[i] = (uint32_t)((o >> 2) * 64 * Kp + (o & 3) * 1024 + 16 * lane);
    }
    // load i of the group's step t (past the last one it reads past the buffers' range: zeros, no traffic)
    const auto fetch = [&](int i, int t, char* base) __attribute__((always_inline)) {
        const int s = KS * t + grp;
        if (i < XL) dma_lds<16>(rx, base + 1024 * (XL * wg + i), xoff[i] + (s < kbs ? 64u * s : 0x80000000u));
        else dma_lds<16>(rw, base + 1024 * (XT + WL * wg + i - XL), woff[i - XL] + (s < kbs ? 4096u * s : 0x80000000u));
    };
    int4v acc[NU][MF];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int mf = 0; mf < MF; ++mf) acc[u][mf] = int4v{0, 0, 0, 0};

    struct Operands {
        int4v x[MF], w[NU];
    };
    constexpr int R = MF + NU;  // operand reads of a step
    const int xat = (16 * MF * wm + r16) * 64 + 16 * (g ^ swizzle(r16)), wat = 1024 * (XT + NU * wn) + 16 * lane;
    const auto read = [&](int i, const char* base, Operands& o) __attribute__((always_inline)) {
        if (i < MF) o.x[i] = *reinterpret_cast<const int4v*>(base + xat + 1024 * i);
        else o.w[i - MF] = *reinterpret_cast<const int4v*>(base + wat + 1024 * (i - MF));
    };
    // Step t, with its operands in `cur` or on their way there: past the wait (and, in a group of several
    // waves, the barrier) they are in the registers, so their buffer takes the loads of step t + RING, and
    // step t + 1 has landed (newer than it are the loads of RING - 2 steps). Its operands are read while step
    // t is multiplied. Reads and loads are issued one by one between the products, which wait for neither:
    // in a burst they hold up the wave at a full queue. Steps go in pairs; one past the last adds zeros.
    int buf = 0;  // byte offset of step t's buffer
    const auto turn = [&](int t, const Operands& cur, Operands& next) __attribute__((always_inline)) {
        if constexpr (G > 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * L) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * L) : "memory");
        char* free = ring + buf;
        buf = buf == (RING - 1) * STEP ? 0 : buf + STEP;
        const char* ready = ring + buf;
        constexpr int P = NU * MF;  // products of a step
        if constexpr (P < R) {
#pragma unroll
            for (int i = 0; i < R; ++i) read(i, ready, next);
#pragma unroll
            for (int i = 0; i < L; ++i) fetch(i, t + RING, free);
        }
#pragma unroll
        for (int n = 0; n < P; ++n) {
            const int u = n / MF, mf = n % MF;
            acc[u][mf] = mfma_i8(cur.w[u], cur.x[mf], acc[u][mf]);
            if constexpr (P >= R) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (n == i * (P * 3 / 4 / R > 0 ? P * 3 / 4 / R : 1)) read(i, ready, next);
#pragma unroll
                for (int i = 0; i < L; ++i)
                    if (n == (2 * i + 1) * P / (2 * L)) fetch(i, t + RING, free);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    Operands even, odd;
#pragma unroll
    for (int t = 0; t < RING; ++t)
#pragma unroll
        for (int i = 0; i < L; ++i) fetch(i, t, ring + t * STEP);
    if constexpr (G > 1) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((RING - 1) * L) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 1) * L) : "memory");
#pragma unroll
    for (int i = 0; i < R; ++i) read(i, ring, even);
    const int steps = (kbs + KS - 1) / KS;
    for (int t = 0; t < steps; t += 2) {
        turn(t, even, odd);
        turn(t + 1, odd, even);
    }
    // no load may write LDS past the workgroup's end, nor over the sums below
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

    if constexpr (KS == 1) {
        constexpr int NE = NU < 4 ? NU : 4;  // operands of a run: 4 NE channels
#pragma unroll
        for (int u = 0; u < NU; u += NE) {
            const int o = o0 + NU * wn + u, n = 64 * (o / 4) + 16 * g + 4 * (o % 4);
            const Channels<4 * NE> ch(a, n);
            const auto sums = [&](int mf, int (&sum)[4 * NE]) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < 4 * NE; ++i) sum[i] = acc[u + i / 4][mf][i % 4];
            };
            const int row0 = m0 + 16 * MF * wm;
            if constexpr (NE == 4) {
                if (16 * o + 64 <= a.N) {  // the same for all lanes
                    // residuals three groups of rows ahead: 8192 x 8192 x 8192 takes 426 us with and 445 without that,
                    // 8192 x 1024 x 8192 107 and 127 (two ahead 427 and 111; by whole lines, turned back in
                    // registers, the same)
                    constexpr int AHEAD = MF < 3 ? MF : 3;
                    const auto rows = [&](auto add_, auto lines_) __attribute__((always_inline)) {
                        constexpr bool ADD = decltype(add_)::value, LINES = decltype(lines_)::value;
                        half8 res[AHEAD + 1][2];
                        const auto read = [&](int mf) __attribute__((always_inline)) {
                            if constexpr (ADD)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    res[mf % (AHEAD + 1)][h] = *reinterpret_cast<const half8u*>(a.residual + at_of(a, min(row0 + 16 * mf + r16, a.M - 1), n) + 8 * h);
                        };
#pragma unroll
                        for (int mf = 0; mf < AHEAD; ++mf) read(mf);
#pragma unroll
                        for (int mf = 0; mf < MF; ++mf) {
                            if (mf + AHEAD < MF) read(mf + AHEAD);
                            __builtin_amdgcn_sched_barrier(0);
                            int sum[16];
                            sums(mf, sum);
                            store_lines<BF, ADD, LINES>(a, row0 + 16 * mf, n, r16, ch, sum, res[mf % (AHEAD + 1)]);
                        }
                    };
                    if (a.residual != nullptr) a.lines ? rows(std::true_type(), std::true_type()) : rows(std::true_type(), std::false_type());
                    else a.lines ? rows(std::false_type(), std::true_type()) : rows(std::false_type(), std::false_type());
                    continue;
                }
            }
#pragma unroll
            for (int mf = 0; mf < MF; ++mf) {
                int sum[4 * NE];
                sums(mf, sum);
                store_run<BF>(a, row0 + 16 * mf + r16, n, ch, sum);
            }
        }
    } else {
        // wave wg of group j finishes runs j, j + KS, ... of its place in the tile
        constexpr int NE = MF * NU >= 4 * KS && NU % 4 == 0 ? 4 : 1, RUNS = MF * NU / NE;
        static_assert(KS * G * MF * NU <= KS * RING * (XT + WT));
        int4v* part = reinterpret_cast<int4v*>(lds);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int mf = 0; mf < MF; ++mf) part[((grp * G + wg) * NU * MF + u * MF + mf) * kWave + lane] = acc[u][mf];
        __syncthreads();
        for (int f = grp; f < RUNS; f += KS) {
            const int u = f / MF * NE, mf = f % MF;
            int sum[4 * NE];
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                int4v s = part[(wg * NU * MF + (u + e) * MF + mf) * kWave + lane];
#pragma unroll
                for (int j = 1; j < KS; ++j) s += part[((j * G + wg) * NU * MF + (u + e) * MF + mf) * kWave + lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[4 * e + i] = s[i];
            }
            const int o = o0 + NU * wn + u, n = 64 * (o / 4) + 16 * g + 4 * (o % 4);
            store_run<BF>(a, m0 + 16 * (MF * wm + mf) + r16, n, Channels<4 * NE>(a, n), sum);
        }
    }
}

// A buffer descriptor as its four words, and a direct-to-LDS load of 16 bytes a lane that the compiler does not
// know as one: with the builtin it waits for every such load in flight before the next LDS read of the
// kernel below. The load has no result, and whoever reads its bytes waits for it by vmcnt. (A write of m0
// needs one wait state before such a load.)
template <typename P>
__device__ __forceinline__ uint4v words_of(const P* p, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return uint4v{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, bytes, 0x00020000u};
}
__device__ __forceinline__ void dma_lds_untracked(uint4v rsrc, void* dst, uint32_t off) {
#ifdef __HIP_DEVICE_COMPILE__
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
#else
    (void)rsrc, (void)dst, (void)off;
#endif
}

// Many rows, short k: the product is the reading of rows and the writing of results, so a wave keeps its weights
// (NU operands of channels, KB steps) in registers and streams rows past them. A workgroup's four waves
// are WM x WN over rows and channels, 16 or 32 rows a wave and tile; tiles come through LDS, two
// ahead; scales and biases wait in LDS, the next tile's row scales and residual in registers. Results go
// out as 16-byte buffer stores, whose range drops what lies past M and N, so that every tile issues the
// same number of memory accesses and a tile's wait can count them. A weight operand's rows are picked so that
// four lanes hold 64 consecutive bytes of a row, which is how the residual is read; stores turn them into whole
// lines. Where rows are whole lines and there is no residual they are nontemporal: 147456 x 128 x 512 takes 28.4 us
// (170 MB, 6.0 TB/s), 40 by nontemporal half lines, 45 by whole lines through the caches; 147456 x 128 x 520,
// whose stores end inside lines, 53 through the caches and 89 nontemporal. With a residual, read through the same
// caches, they go through them too: 59 us (321 MB, 5.4 TB/s; 57 by nontemporal ones), but 65536 rows and a norm
// of the results take 46 us, 55 by nontemporal ones. A row's last piece, cut at an even channel, goes out by its
// words: 147456 x 128 x 510 52 us.
template <bool BF, int KB, int NU, int MF, int WN, bool RES, bool NT>
__global__ __launch_bounds__(256) void q8_stream_kernel(GemmArgs a) {
    constexpr int BR = 16 * MF, WM = 4 / WN, XT = MF * WM * KB, XL = (XT + 3) / 4, RING = 3, SLOT = 4096 * XL;
    constexpr int CW = 16 * NU, H = NU / 2;  // channels a wave; 16-byte pieces of a lane's results a row
    constexpr uint32_t kDrop = 0x80000000u;
    __shared__ __attribute__((aligned(1024))) char lds[RING * SLOT + 8 * CW * WN];  // the ring; scales, biases
    float* params = reinterpret_cast<float*>(lds + RING * SLOT);
    const int item = xcd_item(blockIdx.x, gridDim.x), nt = item % a.ntiles, first = item / a.ntiles;
    const int stride = gridDim.x / a.ntiles, Kp = a.Kp, kbs = Kp / 64;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4, wm = wave / WN, wn = wave % WN;
    const int c0 = CW * WN * nt, n0 = c0 + CW * wn;  // the workgroup's and the wave's first channel
    const bool tail = a.N % 8 != 0 && n0 < a.N && n0 + CW > a.N;  // one of its pieces is cut
    for (int i = threadIdx.x; i < CW * WN; i += 256) {
        params[i] = c0 + i < a.N ? a.ws[c0 + i] : 0.f;
        params[CW * WN + i] = a.b != nullptr && c0 + i < a.N ? a.b[c0 + i] : 0.f;
    }
    const int blocks = (a.N + 63) / 64;
    int4v w[KB][NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int blk = n0 / 64 + u / 4;
        const auto rw = rsrc_of(a.wq + (int64_t)min(blk, blocks - 1) * 64 * Kp, (uint32_t)(64 * Kp));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            // row r16 of operand u % 4 is channel c of the block, which the layout has as row 4 (c / 16) + c % 4 of
            // operand c / 4 % 4
            const int c = 32 * (u % 4 / 2) + 8 * (r16 / 4) + 4 * (u % 2) + r16 % 4;
            w[kb][u] = load16(rw, kb < kbs && blk < blocks ? (uint32_t)(4096 * kb + 1024 * (c / 4 % 4) + 256 * g + 16 * (4 * (c / 16) + c % 4)) : kDrop);
        }
    }
    // 0 .. most, kept on the scalar unit (a median would go to the vector unit, and with it a buffer's range)
    const auto clamp = [](int v, int most) __attribute__((always_inline)) {
        return __builtin_amdgcn_readfirstlane(max(0, min(most, v)));
    };
    // load j of a tile: operand j / KB of rows, step j % KB
    const auto fetch = [&](int mt, char* slot) __attribute__((always_inline)) {
        const int m0 = BR * WM * mt, rows = clamp(a.M - m0, BR * WM);
        const auto rx = words_of(a.q + (int64_t)(rows > 0 ? m0 : 0) * Kp, (uint32_t)(rows * Kp));
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int j = 4 * i + wave, kb = j % KB, r = 16 * (j / KB) + (lane >> 2);
            dma_lds_untracked(rx, slot + 1024 * j, j < XT && kb < kbs ? (uint32_t)(r * Kp + 64 * kb + 16 * ((lane & 3) ^ swizzle(r))) : kDrop);
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");  // what is counted as newer stays newer
    };
    struct Rows {
        float qs[MF];
        half8 res[MF][RES ? H : 1];
    };
    const auto rows_of = [&](int mt, Rows& o) __attribute__((always_inline)) {
        const int m0 = BR * (WM * mt + wm), rows = clamp(a.M - m0, BR), base = rows > 0 ? m0 : 0;
        const auto rs = rsrc_of(a.qs + base, (uint32_t)(rows * 4));
        const auto rr = rsrc_of(RES ? a.residual + (int64_t)base * a.N : a.out, RES ? (uint32_t)rows * (uint32_t)a.N * 2u : 0u);
#pragma unroll
        for (int mf = 0; mf < MF; ++mf) {
            const int r = 16 * mf + r16;
            o.qs[mf] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, (uint32_t)(4 * r), 0, 0));
            if constexpr (RES) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const int n = n0 + 64 * (h / 2) + 32 * (h % 2) + 8 * g;
                    o.res[mf][h] = __builtin_bit_cast(half8, load16(rr, n < a.N ? ((uint32_t)r * (uint32_t)a.N + (uint32_t)n) * 2u : kDrop));
                }
            }
        }
    };
    const auto tile = [&](int mt, const char* slot, const Rows& now) __attribute__((always_inline)) {
        const int m0 = BR * (WM * mt + wm), rows = clamp(a.M - m0, BR);
        const auto ro = rsrc_of(a.out + (int64_t)(rows > 0 ? m0 : 0) * a.N, (uint32_t)rows * (uint32_t)a.N * 2u);
        int4v acc[NU][MF];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            int4v x[MF];
#pragma unroll
            for (int mf = 0; mf < MF; ++mf) {
                x[mf] = *reinterpret_cast<const int4v*>(slot + 1024 * ((MF * wm + mf) * KB + kb) + r16 * 64 + 16 * (g ^ swizzle(r16)));
            }
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int mf = 0; mf < MF; ++mf) acc[u][mf] = mfma_i8(w[kb][u], x[mf], kb == 0 ? int4v{0, 0, 0, 0} : acc[u][mf]);
        }
#pragma unroll
        for (int h = 0; h < H; h += 2) {
            float8v sw[2], bv[2];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int c = CW * wn + 32 * (h + p) + 8 * g;
                sw[p] = *reinterpret_cast<const float8v*>(params + c);
                bv[p] = *reinterpret_cast<const float8v*>(params + CW * WN + c);
            }
            const int n = n0 + 32 * (h + (r16 >> 3)) + 8 * g;
#pragma unroll
            for (int mf = 0; mf < MF; ++mf) {
                half8 o[2];
#pragma unroll
                for (int p = 0; p < 2; ++p)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float v = scaled(acc[2 * (h + p) + i / 4][mf][i % 4], now.qs[mf], sw[p][i], bv[p][i]);
                        if constexpr (RES) v += act_get<BF>(now.res[mf][h + p], i);
                        o[p][i] = act_cvt<BF>(v);
                    }
                rows_of_eight(o[0], o[1]);
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const uint32_t to = ((uint32_t)(16 * mf + 8 * p + (r16 & 7)) * (uint32_t)a.N + (uint32_t)n) * 2u;
                    const uint4v words = __builtin_bit_cast(uint4v, o[p]);
                    __builtin_amdgcn_raw_buffer_store_b128(words, ro, n + 8 <= a.N ? to : kDrop, 0, NT ? 2 : 0);
                    if (tail) {
#pragma unroll
                        for (int i = 0; i < 3; ++i) {
                            __builtin_amdgcn_raw_buffer_store_b32(words[i], ro, n + 8 > a.N && n + 2 * i < a.N ? to + 4 * i : kDrop, 0, 0);
                        }
                    }
                }
            }
        }
    };
    const int tiles = (a.M + BR * WM - 1) / (BR * WM);
    // newer than a tile's loads at its wait: one tile's loads, and two tiles' row scales, residual and stores
    constexpr int kNewer = XL + 2 * (MF + (RES ? MF * H : 0) + MF * H);
    static_assert(kNewer < 64);
    Rows ra, rb;
    int at = 0;
    fetch(first, lds);
    fetch(first + stride, lds + SLOT);
    rows_of(first, ra);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const auto turn = [&](int mt, const Rows& now, Rows& next) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kNewer) : "memory");
        const int free = at == 0 ? (RING - 1) * SLOT : at - SLOT;
        fetch(mt + 2 * stride, lds + free);
        rows_of(mt + stride, next);
        tile(mt, lds + at, now);
        at = at == (RING - 1) * SLOT ? 0 : at + SLOT;
    };
    for (int mt = first; mt < tiles; mt += 2 * stride) {
        turn(mt, ra, rb);
        turn(mt + stride, rb, ra);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may write LDS past the workgroup's end
}

// |sum| <= 128^2 Kp has to stay below 2^31
constexpr int64_t kMaxKp = 131008;

// The tiles for more than 64 rows, by estimated time: a round of 256 tiles, one for each CU, costs a fixed part
// (loads that wait for the first operands, the results) and one for k. Both measured, in us and in us for
// 1024 inputs, from 8192 x k x 8192 at k = 1024 and 8192: 86 and 420 us with the first of the sizes below, 79 and
// 455, 103 and 557, 181 and 842 with the others. Large tiles read less for each product, small ones fill
// the card where there are few.
struct Tile {
    int rows, channels;
    double fixed, per1024;
};
constexpr Tile kTiles[] = {{256, 256, 9.4, 11.9}, {128, 256, 3.2, 6.7}, {128, 128, 2.4, 4.05}, {64, 64, 1.35, 1.48}};

int best_tile(int64_t M, int64_t N, int64_t Kp) {
    int best = 0;
    double least = 0;
    for (int i = 0; i < 4; ++i) {
        const Tile& t = kTiles[i];
        const int64_t tiles = (M + t.rows - 1) / t.rows * ((N + t.channels - 1) / t.channels);
        const double us = (double)((tiles + 255) / 256) * (t.fixed + t.per1024 * (double)Kp / 1024);
        if (i == 0 || us < least) {
            best = i;
            least = us;
        }
    }
    return best;
}

// Whether the kernel for many rows and short k takes a call. From 2048 rows on it was the faster one for all of
// 27 shapes with k of 64 to 512 (147456 x 128 x 512: 28.4 against 50.2 us, 147456 x 128 x 510: 52 against 86, 65536 x 512 x 2048: 84
// against 110, 4096 x 64 x 64: 3.6 against 4.2); at 1024 rows and below it loses as often as it wins. Buffer
// accesses need rows of results at multiples of 4 bytes.
bool streams(const GemmArgs& a) {
    return a.M >= 2048 && a.M <= 1 << 30 && a.Kp <= 512 && a.N % 2 == 0 && a.N <= 1 << 20 && aligned16(a.out) &&
           aligned16(a.residual);
}

template <bool BF, int KB, int NU, int MF, bool RES>
void launch_stream(hipStream_t s, GemmArgs& a, int workgroups) {
    const auto go = [&](auto wn_) {
        constexpr int WN = decltype(wn_)::value;
        a.ntiles = (a.N + 16 * NU * WN - 1) / (16 * NU * WN);
        const int rows = 16 * MF * (4 / WN), mtiles = (a.M + rows - 1) / rows;
        const int most = std::max(1, workgroups / a.ntiles);
        const dim3 grid((unsigned)(std::min(mtiles, most) * a.ntiles)), block(256);
        if (!RES && a.lines) hipLaunchKernelGGL((q8_stream_kernel<BF, KB, NU, MF, WN, RES, !RES>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((q8_stream_kernel<BF, KB, NU, MF, WN, RES, false>), grid, block, 0, s, a);
    };
    if (a.N <= 16 * NU) go(std::integral_constant<int, 1>());
    else if (a.N <= 32 * NU) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
}

template <bool BF>
void launch(hipStream_t s, GemmArgs& a) {
    const int operands = (a.N + 63) / 64 * 4;
    if (a.M <= kFewRows) {
        hipLaunchKernelGGL(q8_rows_kernel<BF>, dim3((unsigned)operands), dim3(256), 0, s, a);
        return;
    }
#define CLK_TILE(MF_, NU_, WM_, WN_, KS_, RING_)                                                                 \
    {                                                                                                            \
        a.mtiles = (a.M + 16 * MF_ * WM_ - 1) / (16 * MF_ * WM_);                                                \
        a.ntiles = (operands + NU_ * WN_ - 1) / (NU_ * WN_);                                                     \
        hipLaunchKernelGGL((q8_tile_kernel<BF, MF_, NU_, WM_, WN_, KS_, RING_>),                                 \
                           dim3((unsigned)a.mtiles * (unsigned)a.ntiles), dim3(64 * WM_ * WN_ * KS_), 0, s, a);  \
        return;                                                                                                  \
    }
    // Up to 64 rows every wave works for itself (no barriers), eight of them splitting k. One operand of
    // channels a workgroup while that gives 256 workgroups at most, for every CU one, then two, which
    // halves the reading of the rows: 32 rows, 8192 to 8192: 15.7 and 13.0 us; 4096 to 4096: 5.9 and 6.6.
    if (a.M <= 16) CLK_TILE(1, 1, 1, 1, 4, 8)
    if (operands <= 256) {
        if (a.M <= 32) CLK_TILE(2, 1, 1, 1, 8, 5)
        if (a.M <= 48) CLK_TILE(3, 1, 1, 1, 8, 4)
        if (a.M <= 64) CLK_TILE(4, 1, 1, 1, 8, 4)
    } else {
        if (a.M <= 32) CLK_TILE(2, 2, 1, 1, 8, 4)
        if (a.M <= 48) CLK_TILE(3, 2, 1, 1, 8, 3)
        if (a.M <= 64) CLK_TILE(4, 2, 1, 1, 8, 3)
    }
    if (streams(a)) {
        // Operands a wave and workgroups, measured at 147456 and 65536 rows: with few channels, or none but
        // the results to move, small waves and more of them; with a residual at many channels, large ones
        // (147456 x 128 x 512 with a residual: 57 us with 8 channel operands a wave and 512 workgroups, 61 to 63
        // us with 4; without one 28.4 us with 4, 31.4 with 8).
        const int kbs = a.Kp / 64;
        const bool res = a.residual != nullptr;
        if (kbs == 1) {
            if (a.N <= 256) res ? launch_stream<BF, 1, 4, 1, true>(s, a, 768) : launch_stream<BF, 1, 4, 1, false>(s, a, 768);
            else res ? launch_stream<BF, 1, 8, 2, true>(s, a, 512) : launch_stream<BF, 1, 4, 2, false>(s, a, 1024);
        } else if (kbs == 2) {
            if (a.N <= 256) res ? launch_stream<BF, 2, 4, 1, true>(s, a, 768) : launch_stream<BF, 2, 4, 1, false>(s, a, 768);
            else res ? launch_stream<BF, 2, 8, 1, true>(s, a, 512) : launch_stream<BF, 2, 4, 2, false>(s, a, 1024);
        } else if (kbs <= 4) {
            res ? launch_stream<BF, 4, 4, 1, true>(s, a, 512) : launch_stream<BF, 4, 4, 1, false>(s, a, 512);
        } else {
            res ? launch_stream<BF, 8, 4, 1, true>(s, a, 512) : launch_stream<BF, 8, 4, 1, false>(s, a, 512);
        }
        return;
    }
    switch (best_tile(a.M, a.N, a.Kp)) {
    case 0: CLK_TILE(4, 8, 4, 2, 1, 4)
    case 1: CLK_TILE(4, 8, 2, 2, 1, 3)
    case 2: CLK_TILE(2, 4, 4, 2, 1, 4)
    default: CLK_TILE(2, 4, 2, 1, 2, 4)
    }
#undef CLK_TILE
}

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
    // a launch holds 2^32 threads: 256 for each 64 x 64 tile, or 512 for each 16 channels of up to 64 rows
    if (M > INT32_MAX - 256 || (M <= 64 ? nt >= 1 << 21 : nt >= 1 << 24 || (M + 63) / 64 * nt >= 1 << 24)) {
        return invalid("q8_projection: too large");
    }
    if (!aligned16(q->data) || !aligned16(wq->data)) return invalid("q8_projection: q and wq must be 16-byte aligned");
    GemmArgs a{static_cast<const int8_t*>(q->data), static_cast<const float*>(q_scale->data),
               static_cast<const int8_t*>(wq->data), static_cast<const float*>(w_scale->data),
               has_b ? static_cast<const float*>(b->data) : nullptr,
               has_residual ? static_cast<const half_t*>(residual->data) : nullptr, static_cast<half_t*>(out->data),
               (int)M, (int)N, (int)Kp, 0, 0,
               N % 64 == 0 && (reinterpret_cast<uintptr_t>(out->data) & 127u) == 0};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    stage_mark(s, 0);
    act == CLK_BF16 ? launch<true>(s, a) : launch<false>(s, a);
    stage_mark(s, 1);
    return launch_status("q8_projection");
}
