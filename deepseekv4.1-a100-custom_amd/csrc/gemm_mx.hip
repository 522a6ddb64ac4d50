// Dense product with FP4 weights on gfx950 block-scaled MFMA: y[m][n] = sum_k x[m][k] w[n][k], x as E2M1 or E4M3 codes and w as E2M1
// codes, both with one E8M0 byte per 32 k. Weights in the stored order of mx.h, activation codes row-major.
//
// v_mfma_scale_f32_32x32x64_f8f6f4: the weights are operand A (32 rows), the tokens operand B (32 columns), so lane l holds four
// consecutive n of token l % 32 in each register quad. FP4 x FP4 runs at twice the rate of FP4 x FP8 (7.4 against 4.0 PFLOP/s in a loop
// on registers; the 16x16x128 form reaches 4.0 for either).
#include "mx.h"

#include <atomic>
#include <type_traits>

struct MxArgs {
    const uint8_t* w; const uint8_t* s; int N, nk;             // weights of ceil(N/16) x nk tiles
    const uint8_t* xc; long long ldx; int row_b; const uint8_t* xs; int M;   // codes row-major, row_b (a multiple of 16) bytes a row; scales [nk][M][4]
    void* y; long long ldy; int dtype;
    int split; uint32_t* count; float* part;                   // parts of K; [tiles][4 waves] counters (zero) and [tiles][parts][4 waves][4][64][4] sums
};

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any 16-bit value's address
typedef __attribute__((address_space(3))) void lds_void;

template <int AF, int S>
__device__ __forceinline__ v16f mfma32(v8i a, v8i b, v16f c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, AF == 4 ? 4 : 0, S, sa, S, sb);
}

__device__ __forceinline__ v8i lo4(v4i a) { return v8i{a.x, a.y, a.z, a.w, 0, 0, 0, 0}; }
__device__ __forceinline__ v8i cat4(v4i a, v4i b) { return v8i{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}; }

template <int N>
__device__ __forceinline__ void wait_vm_lgkm() {   // s_waitcnt vmcnt(N) lgkmcnt(0)
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
}

// Up to a scheduling barrier: N matrix instructions with R operand reads spread behind the first half of them (all, without loads) and V
// loads behind the rest (the copies into LDS stay behind the reads before them). An instruction that waits
// for its turn behind several others leaves the matrix unit idle: a wave issues in order, and one wave per SIMD has no partner.
template <int N, int R, int V, int I = 0>
__device__ __forceinline__ void spread() {
    if constexpr (I < N) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        constexpr int H = V == 0 || N == 1 ? N : N / 2;
        if constexpr (I < H) __builtin_amdgcn_sched_group_barrier(0x100, (I + 1) * R / H - I * R / H, 0);
        if constexpr (V > 0 && I >= N - H) __builtin_amdgcn_sched_group_barrier(0x10, (I - N + H + 1) * V / H - (I - N + H) * V / H, 0);
        spread<N, R, V, I + 1>();
    } else {
        __builtin_amdgcn_sched_barrier(0);
    }
}

}  // namespace

// ------------------------------------------------------------------------------------------ tiles
// One workgroup of 2 x NT waves takes 64 WM weight rows x 32 WT NT tokens over the whole K, in stages of 128 KP k, NS of them in LDS. The
// load unit copies codes straight into LDS: weights in stored order, token rows in whole pieces of their own order, 16-byte piece c of row R
// at position c ^ f(R), so that 16 lanes' operand reads meet every bank once, and the scale bytes behind them (in registers they would have
// to be loaded as far ahead as the codes: a wave's loads complete in order). The tokens' scales are taken from [K / 128][M][4], where a
// stage's rows are contiguous: from row-major scales every row is a request of its own for four bytes, and requests are what a CU's path to
// L2 runs out of (2048 x 2048 x 16384, FP4, 128 x 128: 54.8 -> 41 us). One barrier per stage: behind it stage k's buffer has been read by
// every wave and stage k + 1 is complete; the last step of stage k still has its matrix instructions to go, so they cover the reads behind
// the barrier.
//
// Measured from codes (medians of a trace): 8192 x 8192 x 8192 in 262 us for FP4 (4.2 PFLOP/s; the matrix instructions alone, on the same random
// codes, take 225: the clock falls under them) and 371 us for FP8 (3.0 PFLOP/s of 4.0). 128 x 128 is bound by its rounds over the chip (2048 x 3328 x
// 7168, FP8: 416 tiles on 512 places, 43 us), 64 x 64 by what a CU's LDS gives: 16 KB of copies and 32 KB of operands per 256 k (97 x 5120 x 8192,
// FP4: 12.4 us).
template <int AF, int WM, int WT, int NT, int KP, int NS>
struct Tile {
    static constexpr int RB = KP * (AF == 4 ? 64 : 128);       // bytes of a token row per stage
    static constexpr int NWV = 2 * NT, BW = 64 * WM, BT = 32 * WT * NT;
    static constexpr int XO = BW * 64 * KP, SO = XO + BT * RB, SXO = SO + BW * 4 * KP;   // weights, tokens, their scales
    static constexpr int STAGE = SXO + BT * 4 * KP, RING = NS * STAGE;
    static constexpr bool DEEP = AF == 4 && WM * WT == 1;
    static constexpr int THREADS = 64 * NWV * (DEEP ? 2 : 1);
    // the outputs' way through LDS: 32 tokens of a wave's columns, fp32 rows at most
    static constexpr int OUT_LD = WM * 128 + 16, OUT_B = NWV * 32 * OUT_LD, LDS = RING > OUT_B ? RING : OUT_B;
};

template <int AF, int WM, int WT, int NT, int KP, int NS>
__device__ __forceinline__ void mx_gemm_tile(const MxArgs& a) {
    using C = Tile<AF, WM, WT, NT, KP, NS>;
    constexpr int RB = C::RB, NWV = C::NWV, BW = C::BW, BT = C::BT, XO = C::XO, STAGE = C::STAGE;
    constexpr int NWL = BW * KP / 16 / NWV, NXL = BT * RB / 1024 / NWV;   // 1 KiB copies per wave and stage
    static_assert(NWL * 16 * NWV == BW * KP && NXL * 1024 * NWV == BT * RB, "whole copies");
    constexpr int NSL = KP * (BW + BT) / 64 / NWV;             // 256-byte copies of scales per wave and stage: the weights' in the first waves
    static_assert(NSL * 64 * NWV == KP * (BW + BT) && BW == BT, "whole copies, half of the waves each");
    constexpr int PC = NWL + NXL + NSL;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, all = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool loader = C::DEEP && all >= NWV;
    const int wave = loader ? all - NWV : all;
    const int wr = wave & 1, wt = wave >> 1, l32 = lane & 31, g = lane >> 5;
    // Workgroup i runs on XCD i % 8: each XCD takes a run of consecutive tiles of an order that goes over the token tiles within four weight
    // tiles, so that the tiles at work on an XCD share their rows in its L2
    const int nW = (a.N + BW - 1) / BW, nT = (a.M + BT - 1) / BT, total = nW * nT * a.split, per = (total + 7) >> 3;
    const int at_x = (int)(blockIdx.x >> 3), o = (int)(blockIdx.x & 7) * per + at_x;
    if (at_x >= per || o >= total) return;
    const int tile = o / a.split, part_k = o - tile * a.split;
    const int panel = tile / (4 * nT), in_p = tile - panel * 4 * nT, wide = min(4, nW - panel * 4);
    const int tw = panel * 4 + in_p % wide, tt = in_p / wide;
    const int n0 = tw * BW, m0 = tt * BT;
    // this workgroup's part of K: ns stages from the k0th tile on, nk tiles from there to the end
    const int all_s = (a.nk + KP - 1) / KP, s0 = (int)((long long)all_s * part_k / a.split), ns = (int)((long long)all_s * (part_k + 1) / a.split) - s0;
    const int k0 = s0 * KP, nk = a.nk - k0;

    const int nb = (a.N + 15) / 16 - n0 / 16;                  // 16-row tiles from here on
    const int nbt = nb < BW / 16 ? nb : BW / 16, rows = a.M - m0 < BT ? a.M - m0 : BT;
    const __amdgpu_buffer_rsrc_t r_w = buffer_rsrc(a.w + ((long long)(n0 / 16) * a.nk + k0) * MX_TILE_B, (uint32_t)((nbt * a.nk - k0) * MX_TILE_B));
    const int row_b = a.row_b - s0 * RB;
    const __amdgpu_buffer_rsrc_t r_x = buffer_rsrc(a.xc + m0 * a.ldx + s0 * RB, (uint32_t)((rows - 1) * a.ldx + row_b));
    const bool sw = wave < NWV / 2;                            // this wave copies scales of the weights, or of the tokens
    const __amdgpu_buffer_rsrc_t r_s = sw ? buffer_rsrc(a.s + ((long long)(n0 / 16) * a.nk + k0) * MX_TILE_S, (uint32_t)((nbt * a.nk - k0) * MX_TILE_S))
                                          : buffer_rsrc(a.xs + (m0 + (long long)k0 * a.M) * 4, (uint32_t)((nk - 1) * a.M + rows) * 4u);
    constexpr uint32_t OUT = 0x80000000u;
    // A last stage that rows end in (K % 128 != 0; KP == 2: an odd number of tiles too): token pieces behind a row's end are another row's, and are
    // not fetched, which makes them zeros. KP == 2 and no second tile: nor are the scales of it, since another weight row's may be NaN's
    const int last_pieces = (row_b - (ns - 1) * RB) / 16;
    const bool part_row = last_pieces < RB / 16, odd = KP == 2 && nk < ns * KP;

    uint32_t w_off[NWL], x_off[NXL], s_off[NSL];
#pragma unroll
    for (int j = 0; j < NWL; ++j) {
        const int q = wave * NWL + j;
        w_off[j] = (uint32_t)((q / KP * a.nk + q % KP) * MX_TILE_B + lane * 16);
    }
    constexpr int PR = RB / 16, RI = 64 / PR;                  // pieces of a row, rows of a copy
    auto piece_of = [&](int R, int pos) {                      // the piece at a position of row R, and the position of a piece
        return pos ^ (PR == 4 ? (R >> 2) & 3 : PR == 8 ? (R >> 1) & 7 : R & 15);
    };
#pragma unroll
    for (int j = 0; j < NXL; ++j) {
        const int R = RI * (wave * NXL + j) + lane / PR;
        x_off[j] = R < rows ? (uint32_t)(R * a.ldx + piece_of(R, lane % PR) * 16) : OUT;
    }
    auto x_tail = [&](int j) {
        const int R = RI * (wave * NXL + j) + lane / PR;
        return piece_of(R, lane % PR) >= last_pieces ? OUT : x_off[j];
    };
    bool s_second[NSL];                                        // KP == 2: the lane's word belongs to the stage's second tile
#pragma unroll
    for (int j = 0; j < NSL; ++j) {
        const int at = ((sw ? wave : wave - NWV / 2) * NSL + j) * 64 + lane;   // word of the weights' [16 rows][tile][16 words] or the tokens' [tile][row]
        if (sw) {
            s_off[j] = (uint32_t)(at / (16 * KP) * a.nk * MX_TILE_S + at % (16 * KP) * 4);
            s_second[j] = KP == 2 && (at & 16);
        } else {
            const int R = at % BT;
            s_off[j] = R < rows ? (uint32_t)(at / BT * a.M + R) * 4u : OUT;
            s_second[j] = at >= BT;
        }
    }
    const int s_step = sw ? KP * MX_TILE_S : KP * 4 * a.M;
    const uint32_t s_dst = (uint32_t)((sw ? C::SO : C::SXO) + (sw ? wave : wave - NWV / 2) * NSL * 256);
    // Stage kb into the buffer at `so`. EDGE: kb may be the last stage or past it: offsets past every descriptor, so nothing is fetched and the
    // counts stay; inside, only the uniform offset changes from stage to stage.
    // PART 0: the weights and the scales, 1: the tokens, 2: both.
    auto issue_part = [&](int kb, uint32_t so, auto edge_c, auto part_c) {
        constexpr bool edge = decltype(edge_c)::value;
        constexpr int part = decltype(part_c)::value;
        const bool on = !edge || kb < ns, last = edge && kb == ns - 1;
        const uint32_t add = on ? 0u : OUT;
#pragma unroll
        for (int j = 0; j < (part == 1 ? 0 : NWL); ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_w, (lds_void*)(smem + so + (wave * NWL + j) * 1024), 16, w_off[j] | add,
                                                     on ? kb * KP * MX_TILE_B : 0, 0, 0);
#pragma unroll
        for (int j = 0; j < (part == 0 ? 0 : NXL); ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_x, (lds_void*)(smem + so + XO + (wave * NXL + j) * 1024), 16,
                                                     (last && part_row ? x_tail(j) : x_off[j]) | add, on ? kb * RB : 0, 0, 0);
#pragma unroll
        for (int j = 0; j < (part == 1 ? 0 : NSL); ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r_s, (lds_void*)(smem + so + s_dst + j * 256), 4, (last && odd && s_second[j] ? OUT : s_off[j]) | add,
                                                     on ? kb * s_step : 0, 0, 0);
    };
    v4i A[2][WM], B0[2][WT], B1[2][WT];
    uint32_t SW[2][WM], SX[2][WT];                             // scale half-words of a tile; set: the tile's place in its pair
    const uint32_t a_ofs = (uint32_t)((wr * WM * 2 + (l32 >> 4)) * KP * MX_TILE_B + g * 256 + (l32 & 15) * 16);
    const uint32_t b_row = (uint32_t)(XO + (wt * WT * 32 + l32) * RB);
    const uint32_t sw_ofs = (uint32_t)(C::SO + (wr * WM * 2 + (l32 >> 4)) * KP * MX_TILE_S + g * 32 + (l32 & 15) * 2);
    const uint32_t sx_ofs = (uint32_t)(C::SXO + (wt * WT * 32 + l32) * 4 + 2 * g);
    // Step s (two a tile) of the stage at `so` into an operand set; a tile's first step brings its scales into set `sc`
    auto read_ops = [&](uint32_t so, auto s_c, auto set_c, auto sc_c) {
        constexpr int s = decltype(s_c)::value, set = decltype(set_c)::value, v = s >> 1, h = s & 1, sc = decltype(sc_c)::value;
        const uint8_t* const st = smem + so;
        const auto at = [&](int c) { return b_row + piece_of(l32, c) * 16; };
        if constexpr (h == 0) {
#pragma unroll
            for (int i = 0; i < WM; ++i) SW[sc][i] = *(const uint16_t*)(st + sw_ofs + v * MX_TILE_S + i * 2 * KP * MX_TILE_S);
#pragma unroll
            for (int i = 0; i < WT; ++i) SX[sc][i] = *(const uint16_t*)(st + sx_ofs + v * BT * 4 + i * 32 * 4);
        }
#pragma unroll
        for (int i = 0; i < WM; ++i) A[set][i] = *(const v4i*)(st + a_ofs + v * MX_TILE_B + h * 512 + i * 2 * KP * MX_TILE_B);
#pragma unroll
        for (int i = 0; i < WT; ++i) {
            if constexpr (AF == 4) {
                B0[set][i] = *(const v4i*)(st + at(4 * v + 2 * g + h) + i * 32 * RB);
            } else {
                B0[set][i] = *(const v4i*)(st + at(8 * v + 2 * h + g) + i * 32 * RB);
                B1[set][i] = *(const v4i*)(st + at(8 * v + 4 + 2 * h + g) + i * 32 * RB);
            }
        }
    };
    v16f acc[WM][WT];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    auto mfmas = [&](auto set_c, auto sc_c) {                  // operand set (its step's scale byte too), scale set
        constexpr int set = decltype(set_c)::value, sc = decltype(sc_c)::value;
#pragma unroll
        for (int j = 0; j < WT; ++j) {
            const v8i bv = AF == 4 ? lo4(B0[set][j]) : cat4(B0[set][j], B1[set][j]);
#pragma unroll
            for (int i = 0; i < WM; ++i) acc[i][j] = mfma32<AF, set>(lo4(A[set][i]), bv, acc[i][j], (int)SW[sc][i], (int)SX[sc][j]);
        }
    };
    constexpr auto c0 = std::integral_constant<int, 0>{};
    constexpr auto c1 = std::integral_constant<int, 1>{};
    constexpr auto c2 = std::integral_constant<int, 2>{};
    constexpr auto c3 = std::integral_constant<int, 3>{};
    constexpr int n_mm = WM * WT, n_rd = WM + WT * (AF == 4 ? 1 : 2), n_sc = WM + WT;
    uint32_t cur = 0;                                          // buffer of the running stage
    auto next_of = [&](uint32_t so) { return so + STAGE == C::RING ? 0u : so + STAGE; };
    // Stage k; par: the scale set of its tile (KP == 1: k % 2; KP == 2: 0, and 1 for its second tile). Step s uses operand set s % 2. KP == 1: the
    // copies of stage k + NS go out in two parts, behind this stage's barrier and in the next stage's first step, so that the load path takes
    // them while matrix instructions run.
    uint32_t before = (NS - 1) * STAGE;                        // buffer of the stage before
    auto stage = [&](int k, auto par_c, auto edge_c) __attribute__((always_inline)) {
        constexpr int par = decltype(par_c)::value, last = KP == 2 ? 1 : par;
        read_ops(cur, c1, c1, par_c);
        if constexpr (KP == 1) issue_part(k - 1 + NS, before, edge_c, c1);
        mfmas(c0, par_c);
        spread<n_mm, n_rd, KP == 1 ? NXL : 0>();
        if constexpr (KP == 2) {
            read_ops(cur, c2, c0, c1);
            mfmas(c1, c0);
            spread<n_mm, n_rd + n_sc, 0>();
            read_ops(cur, c3, c1, c1);
            mfmas(c0, c1);
            spread<n_mm, n_rd, 0>();
        }
        wait_vm_lgkm<(NS - 2) * PC>();                         // this wave's copies of stage k + 1: those of NS - 2 stages are younger
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        const uint32_t nxt = next_of(cur);
        read_ops(nxt, c0, c0, std::integral_constant<int, KP == 2 ? 0 : 1 - par>{});
        issue_part(k + NS, cur, edge_c, std::integral_constant<int, KP == 1 ? 0 : 2>{});
        mfmas(c1, std::integral_constant<int, last>{});
        spread<n_mm, n_rd + n_sc, KP == 1 ? NWL + NSL : PC>();
        before = cur;
        cur = nxt;
    };
    constexpr auto inside = std::false_type{};
    constexpr auto edge = std::true_type{};
    // DEEP, FP4's one block of 32 x 32 per wave: its matrix instruction is far shorter than an operand read takes, so a whole stage is read at
    // once, behind the barrier that completes it, while the stage before it is multiplied; and the copies are sent by as many waves of their
    // own, since a wave stands still for the 16 cycles in which the load path takes one, which a stage's four matrix instructions do not hide
    // (97 x 5120 x 8192 15.7 -> 14.8 us, 512 x 4608 x 5120 25.2 -> 23.6). FP8's tokens take so many registers that only one workgroup then fits a
    // CU (512 x 4608 x 5120 31.6 -> 35.4 us): it keeps the steps.
    constexpr bool DEEP = C::DEEP;
    static_assert(!DEEP || (KP == 2 && AF == 4), "whole stages of four steps");
    v4i DA[2][4], DB[2][4];
    uint32_t DW[2][2], DX[2][2];
    auto read_stage = [&](uint32_t so, auto set_c) {
        constexpr int set = decltype(set_c)::value;
        const uint8_t* const st = smem + so;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            DW[set][v] = *(const uint16_t*)(st + sw_ofs + v * MX_TILE_S);
            DX[set][v] = *(const uint16_t*)(st + sx_ofs + v * BT * 4);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int v = q >> 1, h = q & 1;
            const auto at = [&](int c) { return b_row + piece_of(l32, c) * 16; };
            DA[set][q] = *(const v4i*)(st + a_ofs + v * MX_TILE_B + h * 512);
            DB[set][q] = *(const v4i*)(st + at(4 * v + 2 * g + h));
        }
    };
    auto deep_stage = [&](auto set_c) __attribute__((always_inline)) {
        constexpr int set = decltype(set_c)::value;
        wait_vm_lgkm<63>();                                    // stage k is in registers
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        cur = next_of(cur);
        read_stage(cur, std::integral_constant<int, 1 - set>{});
        __builtin_amdgcn_sched_barrier(0);
        acc[0][0] = mfma32<AF, 0>(lo4(DA[set][0]), lo4(DB[set][0]), acc[0][0], (int)DW[set][0], (int)DX[set][0]);
        acc[0][0] = mfma32<AF, 1>(lo4(DA[set][1]), lo4(DB[set][1]), acc[0][0], (int)DW[set][0], (int)DX[set][0]);
        acc[0][0] = mfma32<AF, 0>(lo4(DA[set][2]), lo4(DB[set][2]), acc[0][0], (int)DW[set][1], (int)DX[set][1]);
        acc[0][0] = mfma32<AF, 1>(lo4(DA[set][3]), lo4(DB[set][3]), acc[0][0], (int)DW[set][1], (int)DX[set][1]);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load_stage = [&](int k) {
        wait_vm_lgkm<(NS - 2) * PC>();                         // this wave's copies of stage k + 1
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        issue_part(k + NS, cur, edge, c2);                     // every wave has read stage k
        cur = next_of(cur);
    };
    if (!DEEP || loader) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            if (KP == 1 && i == NS - 1) issue_part(i, i * STAGE, edge, c0);   // its tokens follow in stage 0
            else issue_part(i, i * STAGE, edge, c2);
            __builtin_amdgcn_sched_barrier(0);   // the counted waits need the copies in stage order
        }
        wait_vm_lgkm<(NS - 1) * PC - (KP == 1 ? NXL : 0)>();
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    int k = 0;
    if constexpr (DEEP) {
        if (loader) {
            for (; k < ns; k += 2) {
                load_stage(k);
                load_stage(k + 1);
            }
        } else {
            read_stage(0, c0);
            for (; k < ns; k += 2) {                           // a stage past the last one multiplies zeros
                deep_stage(c0);
                deep_stage(c1);
            }
        }
    } else if constexpr (KP == 2) {
        read_ops(0, c0, c0, c0);
        for (; k + NS < ns - 1; ++k) stage(k, c0, inside);
        for (; k < ns; ++k) stage(k, c0, edge);
    } else {
        read_ops(0, c0, c0, c0);
        for (; k + 2 + NS < ns; k += 2) {
            stage(k, c0, inside);
            stage(k + 1, c1, inside);
        }
        for (; k + 1 < ns; k += 2) {
            stage(k, c0, edge);
            stage(k + 1, c1, edge);
        }
        if (k < ns) stage(k, c0, edge);
    }
    wait_vm_lgkm<0>();   // nothing of this wave may land in LDS any more, and no wave reads operands behind the barrier
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

    if (loader) return;

    if constexpr (WM * WT == 1) {
        // K in parts: every wave leaves its sums in memory, and the last of a tile's waves in this place to arrive adds all parts in their order,
        // its own among them. Nobody waits for anybody. The sums are stored and read at the device's scope, past the XCD's L2. What orders them
        // around the counter's step is that the stores have been acknowledged (the wait for vmcnt 0) before the counter moves, and that the loads
        // are issued after its answer: how gfx950 carries out these instructions. The fences only keep the compiler's order; between workgroups
        // the memory model would ask for a release and an acquire at the device's scope, which write back the whole L2 for every wave (97 x 5120 x
        // 8192 in three parts: 131 us).
        if (a.split > 1) {
            float* const sums = a.part + ((long long)tile * a.split * NWV + wave) * 1024 + lane;   // part p: 1024 NWV p behind
            float* const mine = sums + (long long)part_k * NWV * 1024;
#pragma unroll
            for (int q = 0; q < 16; ++q) __hip_atomic_store(mine + q * 64, acc[0][0][q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            wait_vm_lgkm<0>();
            uint32_t seen = 0;
            if (lane == 0) seen = __hip_atomic_fetch_add(a.count + tile * NWV + wave, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (__builtin_amdgcn_readfirstlane((int)seen) != a.split - 1) return;
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[0][0][q] = 0.f;
            for (int p = 0; p < a.split; ++p) {
                float v[16];
#pragma unroll
                for (int q = 0; q < 16; ++q) v[q] = __hip_atomic_load(sums + (long long)p * NWV * 1024 + q * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[0][0][q] += v[q];
            }
        }
    }

    // The outputs of 32 tokens at a time through this wave's own part of LDS, so that rows leave in 16-byte pieces of up to 512 contiguous
    // bytes (straight from the accumulators a lane holds four values of a row, and 32 rows would share every store).
    auto store = [&](auto dt_c) __attribute__((always_inline)) {
        constexpr int DT = decltype(dt_c)::value, ES = DT == MX_F32 ? 4 : 2, ROW = WM * 32 * ES, LD = ROW + 16;
        static_assert(LD <= C::OUT_LD, "rows of the outputs' way");
        uint8_t* const own = smem + wave * 32 * LD;
        const int nw = n0 + wr * WM * 32, nn = min(a.N - nw, WM * 32);   // this wave's columns
#pragma unroll
        for (int j = 0; j < WT; ++j) {
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint8_t* p = own + l32 * LD + (i * 32 + 8 * q + 4 * g) * ES;
                    const float c[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                    if constexpr (DT == MX_F32) *(v4f*)p = v4f{c[0], c[1], c[2], c[3]};
                    else *(uint2*)p = make_uint2(mx_pack2<DT>(c[0], c[1]), mx_pack2<DT>(c[2], c[3]));
                }
            const int mw = m0 + (wt * WT + j) * 32;
            constexpr int PER = ROW / 16, E = 16 / ES;
#pragma unroll
            for (int u = lane; u < 32 * PER; u += 64) {
                const int r = u / PER, n = (u % PER) * E;
                if (mw + r >= a.M || n >= nn) continue;
                const uint8_t* p = own + r * LD + n * ES;
                uint8_t* o = (uint8_t*)a.y + ((mw + r) * a.ldy + nw + n) * ES;
                if (n + E <= nn) *(v4i_any*)o = *(const v4i*)p;   // rows of y start at any value
                else
                    for (int b = 0; b < (nn - n) * ES; b += ES) {
                        if constexpr (ES == 4) *(uint32_t*)(o + b) = *(const uint32_t*)(p + b);
                        else *(uint16_t*)(o + b) = *(const uint16_t*)(p + b);
                    }
            }
        }
    };
    if (a.dtype == MX_BF16) store(std::integral_constant<int, MX_BF16>{});
    else if (a.dtype == MX_F16) store(std::integral_constant<int, MX_F16>{});
    else store(std::integral_constant<int, MX_F32>{});
}

template <int AF, int WM, int WT, int NT, int KP, int NS>
__global__ void __launch_bounds__((Tile<AF, WM, WT, NT, KP, NS>::THREADS)) mx_gemm_kernel(const MxArgs a) {
    mx_gemm_tile<AF, WM, WT, NT, KP, NS>(a);
}

// The kernel's dynamic LDS limit on the current device, set on its first launch there (`known`: one bit per device)
static int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& known) {
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return (int)e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (known.load(std::memory_order_relaxed) & bit) return 0;
    if (const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); e != hipSuccess) return (int)e;
    known.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

// `launch` false: only whether the launch can be made
template <int AF, int WM, int WT, int NT, int KP, int NS>
static int launch_tiles(const MxArgs& a, bool launch, hipStream_t st) {
    using C = Tile<AF, WM, WT, NT, KP, NS>;
    static_assert(C::LDS <= 160 * 1024, "LDS of one CU");
    static std::atomic<uint64_t> known{0};
    const long long tiles = ((long long)((a.N + C::BW - 1) / C::BW) * ((a.M + C::BT - 1) / C::BT) * a.split + 7) / 8 * 8;
    if (tiles > 0xFFFFFFFFll / C::THREADS) return DSV41_EINVAL;   // a launch holds fewer than 2^32 threads
    if (!launch) return 0;
    if (const int e = allow_lds((const void*)&mx_gemm_kernel<AF, WM, WT, NT, KP, NS>, C::LDS, known)) return e;
    mx_gemm_kernel<AF, WM, WT, NT, KP, NS><<<(unsigned)tiles, C::THREADS, C::LDS, st>>>(a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------ few rows
// Up to 16 rows: the weights are the traffic, read once. A workgroup takes 16 RB weight rows over the whole K. Waves 0 .. 7 stream the
// tiles (8 / RB of them along K, in turn, SK_PF pairs of 2 KiB each in flight from entry on); the others meanwhile bring the rows of x
// into LDS as codes, from the tensor (rounded here: one launch, no operand in memory) or from an operand. After one barrier the
// streaming waves multiply their tiles (v_mfma_scale_f32_16x16x128_f8f6f4: 16 weight rows, up to 16 rows of x), and their sums are
// added in wave order. Splitting the work by wave keeps the two streams' wait counters apart: a wave's loads complete in order, so
// rows loaded behind the tiles would arrive with the last of them.
// Measured with the rounding of x (medians of a trace): 1 x 5120 x 8192 FP4 8.2 us (2.7 TB/s of weights: 2 us until the first arrive, 1 us of joins,
// 320 workgroups on 256 CUs), 16 x 4608 x 5120 FP8 10.6 us (8.1 from codes: every workgroup rounds all rows; 144 workgroups).
// Lane (r = l % 16, q = l / 16) holds blocks 2 q and 2 q + 1 of a pair's eight in its two steps, so its two scale bytes are one half-word.
#define SK_STREAM 8
#define SK_QUANT 8
#define SK_PF 4
#define SK_QB 4
#define SK_MAX_M 16

struct MxRowsArgs {
    const uint8_t* w; const uint8_t* s; int N, K, nk;          // nk = ceil(K / 256): pairs of tiles
    const void* x; long long ldx; const uint8_t* xs; long long ldxs; int M;   // XT < 3: a tensor; XT == 3: codes and scales
    void* y; long long ldy; int dtype;
};

// LDS: codes of M rows (16 bytes of padding: 16 rows' reads meet every bank once), their scale bytes, the partial sums
template <int AF>
__host__ __device__ constexpr int sk_row(int nk) { return nk * (AF == 4 ? 128 : 256) + 16; }
__host__ __device__ constexpr int sk_srow(int nk) { return nk * 8 + 4; }
template <int AF>
static int sk_lds(int M, int nk) { return (M * (sk_row<AF>(nk) + sk_srow(nk)) + 15) / 16 * 16 + SK_STREAM * 1024; }

template <int AF, int XT, int RB>
__device__ __forceinline__ void mx_rows_item(const MxRowsArgs& a) {
    constexpr int KW = SK_STREAM / RB;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nk = a.nk, ldc = sk_row<AF>(nk), lds_s = sk_srow(nk), M = a.M;
    uint8_t* const sc = smem + M * ldc;
    float* const red = (float*)(smem + (M * (ldc + lds_s) + 15) / 16 * 16);
    const int tiles = (a.N + 15) >> 4;
    if (wave >= SK_STREAM) {
        const int qt = tid - SK_STREAM * 64;
        // units qt, qt + 512, .. of rows of `per` units, SK_QB of them loaded before the first is used; a unit past the last row is in row M
        int r = 0, c = qt;
        const auto step = [&](int per, float inv) {              // c < 2^20: the quotient of c + 1/2 is never a rounding away from an integer
            const int k = (int)(((float)c + 0.5f) * inv);
            r += k;
            c -= k * per;
        };
        constexpr uint32_t OUT = 0x80000000u;
        if constexpr (XT < 3) {
            constexpr int UB = XT == MX_F32 ? 32 : 16;           // bytes of a unit of eight values
            const int per = nk * 32, ldb = (int)a.ldx * (UB / 8);
            const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x, (uint32_t)((M - 1) * ldb + a.K * (UB / 8)));
            const float inv = 1.0f / (float)per;
            for (step(per, inv); r < M;) {
                Raw8<XT> v[SK_QB];
                int at[SK_QB], as[SK_QB];                        // where its codes and its scale byte go; -1: nowhere
#pragma unroll
                for (int i = 0; i < SK_QB; ++i) {
                    v[i].load(rx, r < M && c * 8 < a.K ? (uint32_t)(r * ldb + c * UB) : OUT);   // zeros beyond K
                    at[i] = r < M ? r * ldc + c * (AF == 4 ? 4 : 8) : -1;
                    as[i] = r * lds_s + (c >> 2);
                    c += SK_QUANT * 64;
                    step(per, inv);
                }
#pragma unroll
                for (int i = 0; i < SK_QB; ++i) {
                    uint32_t o[2];
                    const uint32_t b = mx_encode<AF == 4 ? 4 : 8>(v[i], o);
                    if (at[i] < 0) continue;
                    if constexpr (AF == 4) *(uint32_t*)(smem + at[i]) = o[0];
                    else *(uint2*)(smem + at[i]) = make_uint2(o[0], o[1]);
                    if ((tid & 3) == 0) sc[as[i]] = (uint8_t)b;
                }
            }
        } else {
            const int row_b = a.K * (AF == 4 ? 1 : 2) / 2, srow_b = a.K >> 5;   // K % 32 == 0: whole 16-byte pieces of codes
            const bool words = !((a.K & 127) | ((int)a.ldxs & 3) | ((int)(uintptr_t)a.xs & 3));   // whole scale words too
            const int per = nk * (AF == 4 ? 8 : 16), sper = nk * 2;
            const __amdgpu_buffer_rsrc_t rx = buffer_rsrc(a.x, (uint32_t)((M - 1) * (int)a.ldx + row_b));
            const __amdgpu_buffer_rsrc_t rxs = buffer_rsrc(a.xs, (uint32_t)((M - 1) * (int)a.ldxs + srow_b));
            const float inv = 1.0f / (float)per, sinv = 1.0f / (float)sper;
            for (step(sper, sinv); r < M;) {
                const uint32_t at = (uint32_t)(r * (int)a.ldxs + c * 4);
                uint32_t w = 0;
                if (words) {
                    w = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rxs, c * 4 < srow_b ? at : OUT, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w |= (uint32_t)(uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rxs, c * 4 + i < srow_b ? at + i : OUT, 0, 0) << (8 * i);
                }
                *(uint32_t*)(sc + r * lds_s + c * 4) = w;
                c += SK_QUANT * 64;
                step(sper, sinv);
            }
            r = 0;
            c = qt;
            for (step(per, inv); r < M;) {
                v4i v[SK_QB];
                int at[SK_QB];
#pragma unroll
                for (int i = 0; i < SK_QB; ++i) {
                    const uint32_t from = r < M && c * 16 < row_b ? (uint32_t)(r * (int)a.ldx + c * 16) : OUT;
                    v[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, from, 0, 0));
                    at[i] = r < M ? r * ldc + c * 16 : -1;
                    c += SK_QUANT * 64;
                    step(per, inv);
                }
#pragma unroll
                for (int i = 0; i < SK_QB; ++i)
                    if (at[i] >= 0) *(v4i*)(smem + at[i]) = v[i];
            }
        }
        __syncthreads();
    } else {
        const int rb = blockIdx.x * RB + wave / KW, kw = wave % KW;
        const bool on = rb < tiles;
        const int nt = (a.K + 127) >> 7;                         // tiles; the odd one of the last pair may be past them and reads zeros
        const __amdgpu_buffer_rsrc_t rw = buffer_rsrc(a.w + (long long)(on ? rb : 0) * nt * MX_TILE_B, on ? (uint32_t)nt * MX_TILE_B : 0u);
        const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(a.s + (long long)(on ? rb : 0) * nt * MX_TILE_S, on ? (uint32_t)nt * MX_TILE_S : 0u);
        const int r16 = lane & 15, q = lane >> 4;
        // q = 2 h + g: block 2 g + step of the even (h = 0) or odd tile
        const uint32_t wo = (uint32_t)((q >> 1) * MX_TILE_B + (q & 1) * 256 + r16 * 16), so = (uint32_t)((q >> 1) * MX_TILE_S + (q & 1) * 32 + r16 * 2);
        v4i A[SK_PF][2];
        int SA[SK_PF];
        const int n = (nk - kw + KW - 1) / KW;                   // this wave's tiles: kw, kw + KW, ..
        // a tile past the last one: offsets beyond the descriptors, zeros without a memory access
        auto load = [&](int slot, int it) {
            const uint32_t add = it < n ? 0u : 0x80000000u;
            const uint32_t t = it < n ? (uint32_t)(kw + it * KW) : 0u;
            A[slot][0] = buffer_load_tile(rw, wo | add, t * 2 * MX_TILE_B);
            A[slot][1] = buffer_load_tile(rw, (wo + 512) | add, t * 2 * MX_TILE_B);
            SA[slot] = (int)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, so | add, t * 2 * MX_TILE_S, 0);
        };
#pragma unroll
        for (int i = 0; i < SK_PF; ++i) {
            load(i, i);
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
        const int row = r16 < M ? r16 : M - 1;
        const uint8_t* const xr = smem + row * ldc;
        const uint8_t* const sr = sc + row * lds_s + 2 * q;
        v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
        auto use = [&](int slot, int it) {
            const int t = min(kw + it * KW, nk - 1);             // zero weights for a tile past the last one
            const int sb = *(const uint16_t*)(sr + t * 8);
            const auto opnd = [&](int step) {
                if constexpr (AF == 4) return lo4(*(const v4i*)(xr + t * 128 + (2 * q + step) * 16));
                else   // the FP8 operand holds half (q & 1) of blocks q / 2 and 2 + q / 2 of the step's four
                    return cat4(*(const v4i*)(xr + t * 256 + (2 * (q >> 1) + step) * 32 + (q & 1) * 16),
                                *(const v4i*)(xr + t * 256 + (2 * (2 + (q >> 1)) + step) * 32 + (q & 1) * 16));
            };
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(lo4(A[slot][0]), opnd(0), acc, 4, AF == 4 ? 4 : 0, 0, SA[slot], 0, sb);
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(lo4(A[slot][1]), opnd(1), acc, 4, AF == 4 ? 4 : 0, 1, SA[slot], 1, sb);
        };
        for (int it = 0; it < n; it += SK_PF) {
#pragma unroll
            for (int i = 0; i < SK_PF; ++i) {
                use(i, it + i);
                load(i, it + SK_PF + i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // lane: rows 4 q .. 4 q + 3 of the weight block for row r16 of x
        *(v4f*)(red + wave * 256 + r16 * 16 + 4 * q) = acc;
    }
    __syncthreads();
    for (int o = tid; o < M * RB * 16; o += (SK_STREAM + SK_QUANT) * 64) {
        const int m = o / (RB * 16), j = o % (RB * 16);
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) v += red[((j >> 4) * KW + k) * 256 + m * 16 + (j & 15)];
        const int nn = blockIdx.x * RB * 16 + j;
        if (nn >= a.N) continue;
        if (a.dtype == MX_F32) ((float*)a.y)[m * a.ldy + nn] = v;
        else ((uint16_t*)a.y)[m * a.ldy + nn] = (uint16_t)(a.dtype == MX_BF16 ? mx_pack<MX_BF16>(v) : mx_pack<MX_F16>(v));
    }
}

template <int AF, int XT, int RB>
__global__ void __launch_bounds__((SK_STREAM + SK_QUANT) * 64, 8) mx_rows_kernel(const MxRowsArgs a) {
    mx_rows_item<AF, XT, RB>(a);
}

template <int AF, int XT, int RB>
static int launch_rows_v(const MxRowsArgs& a, hipStream_t st) {
    static std::atomic<uint64_t> known{0};
    constexpr int threads = (SK_STREAM + SK_QUANT) * 64;
    const int blocks = ((a.N + 15) / 16 + RB - 1) / RB;
    if (blocks > 0xFFFFFFFFll / threads) return DSV41_EINVAL;   // a launch holds fewer than 2^32 threads: N < 2^29
    if (const int e = allow_lds((const void*)&mx_rows_kernel<AF, XT, RB>, 160 * 1024, known)) return e;
    mx_rows_kernel<AF, XT, RB><<<(unsigned)blocks, threads, sk_lds<AF>(a.M, a.nk), st>>>(a);
    return (int)hipGetLastError();
}

// Row blocks per workgroup: more of them (and so fewer waves along K) while the workgroups do not fit the chip at once, two to a CU or
// one, where x takes more than half of LDS or every workgroup has to bring in more than four rows of it. The rule leaves out where x comes
// from, so a tensor and its operand give the same sums.
template <int AF, int XT>
static int launch_rows(const MxRowsArgs& a, hipStream_t st) {
    if (a.M < 1 || a.M > SK_MAX_M || sk_lds<AF>(a.M, a.nk) > 160 * 1024 || (a.M > 1 && a.ldx > (1 << 24))) return DSV41_EINVAL;   // 32-bit offsets of rows
    const int fit = sk_lds<AF>(a.M, a.nk) > 80 * 1024 || a.M > 4 ? 256 : 512, tiles = (a.N + 15) / 16;
    if (tiles <= fit) return launch_rows_v<AF, XT, 1>(a, st);
    if (tiles <= 2 * fit) return launch_rows_v<AF, XT, 2>(a, st);
    if (tiles <= 4 * fit) return launch_rows_v<AF, XT, 4>(a, st);
    return launch_rows_v<AF, XT, 8>(a, st);
}

#define MX_ROWS 3   // plan: the kernel for few rows

// A plan of the C entries: the kernel in the low four bits, for tiles of 64 x 64 the number of K's parts above (0 and 1: whole)
static bool mx_bad_plan(int plan, int K) {
    const int kernel = plan & 15, parts = plan >> 4;
    return plan < 0 || kernel > MX_ROWS || (parts > 1 && (kernel != 0 || parts > (K + 255) / 256));
}
// Workspace behind `at` (the operand's end) for the parts' counters and sums; `end`: its length in all
struct MxParts {
    int n; long long count, part, end; int counters;
    MxParts(int plan, int N, int M, long long at) : n(plan >> 4 > 1 ? plan >> 4 : 1), count((at + 15) / 16 * 16), part(count), end(at), counters(0) {
        if (n == 1) return;
        const long long tiles = (long long)((N + 63) / 64) * ((M + 63) / 64);
        if (tiles > 1 << 20) { end = 0x7FFFFFFFFFFFFFFFll; return; }
        counters = (int)tiles * 4;
        part = count + counters * 4ll;
        end = part + tiles * n * 16384;
    }
};

static bool mx_bad_weights(const uint8_t* w, const uint8_t* s, int N, int K, const void* y, long long ldy, int out_type) {
    return !w || !s || !y || N < 1 || N > (1 << 30) || K < 32 || (K & 31) || K > (1 << 20) || out_type < 0 || out_type > 2 || ldy < N ||
           ((((uintptr_t)w) | ((uintptr_t)s) | ((uintptr_t)y)) & 15);
}

// The tile kernels, on scales [K / 128][M][4] (32-bit offsets into them); `launch` false: only whether they take the call, which is asked
// before the operand is made
static int mx_tiles(const MxArgs& a, int fmt, int plan, bool launch, hipStream_t st) {
    plan &= 15;
    if ((long long)a.M * a.nk > (1ll << 29) - 1) return DSV41_EINVAL;
    if (fmt == 4) {
        if (plan == 0) return launch_tiles<4, 1, 1, 2, 2, 4>(a, launch, st);
        if (plan == 1) return launch_tiles<4, 2, 2, 2, 1, 4>(a, launch, st);
        if (plan == 2) return launch_tiles<4, 4, 2, 4, 2, 2>(a, launch, st);
    } else {
        if (plan == 0) return launch_tiles<0, 1, 1, 2, 2, 3>(a, launch, st);
        if (plan == 1) return launch_tiles<0, 2, 2, 2, 1, 3>(a, launch, st);
        if (plan == 2) return launch_tiles<0, 4, 2, 4, 1, 3>(a, launch, st);
    }
    return DSV41_EINVAL;
}

extern "C" int dsv41_mx_gemm(const uint8_t* w, const uint8_t* s, int N, int K, const uint8_t* xc, long long ldx, const uint8_t* xs, long long ldxs,
                             int fmt, int M, int out_type, void* y, long long ldy, int plan, uint8_t* ws, long long ws_bytes, void* stream) {
    // strides: 32-bit offsets inside a tile
    if (mx_bad_weights(w, s, N, K, y, ldy, out_type) || !xc || !xs || M < 0 || (fmt != 4 && fmt != 8) || ldx < (fmt == 4 ? K / 2 : K) ||
        ldxs < K / 32 || (ldx & 15) || ldx > (1 << 21) || ldxs > (1 << 21) || (((uintptr_t)xc) & 15) || mx_bad_plan(plan, K))
        return DSV41_EINVAL;
    if (M == 0) return 0;
    const hipStream_t st = (hipStream_t)stream;
    if (plan == MX_ROWS) {
        const MxRowsArgs r{w, s, N, K, (K + 255) / 256, xc, ldx, xs, ldxs, M, y, ldy, out_type};
        return fmt == 4 ? launch_rows<4, 3>(r, st) : launch_rows<0, 3>(r, st);
    }
    const int nk = (K + 127) / 128;
    const MxParts parts(plan, N, M, 4ll * M * nk);
    if (!ws || (((uintptr_t)ws) & 15) || ws_bytes < parts.end) return DSV41_EINVAL;
    uint32_t* const count = (uint32_t*)(ws + parts.count);
    const MxArgs a{w, s, N, nk, xc, ldx, K / 8 * fmt, ws, M, y, ldy, out_type, parts.n, count, (float*)(ws + parts.part)};
    if (const int e = mx_tiles(a, fmt, plan, false, st)) return e;
    if (const int e = mx_turn_scales(xs, ldxs, M, K, ws, count, parts.counters, st)) return e;
    return mx_tiles(a, fmt, plan, true, st);
}

extern "C" int dsv41_mx_linear(const uint8_t* w, const uint8_t* s, int N, int K, const void* x, int dtype, long long ldx, int fmt, int M, int out_type,
                               void* y, long long ldy, int plan, uint8_t* ws, long long ws_bytes, void* stream) {
    const int es = dtype == MX_F32 ? 4 : 2;
    if (mx_bad_weights(w, s, N, K, y, ldy, out_type) || !x || dtype < 0 || dtype > 2 || M < 0 || (fmt != 4 && fmt != 8) || ldx < K || (ldx * es) % 16 ||
        (((uintptr_t)x) & 15) || mx_bad_plan(plan, K))
        return DSV41_EINVAL;
    if (M == 0) return 0;
    const hipStream_t st = (hipStream_t)stream;
    if (plan == MX_ROWS) {
        const MxRowsArgs r{w, s, N, K, (K + 255) / 256, x, ldx, nullptr, 0, M, y, ldy, out_type};
        if (dtype == MX_BF16) return fmt == 4 ? launch_rows<4, MX_BF16>(r, st) : launch_rows<0, MX_BF16>(r, st);
        if (dtype == MX_F16) return fmt == 4 ? launch_rows<4, MX_F16>(r, st) : launch_rows<0, MX_F16>(r, st);
        return fmt == 4 ? launch_rows<4, MX_F32>(r, st) : launch_rows<0, MX_F32>(r, st);
    }
    // the operand in the workspace, zero padded to whole 128-k tiles: codes [M][Kp fmt / 8], then scales [Kp / 128][M][4]
    const int nk = (K + 127) / 128;
    const long long row = (long long)nk * 16 * fmt;
    const MxParts parts(plan, N, M, M * (row + nk * 4));
    if (!ws || (((uintptr_t)ws) & 15) || ws_bytes < parts.end) return DSV41_EINVAL;
    uint32_t* const count = (uint32_t*)(ws + parts.count);
    const MxArgs a{w, s, N, nk, ws, row, (int)row, ws + M * row, M, y, ldy, out_type, parts.n, count, (float*)(ws + parts.part)};
    if (const int e = mx_tiles(a, fmt, plan, false, st)) return e;
    if (const int e = mx_quant_operand(x, dtype, M, K, ldx, fmt, nk, ws, ws + M * row, count, parts.counters, st)) return e;
    return mx_tiles(a, fmt, plan, true, st);
}
