// Orthogonalised updates: Newton-Schulz iteration on batches of matrices, and the optimiser step around it.
//
// With X = U / (|U|_F + eps) on its short side m <= n, one step is X <- p(A) X, A = X X^T, p(t) = a + b t + c t^2: every
// singular value s becomes s p(s^2).  A and all polynomials of it are symmetric and commute, so
//   * every m x m product is computed on the tiles of one triangle and written to both;
//   * several steps need X only once: M_i = p(A_i), Q <- M_i Q, A_{i+1} = M_i A_i M_i, then X <- Q X.  A block of k steps costs
//     3 m^2 n + (4 k - 3) m^3 multiplications and additions instead of k (3 m^2 n + m^3).
// The price of a block is precision: a rounding of A grows by a^2 with every A_{i+1} = M_i A_i M_i, where a step from X makes a new A.
// Two steps on one A cost nothing that shows: emulated over 25 spectra of 256 x 512 and 512 x 1024, |X| = 1 at the start, the result of
// five steps is off by at most 1.0e-4 (Frobenius norm, before its rounding) step by step, 8.3e-5 in blocks of two, 9.7e-5 in plain fp32;
// with a block of three first 2.3e-4, all five on one A 6.1e-3, and with coefficients as steep as 4.08, -6.89, 2.93 1.3e-3 and 7.1e-2.
// So blocks are two steps long, and only used where they save time.  On the GPU, against plain fp32 over seven spectra of seven sizes
// from 128 x 256 to 1024 x 4096: 0.4 to 1.5 times its error, at most 1.2e-4 (1.9e-4).
//
// Precision.  The first steps multiply small singular values by a each, 485 times over five steps with the usual coefficients,
// and rounding errors with them: with bf16 products the result is off by 2 to 20 %, with fp16 by 0.2 to 3 %.  Operands are
// therefore held as two fp16 halves, v = hi + lo (22 bits), and a product is hi hi + hi lo + lo hi with fp32 sums: fp32 grade
// at a third of the fp16 matrix rate.  Powers of two keep the halves inside fp16's range; they are chosen on the host from
// bounds of the polynomial over the range of singular values.
//
// A bf16 matrix scaled by a power of two fits one fp16 half, and stays so ("plain") until the first block has been applied to it:
// its Gram matrix is one product and Q X two (24 of 1024 x 4096: 150 us instead of 289 and 420 instead of 554, and 110 instead of
// 216 to lay them out; 3.45 ms instead of 3.72 in all, under a profiler).  What the power leaves of 2^e / (|U| + eps), a factor rho
// in [1, 2) of each matrix, multiplies the products' results.
//
// Storage of an operand with K columns: "split rows" with row stride ceil(K / 32) * 128 bytes, per 32 columns 64 bytes of hi and
// 64 of lo; "plain rows" of fp16 with row stride ceil(K / 64) * 128 bytes; zeros behind K.  A stage of the product's loop is one
// piece of 128 bytes of each row of split operands, 64 bytes of a plain operand beside it, or 128 of two plain ones.
#include "tile_common.h"

#include <math.h>

#include <type_traits>
#include <utility>

namespace sgclip {

typedef _Float16 f16_t;
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));

constexpr int OR_BATCH = 64;      // matrices per launch: their pointers travel as kernel arguments
constexpr int OR_PARTS = 64;      // partial sums of a matrix's squared norm
constexpr int OR_STEPS = 32;

static __host__ __device__ inline int or_chunks(int k) { return (k + 31) / 32; }
static __host__ __device__ inline int or_split_ld(int k) { return (k + 31) / 32 * 128; }
static __host__ __device__ inline int or_plain_ld(int k) { return (k + 63) / 64 * 128; }

struct OrPointers {
    void *p[OR_BATCH];
};

// The statement between: where v is a product in the compiler's sight, it rounds that to hi once in one place and by way of fp32 in
// another, and now and then lo belongs to a neighbour of hi (one element in 2^17 off by 2^-11).
__device__ __forceinline__ void or_split(float v, f16_t &hi, f16_t &lo) {
    asm("" : "+v"(v));
    hi = (f16_t)v;
    lo = (f16_t)(v - (float)hi);
}

// ---------------------------------------------------------------------------
// The products.  out[i][j] = sum_k L[i][k] R[j][k].
// ---------------------------------------------------------------------------
enum { OR_SYM = 0, OR_POLY = 1, OR_BOTH = 2, OR_OUT = 3, OR_UPDATE = 4 };
enum { OR_SPLIT = 0, OR_PLAIN = 1, OR_PLAIN_R = 2, OR_PLAIN_L = 3 };     // both operands split, both plain, one plain

struct OrGemm {
    const unsigned char *L[2], *R;     // [2]: two products with the same R in one launch (grid z)
    unsigned char *O[2];               // split rows [M][N], or with OR_BOTH also
    unsigned char *OT;                 // their transpose [N][M]
    const unsigned char *A;            // OR_POLY: A's split rows
    long long sL, sR, sO, sOT, sA;     // bytes from one matrix of the batch to the next
    float alpha[2];                    // from the accumulator's scale to the output's
    float ca, cb;                      // OR_POLY: out = alpha (ca I + cb A + A A), the first two in the accumulators from the start
    float decay, rate;                 // OR_UPDATE: p = decay p - rate out, rounded twice: decay p, and the whole (alpha is a power of two)
    long long ldo;                     // OR_OUT / OR_UPDATE: row stride in elements
    int M, N, kc, ldl, ldr;            // rows of L, rows of R, stages (0: none), bytes of their rows
    int tiles_m, tiles_n, wide;
    const float *rho;                  // with plain operands: each matrix's factor, once for every plain operand
    OrPointers out;                    // OR_OUT: bf16, OR_UPDATE: f32 parameters
};

// A wave's results in split rows: per 16 rows through the wave's own LDS, so that the stores are 16 bytes of whole pieces.
// Items of a row in memory order: per 32 columns four 16-byte units of hi, then four of lo.
__device__ __forceinline__ long long or_unit(int col) { return (long long)(col >> 5) * 128 + (col & 31) * 2; }

// v: the wave's results for 16 rows (m0 ..) x 16 SN columns (n0 ..); columns at or behind N are zeros in the padding.  lower: only the
// 16 x 16 blocks on and below the diagonal.
template <int SN>
__device__ __forceinline__ void or_store_rows(const f32x4 (&v)[SN], unsigned char *region, unsigned char *O, long long ld, int m0, int n0, int M,
                                              int N, bool lower, int lane) {
    constexpr int RS = SN * 64 + 16;     // bytes of a staged row: 16 SN columns x 4, and 16 against bank conflicts
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < SN; j++) {
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f16_t h, l;
            or_split(n0 + j * 16 + q * 4 + e < N ? v[j][e] : 0.f, h, l);
            hi[e] = h;
            lo[e] = l;
        }
        unsigned char *p = region + r * RS + (j * 2 + (q >> 1)) * 32 + (q & 1) * 8;
        *(f16x4 *)p = hi;
        *(f16x4 *)(p + 16) = lo;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int npad = or_chunks(N) * 32;
#pragma unroll
    for (int it0 = 0; it0 < 16 * SN * 4; it0 += 64) {
        const int it = it0 + lane, row = it / (SN * 4), w = it - row * (SN * 4);     // w: unit of 8 columns, hi / lo
        const int u = SN % 2 ? w >> 1 : (w >> 3) * 4 + (w & 3), half = SN % 2 ? w & 1 : (w >> 2) & 1;   // in memory order for whole pieces
        const int m = m0 + row, n = n0 + u * 8;
        if (m < M && n < npad && !(lower && (n >> 4) > (m >> 4))) *(f16x8 *)(O + m * ld + or_unit(n) + half * 64) = *(const f16x8 *)(region + row * RS + u * 32 + half * 16);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The transpose: 16 columns (n0 ..) of the wave's 16 SM rows (m0 ..) become 16 rows of OT; lower: only what lies below the diagonal.
template <int SM>
__device__ __forceinline__ void or_store_cols(const f32x4 (&v)[SM], unsigned char *region, unsigned char *OT, long long ld, int m0, int n0, int M,
                                              int N, bool lower, int lane) {
    constexpr int RS = SM * 64 + 16;
    const int r = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < SM; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            f16_t h, l;
            or_split(m0 + i * 16 + r < M ? v[i][e] : 0.f, h, l);
            unsigned char *p = region + (q * 4 + e) * RS + (i * 2 + (r >> 3)) * 32 + (r & 7) * 2;
            *(f16_t *)p = h;
            *(f16_t *)(p + 16) = l;
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int mpad = or_chunks(M) * 32;
#pragma unroll
    for (int it0 = 0; it0 < 16 * SM * 4; it0 += 64) {
        const int it = it0 + lane, row = it / (SM * 4), w = it - row * (SM * 4);
        const int u = SM % 2 ? w >> 1 : (w >> 3) * 4 + (w & 3), half = SM % 2 ? w & 1 : (w >> 2) & 1;   // in memory order for whole pieces
        const int n = n0 + row, m = m0 + u * 8;
        if (n < N && m < mpad && !(lower && (m >> 4) <= (n >> 4))) *(f16x8 *)(OT + n * ld + or_unit(m) + half * 64) = *(const f16x8 *)(region + row * RS + u * 32 + half * 16);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// A 16 x 16 block on the diagonal of a symmetric result, made exactly symmetric from its lower triangle.  What is left of
// asymmetry grows from step to step of a block (five on one Gram matrix were off by 1e-5 with it, by 1e-3 to 2e-2 without).
__device__ __forceinline__ void or_symmetrize(f32x4 &v, unsigned char *region, int lane) {
    const int r = lane & 15, q = lane >> 4;
    float *buf = (float *)region;
    *(f32x4 *)(buf + r * 20 + q * 4) = v;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float t = buf[(q * 4 + e) * 20 + r];     // the element across the diagonal
        if (q * 4 + e > r) v[e] = t;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// WM x WN waves of 16 SM rows x 16 SN columns.  SLOTS LDS slots of one stage each (32 columns, with OR_PLAIN 64); per stage
// three products, hi hi, hi lo and lo hi (of L and R), or with plain operands two: hi x and lo x, or the first and the last 32
// columns.  Fragments roll through one set of registers: those of L arrive a few products before their use and are replaced, hi
// by lo, row by row; in the middle of the last product every wave holds the rest of the stage, the next stage has landed (the
// one barrier), and the DMA of stage s + SLOTS starts into the slot just freed.
//   256 x 256: eight waves, 246 registers, 16.1 results per cycle and CU of 21.3 the matrix pipe could do;
//   192 x 192: eight waves, three slots; 128 x 128: four waves, two workgroups on a CU;
//   64 x 64: four waves, four slots, for few tiles, where a stage is shorter than its fetch.
// Bound by the matrix pipe and the fetches beside it (two 128 x 128 tiles on a CU: 2360 cycles a stage, 1500 without fetches, 1536
// at the matrix rate); the LDS is read half of the time.
template <int EPI, int FORM, int WM, int WN, int SM, int SN, int SLOTS>
__global__ __launch_bounds__(64 * WM * WN, 2) void or_gemm_kernel(OrGemm g) {
    constexpr int W = WM * WN, T = WM * SM * 16, LB = FORM == OR_PLAIN_L ? 64 : 128, RB = FORM == OR_PLAIN_R ? 64 : 128;   // bytes of a row's stage
    constexpr int OP = T * LB, SLOT = OP + T * RB, LP = OP / 1024 / W, RP = T * RB / 1024 / W;
    static_assert(T == WN * SN * 16 && LP * W * 1024 == OP && RP * W * 1024 == T * RB, "square tiles, whole pieces per wave");
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, r = lane & 15, q = lane >> 4;
    constexpr bool SYM = EPI == OR_SYM || EPI == OR_POLY;
    const int per = SYM ? g.tiles_m * (g.tiles_m + 1) / 2 : g.tiles_m * g.tiles_n;
    const int swz = xcd_remap(blockIdx.x, gridDim.x);
    const int b = swz / per, t = swz - b * per, z = blockIdx.z;
    int ti, tj;
    if (SYM) {      // t-th tile of the lower triangle, row by row
        ti = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= t) ti++;
        while (ti * (ti + 1) / 2 > t) ti--;
        tj = t - ti * (ti + 1) / 2;
    } else {
        ti = t / g.tiles_n;
        tj = t - ti * g.tiles_n;
    }
    ti = __builtin_amdgcn_readfirstlane(ti);
    tj = __builtin_amdgcn_readfirstlane(tj);
    const int m0 = ti * T, n0 = tj * T;
    const long long ldn = (long long)or_chunks(g.N) * 128, ldm = (long long)or_chunks(g.M) * 128;

    // DMA of a stage: pieces of 1024 bytes (8 or 16 rows), the wave's wave + W p, rows behind the matrix clamped to its last one
    auto piece_row = [&](int bytes) { return bytes == 128 ? wave * 8 + (lane >> 3) : wave * 16 + (lane >> 2); };
    auto piece_chunk = [&](int bytes, int row) {
        return (unsigned)((bytes == 128 ? (lane & 7) ^ ((row >> 1) & 7) : (lane & 3) ^ ((row >> 2) & 3)) * 16);
    };
    const int lrow = piece_row(LB), rrow = piece_row(RB);
    const unsigned lchunk = piece_chunk(LB, lrow), rchunk = piece_chunk(RB, rrow);
    const unsigned loff = (unsigned)(lrow * g.ldl) + lchunk, roff = (unsigned)(rrow * g.ldr) + rchunk;
    const unsigned lstep = (unsigned)(1024 / LB * W * g.ldl), rstep = (unsigned)(1024 / RB * W * g.ldr);
    const unsigned maxl = (unsigned)(min(g.M - 1 - m0, T - 1) * g.ldl) + lchunk, maxr = (unsigned)(min(g.N - 1 - n0, T - 1) * g.ldr) + rchunk;
    const unsigned char *lbase = (z ? g.L[1] : g.L[0]) + b * g.sL + m0 * (long long)g.ldl, *rbase = g.R + b * g.sR + n0 * (long long)g.ldr;
    const unsigned slots = (unsigned)(uintptr_t)LDS_PTR(lds) + wave * 1024;
    // piece p of the next stage to fetch: the wave's LP of L, then RP of R
    auto fetch_piece = [&](unsigned slot, int p) {
        if (p < LP) p64_dma16(lbase, loff, p * lstep, maxl, slot + p * (W * 1024));
        else p64_dma16(rbase, roff, (p - LP) * rstep, maxr, slot + OP + (p - LP) * (W * 1024));
    };
    const int mw = m0 + wm * SM * 16, nw = n0 + wn * SN * 16;
    f32x4 acc[SM][SN];
#pragma unroll
    for (int i = 0; i < SM; i++)
#pragma unroll
        for (int j = 0; j < SN; j++) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI == OR_POLY) {
        auto init = [&](f32x4 &v, f16x4 hi, f16x4 lo, int m, int n) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = g.cb * ((float)hi[e] + (float)lo[e]) + (m == n + e ? g.ca : 0.f);
        };
        const int npad = or_chunks(g.N) * 32;
#pragma unroll
        for (int i = 0; i < SM; i++) {
            const int m = mw + i * 16 + r;
            const unsigned char *a = g.A + b * g.sA + min(m, g.M - 1) * ldn;
            if constexpr (SN % 2 == 0) {
                // 32 columns, eight a lane; then neighbouring rows of 16 lanes, and halves of the wave, exchange to four of each 16
                typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
                for (int j = 0; j < SN; j += 2) {
                    u32x2 w[2][2];      // block j, j + 1; hi, lo
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const u32x4 v = *(const u32x4 *)(a + or_unit(min(nw + j * 16, npad - 32)) + h * 64 + q * 16);
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            const u32x2 x = __builtin_amdgcn_permlane16_swap(v[d], v[d + 2], false, false);
                            const u32x2 y = __builtin_amdgcn_permlane32_swap(x[0], x[1], false, false);
                            w[0][h][d] = y[0];
                            w[1][h][d] = y[1];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 2; k++)
                        init(acc[i][j + k], __builtin_bit_cast(f16x4, w[k][0]), __builtin_bit_cast(f16x4, w[k][1]), m, nw + (j + k) * 16 + q * 4);
                }
            } else {
#pragma unroll
                for (int j = 0; j < SN; j++) {
                    const unsigned char *p = a + or_unit(min(nw + j * 16, npad - 16) + q * 4);
                    init(acc[i][j], *(const f16x4 *)p, *(const f16x4 *)(p + 64), m, nw + j * 16 + q * 4);
                }
            }
        }
    }
    // a row 16 further has the same chunk order
    auto at = [](int bytes, int row, int chunk) { return bytes == 128 ? lds_off(row, chunk) : row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4); };
    const int lh0 = at(LB, wm * SM * 16 + r, q), ll0 = at(128, wm * SM * 16 + r, 4 + q);
    const int rh0 = OP + at(RB, wn * SN * 16 + r, q), rl0 = OP + at(128, wn * SN * 16 + r, 4 + q);
    f16x8 l[SM], rh[SN], rl[SN];
    constexpr int F = LP + RP, F1 = F / 2;
    static_assert(SLOTS >= 2 && (SLOTS - 1) * F < 64, "outstanding fetches within the counter");
    // Waits until at most `newer` of this wave's fetches are outstanding (whole), or none, with its LDS reads done; then for all waves.
    auto landed = [&](auto newer, bool whole) {
        if (whole) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(newer)::value) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // stage s + 1: stages up to s + SLOTS - 1 have been fetched as far as there are that many
    auto next_landed = [&](int s) { landed(std::integral_constant<int, (SLOTS - 2) * F>{}, s + SLOTS <= g.kc); };
    // A stage's F fetches start when its slot is free, behind the barrier: the first F1 in that stage's last product, the others in the
    // next stage's first one, so that they are taken (16 cycles each) as evenly as the products allow.
    auto fetch = [&](int slot, int from, int to) {
#pragma unroll
        for (int p = 0; p < F; p++)
            if (p >= from && p < to) fetch_piece(slots + slot, p);
        if (to == F) {
            lbase += LB;
            rbase += RB;
        }
    };
    const int full = g.kc >= SLOTS ? SLOTS - 1 : g.kc;
    for (int s = 0; s < full; s++) fetch(s * SLOT, 0, F);
    if (g.kc >= SLOTS) fetch((SLOTS - 1) * SLOT, 0, F1);
    landed(std::integral_constant<int, (SLOTS - 2) * F + F1>{}, g.kc >= SLOTS);
    constexpr int H = SM / 2;
#pragma unroll
    for (int i = 0; i < H; i++) l[i] = *(const f16x8 *)(lds + lh0 + i * 16 * LB);
#pragma unroll
    for (int j = 0; j < SN; j++) rh[j] = *(const f16x8 *)(lds + rh0 + j * 16 * RB);
    // a diagonal tile's wave above the diagonal only fetches: its block is written from below
    int slot = 0;
    if (SYM && mw + SM * 16 <= nw) {
        for (int s = 0; s < g.kc; s++) {
            if (s + SLOTS <= g.kc) fetch(slot == 0 ? (SLOTS - 1) * SLOT : slot - SLOT, F1, F);
            next_landed(s);
            if (s + SLOTS < g.kc) fetch(slot, 0, F1);
            slot = slot == (SLOTS - 1) * SLOT ? 0 : slot + SLOT;
        }
        __builtin_amdgcn_s_barrier();      // the one before the staging of the results
        return;
    }
    auto multiply = [&](int i, const f16x8(&rr)[SN]) {     // R first: a lane's four results are four consecutive columns of one row
#pragma unroll
        for (int j = 0; j < SN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(rr[j], l[i], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    // early: the rest of stage s + SLOTS - 1 is fetched; late: the start of stage s + SLOTS
    auto stage = [&](int s, auto early, auto late) {
        const int last = slot == 0 ? (SLOTS - 1) * SLOT : slot - SLOT;
        const int next = slot == (SLOTS - 1) * SLOT ? 0 : slot + SLOT;
        const unsigned char *cur = lds + slot, *nxt = lds + next;
        constexpr int G = SM - H;
        constexpr bool L2 = FORM != OR_PLAIN_L, R2 = FORM != OR_PLAIN_R;     // a second half in the stage
#pragma unroll
        for (int i = 0; i < SM; i++) {          // hi hi; the rest of L's hi fragments and R's lo fragments arrive
            if (i < G) l[H + i] = *(const f16x8 *)(cur + lh0 + (H + i) * 16 * LB);
            if constexpr (R2) {
#pragma unroll
                for (int j = i * SN / SM; j < (i + 1) * SN / SM; j++) rl[j] = *(const f16x8 *)(cur + rl0 + j * 2048);
            }
            if constexpr (decltype(early)::value) fetch(last, F1 + i * (F - F1) / SM, F1 + (i + 1) * (F - F1) / SM);
            multiply(i, rh);
            if constexpr (FORM != OR_SPLIT && L2) l[i] = *(const f16x8 *)(cur + ll0 + i * 2048);
        }
        if constexpr (FORM == OR_SPLIT) {
#pragma unroll
            for (int i = 0; i < SM; i++) {      // hi lo; L's lo fragments take the places of the hi ones
                multiply(i, rl);
                l[i] = *(const f16x8 *)(cur + ll0 + i * 2048);
            }
        }
        // the last product's R, and where the next stage's arrives
        constexpr bool LO = FORM == OR_PLAIN || FORM == OR_PLAIN_L;
        auto &rr = LO ? rl : rh, &rn = LO ? rh : rl;
#pragma unroll
        for (int i = 0; i < H; i++) multiply(i, rr);
        next_landed(s);
        // behind the last stage the reads return what the slot held before: not used
#pragma unroll
        for (int i = 0; i < G; i++) {           // lo hi; half of the next stage's hi fragments arrive
            if constexpr (decltype(late)::value) fetch(slot, i * F1 / G, (i + 1) * F1 / G);
            if (i < H) l[i] = *(const f16x8 *)(nxt + lh0 + i * 16 * LB);
#pragma unroll
            for (int j = i * SN / G; j < (i + 1) * SN / G; j++) rn[j] = *(const f16x8 *)(nxt + rh0 + j * 16 * RB);
            multiply(H + i, rr);
        }
        if constexpr (!LO) {
#pragma unroll
            for (int j = 0; j < SN; j++) rh[j] = rl[j];
        }
        slot = next;
    };
    int s = 0;
    for (; s + SLOTS < g.kc; s++) stage(s, std::true_type{}, std::true_type{});
    if (s + SLOTS == g.kc) stage(s++, std::true_type{}, std::false_type{});
    for (; s < g.kc; s++) stage(s, std::false_type{}, std::false_type{});

    float alpha = z ? g.alpha[1] : g.alpha[0];
    if constexpr (FORM != OR_SPLIT) alpha *= FORM == OR_PLAIN ? g.rho[b] * g.rho[b] : g.rho[b];
    if constexpr (EPI == OR_OUT || EPI == OR_UPDATE) {
#pragma unroll
        for (int i = 0; i < SM; i++)
#pragma unroll
            for (int j = 0; j < SN; j++) {
                const int m = mw + i * 16 + r, n = nw + j * 16 + q * 4;
                if (m >= g.M || n >= g.N) continue;
                const f32x4 v = acc[i][j];
                const long long at = m * g.ldo + n;
                if constexpr (EPI == OR_OUT) {
                    bf16_t *o = (bf16_t *)g.out.p[b] + at;
                    if (g.wide) {
                        bf16x4 w;
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = (bf16_t)(v[e] * alpha);
                        *(bf16x4 *)o = w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n + e < g.N) o[e] = (bf16_t)(v[e] * alpha);
                    }
                } else {
                    float *o = (float *)g.out.p[b] + at;
                    if (g.wide) {
                        float4 w = *(const float4 *)o;
                        w.x = fmaf(-g.rate, v[0] * alpha, w.x * g.decay);
                        w.y = fmaf(-g.rate, v[1] * alpha, w.y * g.decay);
                        w.z = fmaf(-g.rate, v[2] * alpha, w.z * g.decay);
                        w.w = fmaf(-g.rate, v[3] * alpha, w.w * g.decay);
                        *(float4 *)o = w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n + e < g.N) o[e] = fmaf(-g.rate, v[e] * alpha, o[e] * g.decay);
                    }
                }
            }
    } else {
        unsigned char *O = (z ? g.O[1] : g.O[0]) + b * g.sO;
#pragma unroll
        for (int i = 0; i < SM; i++)
#pragma unroll
            for (int j = 0; j < SN; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] *= alpha;
        // the last stage's unused reads are done with the LDS (lgkmcnt), every wave has passed its last barrier's reads
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        constexpr int REGION = SLOTS * SLOT / W / 16 * 16;
        unsigned char *region = lds + wave * REGION;
        static_assert(16 * (SM * 64 + 16) <= REGION && 16 * (SN * 64 + 16) <= REGION && 16 * 20 * 4 <= REGION, "a wave's staging fits its share of the LDS");
        const bool diagonal = SYM && ti == tj;
        if (diagonal) {
#pragma unroll
            for (int i = 0; i < SM; i++)
#pragma unroll
                for (int j = 0; j < SN; j++)
                    if (mw + i * 16 == nw + j * 16) or_symmetrize(acc[i][j], region, lane);
        }
#pragma unroll
        for (int i = 0; i < SM; i++) or_store_rows<SN>(acc[i], region, O, ldn, mw + i * 16, nw, g.M, g.N, diagonal, lane);
        unsigned char *OT = EPI == OR_BOTH ? g.OT + b * g.sOT : O;
#pragma unroll
        for (int j = 0; j < SN; j++) {
            f32x4 col[SM];
#pragma unroll
            for (int i = 0; i < SM; i++) col[i] = acc[i][j];
            or_store_cols<SM>(col, region, OT, ldm, mw, nw + j * 16, g.M, g.N, diagonal, lane);
        }
    }
}

// ---------------------------------------------------------------------------
// Before the products: the squared norm (and the momentum), then the two split forms of U / (|U| + eps).
// ---------------------------------------------------------------------------
struct OrInput {
    OrPointers g, buf;      // buf: momentum buffers (null without a step)
    long long ldg;
    int rows, cols;
    float mu;
    int nesterov, vec;      // vec: four columns per access
};

template <typename T, bool STEP>
__device__ __forceinline__ float or_direction(const OrInput &a, float g, float buf) {
    if constexpr (!STEP) return g;
    return a.nesterov ? fmaf(a.mu, buf, (1.0f - a.mu) * g) : buf;
}

template <typename T>
__device__ __forceinline__ float4 or_load4(const T *p) {
    if constexpr (sizeof(T) == 4) return *(const float4 *)p;
    const bf16x4 v = *(const bf16x4 *)p;
    return make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
}

// parts[matrix][part] = the part's sum of squares, in 64 bits: squares of large fp32 gradients pass fp32's range.  With STEP the
// momentum buffer is updated on the way: buf = mu buf + (1 - mu) g.
template <typename T, bool STEP>
__global__ __launch_bounds__(256) void or_norm_kernel(OrInput a, double *__restrict__ parts) {
    __shared__ double wsum[4];
    const T *g = (const T *)a.g.p[blockIdx.y];
    float *buf = (float *)a.buf.p[blockIdx.y];
    double s = 0.0;
    const int step = a.vec ? 4 : 1, per = a.cols / step;
    const long long total = (long long)a.rows * per;     // 65536^2 at most: i fits 32 bits
#pragma unroll 4
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += 256 * OR_PARTS) {
        long long at = i * step;
        if (a.ldg != a.cols) at += (unsigned)i / (unsigned)per * (a.ldg - a.cols);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), m = v;
        if (a.vec) v = or_load4(g + at);
        else v.x = (float)g[at];
        if constexpr (STEP) {
            float *bp = buf + i * step;
            if (a.vec) m = *(const float4 *)bp;
            else m.x = *bp;
            m.x = fmaf(a.mu, m.x, (1.0f - a.mu) * v.x);
            m.y = fmaf(a.mu, m.y, (1.0f - a.mu) * v.y);
            m.z = fmaf(a.mu, m.z, (1.0f - a.mu) * v.z);
            m.w = fmaf(a.mu, m.w, (1.0f - a.mu) * v.w);
            if (a.vec) *(float4 *)bp = m;
            else *bp = m.x;
        }
        const float x = or_direction<T, STEP>(a, v.x, m.x), y = or_direction<T, STEP>(a, v.y, m.y);
        const float z = or_direction<T, STEP>(a, v.z, m.z), w = or_direction<T, STEP>(a, v.w, m.w);
        s += ((double)x * x + (double)y * y) + ((double)z * z + (double)w * w);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) parts[blockIdx.y * OR_PARTS + blockIdx.x] = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
}

// 64 x 64 tiles: rows [rows][cols] and their transpose [cols][rows].  Split rows scaled by 2^e / (norm + eps); of bf16 matrices plain
// ones, exact but for what lies 2^-39 below the norm, scaled by the power of two below that, the rest of it in rho.
template <typename T, bool STEP>
__global__ __launch_bounds__(256) void or_split_kernel(OrInput a, const double *__restrict__ parts, float scale, float eps,
                                                       unsigned char *__restrict__ rowp, unsigned char *__restrict__ colp,
                                                       long long srow, long long scol, float *__restrict__ rho) {
    constexpr bool PLAIN = sizeof(T) == 2;
    __shared__ float tile[64][65];
    __shared__ double inv_s;
    const int tid = threadIdx.x, b = blockIdx.y;
    if (tid < 64) {
        double s = parts[b * OR_PARTS + tid];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        if (tid == 0) {
            const double inv = (double)scale / (sqrt(s) + (double)eps);
            inv_s = inv;
            if constexpr (PLAIN) {
                // the power of two: inv without its fraction; nothing (norm not finite), infinities and NaN stay what they are
                const double p = __longlong_as_double(__double_as_longlong(inv) & 0x7ff0000000000000LL);
                const bool usual = p > 0.0 && p <= 1.7976931348623157e308;
                if (usual) inv_s = p;
                if (blockIdx.x == 0) rho[b] = usual ? (float)(inv / p) : 1.0f;
            }
        }
    }
    __syncthreads();
    const double inv = inv_s;
    const T *g = (const T *)a.g.p[b];
    const float *buf = (const float *)a.buf.p[b];
    const int tc = (a.cols + 63) / 64;
    const int r0 = blockIdx.x / tc * 64, c0 = blockIdx.x % tc * 64;
    if (a.vec) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const int lr = (tid >> 4) + 16 * p, lc = (tid & 15) * 4, row = r0 + lr, col = c0 + lc;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f), m = v;
            if (row < a.rows && col < a.cols) {
                v = or_load4(g + row * a.ldg + col);
                if constexpr (STEP) m = *(const float4 *)(buf + (long long)row * a.cols + col);
            }
            tile[lr][lc] = (float)(or_direction<T, STEP>(a, v.x, m.x) * inv);
            tile[lr][lc + 1] = (float)(or_direction<T, STEP>(a, v.y, m.y) * inv);
            tile[lr][lc + 2] = (float)(or_direction<T, STEP>(a, v.z, m.z) * inv);
            tile[lr][lc + 3] = (float)(or_direction<T, STEP>(a, v.w, m.w) * inv);
        }
    } else {
        for (int p = 0; p < 16; p++) {
            const int lr = (tid >> 6) + 4 * p, lc = tid & 63, row = r0 + lr, col = c0 + lc;
            float v = 0.f;
            if (row < a.rows && col < a.cols)
                v = (float)(or_direction<T, STEP>(a, (float)g[row * a.ldg + col], STEP ? buf[(long long)row * a.cols + col] : 0.f) * inv);
            tile[lr][lc] = v;
        }
    }
    __syncthreads();
    if constexpr (PLAIN) {
        const long long ldr = or_plain_ld(a.cols), ldc = or_plain_ld(a.rows);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int lr = (tid >> 3) + 32 * p, l8 = (tid & 7) * 8;
            f16x8 v;
            if (r0 + lr < a.rows) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = (f16_t)tile[lr][l8 + e];
                *(f16x8 *)(rowp + b * srow + (r0 + lr) * ldr + (c0 + l8) * 2) = v;
            }
            if (c0 + lr < a.cols) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = (f16_t)tile[l8 + e][lr];
                *(f16x8 *)(colp + b * scol + (c0 + lr) * ldc + (r0 + l8) * 2) = v;
            }
        }
        return;
    }
    const long long ldr = or_split_ld(a.cols), ldc = or_split_ld(a.rows);
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const int lr = (tid >> 3) + 32 * p, l8 = (tid & 7) * 8;
        f16x8 hi, lo;
        if (r0 + lr < a.rows && c0 + l8 < or_chunks(a.cols) * 32) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f16_t h, l;
                or_split(tile[lr][l8 + e], h, l);
                hi[e] = h;
                lo[e] = l;
            }
            unsigned char *o = rowp + b * srow + (r0 + lr) * ldr + ((c0 + l8) >> 5) * 128 + (l8 & 31) * 2;
            *(f16x8 *)o = hi;
            *(f16x8 *)(o + 64) = lo;
        }
        if (c0 + lr < a.cols && r0 + l8 < or_chunks(a.rows) * 32) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                f16_t h, l;
                or_split(tile[l8 + e][lr], h, l);
                hi[e] = h;
                lo[e] = l;
            }
            unsigned char *o = colp + b * scol + (c0 + lr) * ldc + ((r0 + l8) >> 5) * 128 + (l8 & 31) * 2;
            *(f16x8 *)o = hi;
            *(f16x8 *)(o + 64) = lo;
        }
    }
}

// ---------------------------------------------------------------------------
// Matrices of few rows (m <= 128): up to 256 columns the whole step of one matrix in one workgroup, where a chain of launches would
// cost more than its products; beyond that (WIDE) a workgroup per 256 columns and a launch per step, between which X and each strip's
// part of X X^T pass through memory; every workgroup adds the parts, in order, and computes p(A) for itself.
// A wave keeps 16 columns of X (m <= 16 MT rows) in registers, from step to step.  They lie there as the matrix instruction leaves a
// result and, with the columns of M in the same order (32 of them: four of the first 16, then four of the second), takes its
// second operand, so that M X needs nothing of X but registers.  For A = X X^T the waves lay out X's rows in LDS, then A, then M; the
// lower 16 x 16 tiles of A and M are computed and written to both sides.
// Bound by one CU: of the 12 us of a step of 127 x 255, 5.4 are its matrix pipe's and 7.7 the LDS's (fragments, mostly of A and M),
// between five barriers.  Against the launches of or_gemm_kernel, us: 4 of 33 x 64 18 (67), of 64 x 64 19 (68), of 65 x 255 39 (85), of 128 x 128 45
// (79), of 127 x 255 66 (86); 200 of them 284 (442).  In strips: 4 of 64 x 513 46 (89), of 64 x 2000 55 (136), of 96 x 1023 72 (116), of
// 127 x 513 96 (97), of 127 x 2000 128 (163).
// A product's results are used in its own block of instructions, never behind a branch beside it: the compiler leaves the wait for the
// matrix instruction out where a longer path to the same place exists.
// ---------------------------------------------------------------------------
struct OrSmall {
    OrInput in;
    OrPointers out;
    long long ldo;
    int m, n, flip, steps;
    float scale, eps, decay, rate;
    // WIDE: the launch's place, 0 (X and its Gram matrix) to steps (step s - 1; the last writes the result), and what passes between them
    int launch;
    const double *parts;
    float *x, *gram[2];     // [batch][strips][..]: X as the threads hold it; sums of a strip's part of X X^T, written and read by turns
    struct {
        float gram, ca, cb, poly, apply;     // A = gram X X^T, M = poly (ca I + cb A + A A), X = apply M X
        int square;                          // 0: without A A
    } s[OR_STEPS];
};

// A and M, MT tiles wide: 16-byte units of a row, hi then lo
template <int MT>
struct OrSmallRows {
    static constexpr int UNITS = MT > 4 ? 16 : 8, LO = UNITS * 16, ROW = 2 * LO, REGION = MT * 16 * ROW;
    // where the four elements of row from column col lie
    static __device__ __forceinline__ int at(int row, int col) {
        return row * ROW + ((((col >> 5) * 4 + ((col & 15) >> 2)) ^ (row & (UNITS - 1))) << 4) + ((col >> 4) & 1) * 8;
    }
};

// Four neighbouring lanes' four values each, transposed: lane s of the four gets value s of all of them.
__device__ __forceinline__ f16x4 or_transpose4(f16x4 v, int lane) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const bool upper = lane & 2, odd = lane & 1;
    const unsigned keep = upper ? w[1] : w[0];
    const unsigned got = __builtin_amdgcn_update_dpp(0, upper ? w[0] : w[1], 0x4e, 0xf, 0xf, true);      // quad_perm 2 3 0 1
    const unsigned a = upper ? got : keep, b = upper ? keep : got;                                       // of the lower and of the upper pair
    const unsigned first = 0x05040100u, second = 0x07060302u;
    const unsigned mine = __builtin_amdgcn_perm(b, a, odd ? second : first);
    const unsigned other = __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_perm(b, a, odd ? first : second), 0xb1, 0xf, 0xf, true);   // 1 0 3 2
    return __builtin_bit_cast(f16x4, (u32x2){__builtin_amdgcn_perm(other, mine, odd ? 0x01000504u : first),
                                             __builtin_amdgcn_perm(other, mine, odd ? 0x03020706u : second)});
}

// a lane's four results, row i 16 + r, columns j 16 + q 4 .., and the same across the diagonal
template <int MT>
__device__ __forceinline__ void or_small_store(unsigned char *base, const f32x4 &v, int i, int j, int lane) {
    using Rows = OrSmallRows<MT>;
    const int r = lane & 15, q = lane >> 4;
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        f16_t h, l;
        or_split(v[e], h, l);
        hi[e] = h;
        lo[e] = l;
    }
    unsigned char *p = base + Rows::at(i * 16 + r, j * 16 + q * 4);
    *(f16x4 *)p = hi;
    *(f16x4 *)(p + Rows::LO) = lo;
    if (i == j) return;
    p = base + Rows::at(j * 16 + q * 4 + (r & 3), i * 16 + (r >> 2) * 4);
    *(f16x4 *)p = or_transpose4(hi, lane);
    *(f16x4 *)(p + Rows::LO) = or_transpose4(lo, lane);
}

// hi hi, then hi lo and lo hi
__device__ __forceinline__ void or_small_multiply(f32x4 &big, f32x4 &small, f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl) {
    big = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, big, 0, 0, 0);
    small = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, small, 0, 0, 0);
    small = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, small, 0, 0, 0);
}

// `count` of four elements `step` apart (the others zeros); four side by side in one access of any alignment
template <typename T>
__device__ __forceinline__ f32x4 or_small_load(const T *p, long long step, int count) {
    typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (step == 1 && count == 4) {
        const any4 w = *(const any4 *)p;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (float)w[e];
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < count) v[e] = (float)p[e * step];
    return v;
}

template <typename T, typename V>
__device__ __forceinline__ void or_small_write(T *p, long long step, int count, V v) {
    typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (step == 1 && count == 4) {
        *(any4 *)p = (any4){v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < count) p[e * step] = v[e];
}

template <typename T, bool STEP, int MT, int NW, bool WIDE>
__global__ __launch_bounds__(64 * NW) void or_small_kernel(OrSmall a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    __shared__ double wsum[NW];
    using Rows = OrSmallRows<MT>;
    constexpr int XROW = NW * 64, XLO = XROW / 2, NT = MT * (MT + 1) / 2, TILES = (NT + NW - 1) / NW;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, q = lane >> 4;
    const int strip = WIDE ? blockIdx.x : 0, strips = WIDE ? gridDim.x : 1, b = WIDE ? blockIdx.y : blockIdx.x;
    const int n = strip * (NW * 16) + wave * 16 + r;
    f32x4 x[MT], t[TILES];
    f16x8 xh[MT / 2], xl[MT / 2];

    // the wave's tiles of the lower triangle, row by row
    int ti[TILES], tj[TILES];
#pragma unroll
    for (int k = 0; k < TILES; k++) {
        const int t = wave + k * NW;
        ti[k] = (t >= 1) + (t >= 3) + (t >= 6) + (t >= 10) + (t >= 15) + (t >= 21) + (t >= 28);
        tj[k] = t - ti[k] * (ti[k] + 1) / 2;
    }
    const int sw = r & (Rows::UNITS - 1);

    // X = U 2^e / (|U| + eps)
    auto load = [&]() {
        const T *g = (const T *)a.in.g.p[b];
        float *buf = (float *)a.in.buf.p[b];
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < MT; i++) {
            const int m = i * 16 + q * 4, count = n < a.n ? min(max(a.m - m, 0), 4) : 0;
            x[i] = or_small_load(g + (a.flip ? n * a.in.ldg + m : m * a.in.ldg + n), a.flip ? 1 : a.in.ldg, count);
            if constexpr (STEP) {
                float *bp = buf + (a.flip ? (long long)n * a.in.cols + m : (long long)m * a.in.cols + n);
                const long long step = a.flip ? 1 : a.in.cols;
                f32x4 v = or_small_load(bp, step, count);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (!WIDE) v[e] = fmaf(a.in.mu, v[e], (1.0f - a.in.mu) * x[i][e]);      // (WIDE: done with the norm)
                    x[i][e] = or_direction<T, STEP>(a.in, x[i][e], v[e]);
                }
                if constexpr (!WIDE) or_small_write(bp, step, count, v);
            }
            if constexpr (!WIDE) {
#pragma unroll
                for (int e = 0; e < 4; e++) sum += (double)x[i][e] * x[i][e];
            }
        }
        if constexpr (WIDE) sum = a.parts[(long long)b * OR_PARTS + lane];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if constexpr (!WIDE) {
            if (lane == 0) wsum[wave] = sum;
            __syncthreads();
            sum = 0.0;
#pragma unroll
            for (int w = 0; w < NW; w++) sum += wsum[w];
        }
        const double inv = (double)a.scale / (sqrt(sum) + (double)a.eps);
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = (float)(x[i][e] * inv);
    };
    auto split = [&]() {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                f16_t h, l;
                or_split(x[i][e], h, l);
                xh[i / 2][i % 2 * 4 + e] = h;
                xl[i / 2][i % 2 * 4 + e] = l;
            }
    };
    // X's rows in LDS, and t = X X^T
    auto gram = [&]() {
#pragma unroll
        for (int i = 0; i < MT; i++) {
            f16x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                hi[e] = xh[i / 2][i % 2 * 4 + e];
                lo[e] = xl[i / 2][i % 2 * 4 + e];
            }
            const int row = i * 16 + q * 4 + (r & 3);
            unsigned char *p = lds + row * XROW + (((wave * 2 + (r >> 3)) ^ (row & 15)) << 4) + ((r >> 2) & 1) * 8;
            *(f16x4 *)p = or_transpose4(hi, lane);
            *(f16x4 *)(p + XLO) = or_transpose4(lo, lane);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TILES; k++) {
            t[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (wave + k * NW >= NT) continue;
            const unsigned char *left = lds + (ti[k] * 16 + r) * XROW, *right = lds + (tj[k] * 16 + r) * XROW;
            f32x4 small = t[k];
#pragma unroll
            for (int c = 0; c < NW / 2; c++) {
                const int u = ((c * 4 + q) ^ r) << 4;
                or_small_multiply(t[k], small, *(const f16x8 *)(right + u), *(const f16x8 *)(right + XLO + u), *(const f16x8 *)(left + u),
                                  *(const f16x8 *)(left + XLO + u));
            }
#pragma unroll
            for (int e = 0; e < 4; e++) t[k][e] += small[e];
        }
    };
    // X = p(A) X, A from t; nothing else may be using the LDS
    auto apply = [&](const auto &p) {
#pragma unroll
        for (int k = 0; k < TILES; k++) {
#pragma unroll
            for (int e = 0; e < 4; e++) t[k][e] *= p.gram;
            if (wave + k * NW < NT) or_small_store<MT>(lds, t[k], ti[k], tj[k], lane);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TILES; k++) {
            if (wave + k * NW >= NT) continue;
            f32x4 v = {0.f, 0.f, 0.f, 0.f}, small = v;
            const unsigned char *left = lds + (ti[k] * 16 + r) * Rows::ROW, *right = lds + (tj[k] * 16 + r) * Rows::ROW;
#pragma unroll
            for (int c = 0; c < MT / 2; c++) {
                const int u = ((c * 4 + q) ^ sw) << 4;
                or_small_multiply(v, small, *(const f16x8 *)(right + u), *(const f16x8 *)(right + Rows::LO + u), *(const f16x8 *)(left + u),
                                  *(const f16x8 *)(left + Rows::LO + u));
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float line = p.cb * t[k][e] + (ti[k] == tj[k] && q * 4 + e == r ? p.ca : 0.f);
                v[e] = (p.square ? line + (v[e] + small[e]) : line) * p.poly;
            }
            or_small_store<MT>(lds + Rows::REGION, v, ti[k], tj[k], lane);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MT; i++) {
            f32x4 v = {0.f, 0.f, 0.f, 0.f}, small = v;
            const unsigned char *left = lds + Rows::REGION + (i * 16 + r) * Rows::ROW;
#pragma unroll
            for (int c = 0; c < MT / 2; c++) {
                const int u = ((c * 4 + q) ^ sw) << 4;
                or_small_multiply(v, small, *(const f16x8 *)(left + u), *(const f16x8 *)(left + Rows::LO + u), xh[c], xl[c]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = (v[e] + small[e]) * p.apply;
            if constexpr (MT * NW > 64) __builtin_amdgcn_sched_barrier(0);     // or too many fragments are read ahead for the registers
        }
        __syncthreads();     // before the next X takes the place of M
    };

    if constexpr (!WIDE) {
        load();
        for (int s = 0; s < a.steps; s++) {
            split();
            gram();
            __syncthreads();
            apply(a.s[s]);
        }
    } else {
        float *dump = a.x + ((long long)b * strips + strip) * (MT * NW * 256) + tid * 4;
        if (a.launch == 0) load();
        else {
#pragma unroll
            for (int i = 0; i < MT; i++) x[i] = *(const f32x4 *)(dump + i * (NW * 256));
            const float *in = a.gram[a.launch & 1] + (long long)b * strips * (NT * 256) + lane * 4;
#pragma unroll
            for (int k = 0; k < TILES; k++) t[k] = (f32x4){0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < strips; s++)
#pragma unroll
                for (int k = 0; k < TILES; k++)
                    if (wave + k * NW < NT) t[k] += *(const f32x4 *)(in + ((long long)s * NT + wave + k * NW) * 256);
            split();
            apply(a.s[a.launch - 1]);
        }
        if (a.launch < a.steps) {
            split();
            gram();
            float *out = a.gram[(a.launch & 1) ^ 1] + ((long long)b * strips + strip) * (NT * 256) + lane * 4;
#pragma unroll
            for (int k = 0; k < TILES; k++)
                if (wave + k * NW < NT) *(f32x4 *)(out + (wave + k * NW) * 256) = t[k];
#pragma unroll
            for (int i = 0; i < MT; i++) *(f32x4 *)(dump + i * (NW * 256)) = x[i];
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < MT; i++) {
        const int m = i * 16 + q * 4, count = n < a.n ? min(max(a.m - m, 0), 4) : 0;
        const long long at = a.flip ? n * a.ldo + m : m * a.ldo + n, step = a.flip ? 1 : a.ldo;
        if constexpr (STEP) {
            float *o = (float *)a.out.p[b] + at;
            f32x4 p = or_small_load(o, step, count);
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = fmaf(-a.rate, x[i][e], p[e] * a.decay);
            or_small_write(o, step, count, p);
        } else {
            bf16x4 v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (bf16_t)x[i][e];
            or_small_write((bf16_t *)a.out.p[b] + at, step, count, v);
        }
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct OrPlan {
    int m, n, flip;                          // short and long side; flip: the matrix has more rows than columns
    size_t x, xt, sq, total;                 // bytes per matrix: X, X^T, one m x m operand; all of it
    int few, mt, strips;                     // few rows: or_small_kernel's, 16-row tiles and strips of OR_STRIP columns
};

constexpr int OR_STRIP = 256;

static OrPlan or_plan(int rows, int cols) {
    OrPlan p;
    p.flip = rows > cols;
    p.m = p.flip ? cols : rows;
    p.n = p.flip ? rows : cols;
    p.x = (size_t)p.m * or_split_ld(p.n);
    p.xt = (size_t)p.n * or_split_ld(p.m);
    p.sq = (size_t)p.m * or_split_ld(p.m);
    p.total = p.x + 2 * p.xt + 5 * p.sq + (OR_PARTS + 1) * sizeof(double);     // with the norm's parts and rho
    p.few = p.m <= 128 && p.n <= 16 * OR_STRIP;
    p.mt = p.m <= 64 ? 4 : p.m <= 96 ? 6 : 8;
    p.strips = (p.n + OR_STRIP - 1) / OR_STRIP;
    const size_t wide = OR_PARTS * sizeof(double) + (size_t)p.strips * (p.mt * 16 * OR_STRIP + p.mt * (p.mt + 1) * 256) * sizeof(float);
    if (p.few && p.strips > 1 && p.total < wide) p.total = wide;
    return p;
}

// largest e with bound 2^e <= 2^15 (half of fp16's range is left for rounding), at most 14; false where the bound is too large
static bool or_exponent(double bound, int &e) {
    if (!(bound <= 4096.0)) return false;
    e = bound <= 0 ? 14 : (int)floor(15.0 - log2(bound));
    if (e > 14) e = 14;
    return true;
}

struct OrStep {
    double a, b, c;
    int em, et, ea;     // exponents of M = p(A), of T = A M and of A' = M A M
};

// The steps' blocks and exponents from bounds over the range of singular values.
struct OrSchedule {
    int steps, blocks, len[OR_STEPS];
    int ex[OR_STEPS + 1], ea0[OR_STEPS], eq[OR_STEPS];   // X at a block's start, its Gram matrix; Q after each step of its block
    OrStep s[OR_STEPS];
};

static bool or_schedule(const float *coefficients, int steps, int m, int n, OrSchedule &o) {
    o.steps = steps;
    // Two steps at most (the head of this file says why), where they save time: updates in us, two steps on one Gram matrix against single
    // ones, 24 of 256 x 512 166 and 171, of 512 x 1024 589 and 596, of 1024 x 2048 2511 and 2829, of 1024 x 4096 4015 and 5179; but 24 of
    // 512 x 640 480 and 427, one of 768 x 1152 207 and 190, 24 of 200 x 400 149 and 151, one of them 112 and 105 (more launches)
    const int most = n < 2LL * m || m < 256 ? 1 : 2;
    o.blocks = (steps + most - 1) / most;
    for (int i = 0; i < o.blocks; i++) o.len[i] = steps / o.blocks + (i < steps % o.blocks);
    double top = 1.0, qb = 1.0;     // bounds of the singular values (1 after the normalisation) and of Q
    for (int k = 0, blk = 0, in = 0; k < steps; k++) {
        const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
        if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
        o.s[k].a = a;
        o.s[k].b = b;
        o.s[k].c = c;
        if (in == 0 && (!or_exponent(top, o.ex[blk]) || !or_exponent(top * top, o.ea0[blk]))) return false;
        double pm = 0, tm = 0, next = 0;
        for (int i = 0; i <= 1024; i++) {
            const double s = top * i / 1024, t = s * s, p = fabs(a + b * t + c * t * t);
            pm = fmax(pm, p);
            tm = fmax(tm, t * p);
            next = fmax(next, s * p);
        }
        if (!or_exponent(pm, o.s[k].em) || !or_exponent(tm, o.s[k].et) || !or_exponent(next * next, o.s[k].ea)) return false;
        qb = in == 0 ? pm : qb * pm;
        if (!or_exponent(qb, o.eq[k])) return false;
        top = next;
        if (++in == o.len[blk]) {
            in = 0;
            blk++;
        }
    }
    return or_exponent(top, o.ex[o.blocks]);
}

template <int EPI, int FORM, int WM, int WN, int SM, int SN, int SLOTS>
static int or_launch_tile(const OrGemm &g, long long blocks, int products, hipStream_t stream) {
    constexpr int LDS = SLOTS * (WM * SM * 16) * (FORM == OR_PLAIN_L || FORM == OR_PLAIN_R ? 192 : 256);
    if (!lds_attr((const void *)or_gemm_kernel<EPI, FORM, WM, WN, SM, SN, SLOTS>, LDS)) return SGCLIP_ELAUNCH;
    or_gemm_kernel<EPI, FORM, WM, WN, SM, SN, SLOTS><<<dim3((unsigned)blocks, 1, products), 64 * WM * WN, LDS, stream>>>(g);
    return launch_check("sgclip_orthogonalize");
}

template <int EPI, int FORM = OR_SPLIT>
static int or_launch(const OrGemm &gin, int batch, int products, hipStream_t stream) {
    OrGemm g = gin;
    constexpr bool SYM = EPI == OR_SYM || EPI == OR_POLY;
    auto tiles = [&](int T) {
        g.tiles_m = ceil_div(g.M, T);
        g.tiles_n = ceil_div(g.N, T);
        return (long long)batch * (SYM ? (long long)g.tiles_m * (g.tiles_m + 1) / 2 : (long long)g.tiles_m * g.tiles_n);
    };
    if (tiles(64) * products * 256 > 0xffffffffLL) {   // a launch counts its threads in 32 bits
        set_error("sgclip_orthogonalize: %d matrices of %d x %d are more than one launch holds", batch, g.M, g.N);
        return SGCLIP_EINVAL;
    }
    // 64 x 64 tiles where 128 x 128 do not give every CU one (two of 127 x 255: 104 us, with 128 x 128 151 us).  Otherwise the tile whose
    // rounds over the chip cost least: cycles of a stage measured at 1024 x 4096 and 768 x 768, 4080 for a 256 x 256 tile, 2400 for
    // 192 x 192, 2330 for two 128 x 128 tiles that share a CU (16.1, 15.4 and 14.1 results per cycle: the larger the tile, the fewer
    // bytes fetched per product).  48 of 768 x 768: 192 where X is written (3 rounds), 128 on the triangles; 24 of 1024 x 4096: 256.
    const int cus = device_cus();
    constexpr bool HALF = FORM == OR_PLAIN_L || FORM == OR_PLAIN_R;     // smaller stages: three slots instead of two
    if (tiles(128) * products < cus) return or_launch_tile<EPI, FORM, 2, 2, 2, 2, 4>(g, tiles(64), products, stream);
    auto cost = [&](int T, int slots, int cycles) { return (tiles(T) * products + slots - 1) / slots * cycles; };
    const long long c128 = cost(128, 2 * cus, 2330), c192 = cost(192, cus, 2400), c256 = cost(256, cus, 4080);
    if (c256 <= c128 && (HALF || c256 <= c192)) return or_launch_tile<EPI, FORM, 2, 4, 8, 4, HALF ? 3 : 2>(g, tiles(256), products, stream);
    if constexpr (!HALF) {     // pieces of a 64-byte operand do not divide a 192 x 192 tile among eight waves
        if (c192 < c128) return or_launch_tile<EPI, FORM, 2, 4, 6, 3, 3>(g, tiles(192), products, stream);
    }
    return or_launch_tile<EPI, FORM, 2, 2, 4, 4, HALF ? 3 : 2>(g, tiles(128), products, stream);
}

static inline float or_pow2(int e) { return ldexpf(1.0f, e); }

// M = p(A) in the accumulators' scale: alpha (ca I + cb A + A A), for A scaled by 2^ea and M by 2^em.  A coefficient c below the
// rounding of the others' terms is none: then nothing is multiplied.
struct OrPoly {
    float alpha, ca, cb;
    bool square;
};

static OrPoly or_poly(const OrStep &s, int ea) {
    OrPoly p;
    p.square = fabs(s.c) > 1e-12 * fmax(fabs(s.a), fabs(s.b));
    const double c = p.square ? ldexp(s.c, s.em - 2 * ea) : 1.0;
    p.alpha = (float)c;
    p.ca = (float)(ldexp(s.a, s.em) / c);
    p.cb = (float)(ldexp(s.b, s.em - ea) / c);
    return p;
}

template <typename T, bool STEP, int MT, int NW, bool WIDE>
static int or_launch_small(const OrSmall &a, int batch, hipStream_t stream) {
    constexpr int X = MT * 16 * NW * 64, AM = 2 * OrSmallRows<MT>::REGION, LDS = X > AM ? X : AM;
    static_assert(!WIDE || NW * 16 == OR_STRIP, "a strip per workgroup");
    if (!lds_attr((const void *)or_small_kernel<T, STEP, MT, NW, WIDE>, LDS)) return SGCLIP_ELAUNCH;
    const dim3 grid = WIDE ? dim3(ceil_div(a.n, OR_STRIP), batch) : dim3(batch);
    or_small_kernel<T, STEP, MT, NW, WIDE><<<grid, 64 * NW, LDS, stream>>>(a);
    return launch_check("sgclip_orthogonalize");
}

// Up to 128 x 4096, step by step.
template <typename T, bool STEP>
static int or_run_few(const OrInput &in, const OrPointers &out, long long ldo, int batch, const OrSchedule &sch, float eps, float decay, float rate,
                      unsigned char *ws, hipStream_t stream) {
    const OrPlan plan = or_plan(in.rows, in.cols);
    OrSmall a{};
    a.in = in;
    a.out = out;
    a.ldo = ldo;
    a.flip = plan.flip;
    a.m = plan.m;
    a.n = plan.n;
    a.steps = sch.steps;
    a.scale = or_pow2(sch.ex[0]);
    a.eps = eps;
    a.decay = decay;
    a.rate = rate;
    for (int k = 0; k < sch.steps; k++) {
        const OrStep &s = sch.s[k];
        const OrPoly p = or_poly(s, sch.ea0[k]);
        a.s[k].gram = or_pow2(sch.ea0[k] - 2 * sch.ex[k]);
        a.s[k].ca = p.ca;
        a.s[k].cb = p.cb;
        a.s[k].poly = p.alpha;
        a.s[k].square = p.square;
        a.s[k].apply = or_pow2((k + 1 < sch.steps ? sch.ex[k + 1] : 0) - s.em - sch.ex[k]);
    }
    if (plan.strips == 1) {
        if (plan.mt == 4) return a.n <= 128 ? or_launch_small<T, STEP, 4, 8, false>(a, batch, stream) : or_launch_small<T, STEP, 4, 16, false>(a, batch, stream);
        if (plan.mt == 6) return a.n <= 128 ? or_launch_small<T, STEP, 6, 8, false>(a, batch, stream) : or_launch_small<T, STEP, 6, 16, false>(a, batch, stream);
        return a.n <= 128 ? or_launch_small<T, STEP, 8, 8, false>(a, batch, stream) : or_launch_small<T, STEP, 8, 16, false>(a, batch, stream);
    }
    double *parts = (double *)ws;
    a.parts = parts;
    a.x = (float *)(parts + (size_t)OR_PARTS * batch);
    a.gram[0] = a.x + (size_t)batch * plan.strips * plan.mt * 16 * OR_STRIP;
    a.gram[1] = a.gram[0] + (size_t)batch * plan.strips * plan.mt * (plan.mt + 1) / 2 * 256;
    or_norm_kernel<T, STEP><<<dim3(OR_PARTS, batch), 256, 0, stream>>>(in, parts);
    int rc = launch_check("sgclip_orthogonalize");
    for (a.launch = 0; a.launch <= a.steps && rc == SGCLIP_OK; a.launch++)
        rc = plan.mt == 4   ? or_launch_small<T, STEP, 4, 16, true>(a, batch, stream)
             : plan.mt == 6 ? or_launch_small<T, STEP, 6, 16, true>(a, batch, stream)
                            : or_launch_small<T, STEP, 8, 16, true>(a, batch, stream);
    return rc;
}

// One launch group of up to OR_BATCH matrices.  in: gradients (and momentum buffers); out: bf16 results or parameters.
template <typename T, bool STEP>
static int or_run(const OrInput &in, const OrPointers &out, long long ldo, int batch, const OrSchedule &sch, float eps, float decay, float rate,
                  unsigned char *ws, hipStream_t stream) {
    const OrPlan p = or_plan(in.rows, in.cols);
    // One workgroup: at every size and number. Strips: while they fill the chip once (16 of 127 x 4000 225 us, by launches of
    // or_gemm_kernel 320; 40 of them 578, 475), up to 64 rows always (40 of 64 x 4000 192, 360).
    if (p.few && (p.strips == 1 || p.mt == 4 || batch * p.strips <= device_cus()))
        return or_run_few<T, STEP>(in, out, ldo, batch, sch, eps, decay, rate, ws, stream);
    unsigned char *X = ws, *XT = X + p.x * batch, *XT2 = XT + p.xt * batch, *A = XT2 + p.xt * batch, *M = A + p.sq * batch, *Tm = M + p.sq * batch,
                  *Q = Tm + p.sq * batch, *Q2 = Q + p.sq * batch;
    double *parts = (double *)(Q2 + p.sq * batch);
    float *rho = (float *)(parts + (size_t)OR_PARTS * batch);
    bool plain = sizeof(T) == 2;     // X and X^T, until the first block has been applied
    or_norm_kernel<T, STEP><<<dim3(OR_PARTS, batch), 256, 0, stream>>>(in, parts);
    const int tiles = ceil_div(in.rows, 64) * ceil_div(in.cols, 64);
    or_split_kernel<T, STEP><<<dim3(tiles, batch), 256, 0, stream>>>(in, parts, or_pow2(sch.ex[0]), eps, p.flip ? XT : X, p.flip ? X : XT,
                                                                     p.flip ? p.xt : p.x, p.flip ? p.x : p.xt, rho);
    int rc = launch_check("sgclip_orthogonalize");
    const int km = or_chunks(p.m);
    for (int blk = 0, k = 0; blk < sch.blocks && rc == SGCLIP_OK; blk++) {
        int ea = sch.ea0[blk], eq = 0;
        OrGemm g{};
        g.M = g.N = p.m;
        g.L[0] = g.R = X;
        g.O[0] = A;
        g.sL = g.sR = (long long)p.x;
        g.sO = (long long)p.sq;
        g.ldl = g.ldr = plain ? or_plain_ld(p.n) : or_split_ld(p.n);
        g.kc = g.ldl / 128;
        g.rho = rho;
        g.alpha[0] = or_pow2(ea - 2 * sch.ex[blk]);
        rc = plain ? or_launch<OR_SYM, OR_PLAIN>(g, batch, 1, stream) : or_launch<OR_SYM>(g, batch, 1, stream);
        g.sL = g.sR = g.sA = (long long)p.sq;
        g.kc = km;
        g.ldl = g.ldr = or_split_ld(p.m);
        for (int i = 0; i < sch.len[blk] && rc == SGCLIP_OK; i++, k++) {
            const OrStep &s = sch.s[k];
            const bool last = i + 1 == sch.len[blk];
            // M = a I + b A + c A A (into Q on the block's first step)
            g.L[0] = g.R = g.A = A;
            unsigned char *Mi = i == 0 ? Q : M;
            g.O[0] = Mi;
            const OrPoly poly = or_poly(s, ea);
            g.alpha[0] = poly.alpha;
            g.ca = poly.ca;
            g.cb = poly.cb;
            g.kc = poly.square ? km : 0;
            if ((rc = or_launch<OR_POLY>(g, batch, 1, stream)) != SGCLIP_OK) break;
            g.kc = km;
            if (i == 0) eq = s.em;
            // T = A M and Q = Q M, whichever are needed
            int np = 0;
            g.R = Mi;
            if (!last) {
                g.L[np] = A;
                g.O[np] = Tm;
                g.alpha[np++] = or_pow2(s.et - ea - s.em);
            }
            if (i > 0) {
                g.L[np] = Q;
                g.O[np] = Q2;
                g.alpha[np++] = or_pow2(sch.eq[k] - eq - s.em);
                eq = sch.eq[k];
            }
            if (np && (rc = or_launch<OR_SYM>(g, batch, np, stream)) != SGCLIP_OK) break;
            if (i > 0) {
                unsigned char *swap = Q;
                Q = Q2;
                Q2 = swap;
            }
            if (!last) {     // A = T M
                g.L[0] = Tm;
                g.O[0] = A;
                g.alpha[0] = or_pow2(s.ea - s.et - s.em);
                ea = s.ea;
                if ((rc = or_launch<OR_SYM>(g, batch, 1, stream)) != SGCLIP_OK) break;
            }
        }
        if (rc != SGCLIP_OK) break;
        // X = Q X: rows of Q against rows of X^T; the last one goes out in the matrix's own orientation
        g.L[0] = Q;
        g.R = XT;
        g.sL = (long long)p.sq;
        g.sR = (long long)p.xt;
        g.ldr = plain ? or_plain_ld(p.m) : or_split_ld(p.m);
        g.M = p.m;
        g.N = p.n;
        if (blk + 1 < sch.blocks) {
            g.O[0] = X;          // read by nothing in this product; X^T is, so its successor goes to the other buffer
            g.sO = (long long)p.x;
            g.OT = XT2;
            g.sOT = (long long)p.xt;
            g.alpha[0] = or_pow2(sch.ex[blk + 1] - eq - sch.ex[blk]);
            rc = plain ? or_launch<OR_BOTH, OR_PLAIN_R>(g, batch, 1, stream) : or_launch<OR_BOTH>(g, batch, 1, stream);
            plain = false;
            unsigned char *swap = XT;
            XT = XT2;
            XT2 = swap;
        } else {
            if (p.flip) {
                g.L[0] = XT;
                g.R = Q;
                g.sL = (long long)p.xt;
                g.sR = (long long)p.sq;
                std::swap(g.ldl, g.ldr);
                g.M = p.n;
                g.N = p.m;
            }
            g.out = out;
            g.ldo = ldo;
            g.alpha[0] = or_pow2(-eq - sch.ex[blk]);
            g.decay = decay;
            g.rate = rate;
            g.wide = g.N % 4 == 0 && ldo % 4 == 0;
            for (int i = 0; i < batch; i++) g.wide = g.wide && ((uintptr_t)out.p[i] & 15) == 0;
            if constexpr (STEP) rc = or_launch<OR_UPDATE>(g, batch, 1, stream);
            else if (!plain) rc = or_launch<OR_OUT>(g, batch, 1, stream);
            else rc = p.flip ? or_launch<OR_OUT, OR_PLAIN_L>(g, batch, 1, stream) : or_launch<OR_OUT, OR_PLAIN_R>(g, batch, 1, stream);
        }
    }
    return rc;
}

}  // namespace sgclip

using namespace sgclip;

static bool or_args_ok(const char *who, int rows, int cols, const float *coefficients, int steps, float eps, OrSchedule &sch) {
    if (rows <= 0 || cols <= 0 || rows > 65536 || cols > 65536) {
        set_error("%s: bad shape rows=%d cols=%d (1 to 65536)", who, rows, cols);
        return false;
    }
    if (!coefficients || steps < 1 || steps > OR_STEPS || !(eps >= 0.f)) {
        set_error("%s: bad steps=%d (1 to %d), coefficients or eps=%g", who, steps, OR_STEPS, (double)eps);
        return false;
    }
    const OrPlan p = or_plan(rows, cols);
    if (!or_schedule(coefficients, steps, p.m, p.n, sch)) {
        set_error("%s: with these coefficients singular values or a step's polynomial grow beyond fp16's range", who);
        return false;
    }
    return true;
}

static bool or_workspace_ok(const char *who, const void *ws, size_t have, int batch, int rows, int cols) {
    const size_t need = sgclip_orthogonalize_workspace_bytes(batch, rows, cols);
    if (!ws || have < need || ((uintptr_t)ws & 15)) {
        set_error("%s: workspace of %zu bytes, %zu needed (16-byte aligned)", who, ws ? have : (size_t)0, need);
        return false;
    }
    return true;
}

extern "C" {

size_t sgclip_orthogonalize_workspace_bytes(int batch, int rows, int cols) {
    if (batch <= 0 || rows <= 0 || cols <= 0) return 0;
    return or_plan(rows, cols).total * (size_t)(batch < OR_BATCH ? batch : OR_BATCH);
}

int sgclip_orthogonalize(const void *g_dev, int g_dtype, int64_t batch_stride, int64_t ldg, int batch, int rows, int cols,
                         const float *coefficients, int steps, float eps, void *out_dev, int64_t out_batch_stride, int64_t ldo,
                         void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *who = "sgclip_orthogonalize";
    if (batch == 0) return SGCLIP_OK;
    OrSchedule sch;
    if (!or_args_ok(who, rows, cols, coefficients, steps, eps, sch)) return SGCLIP_EINVAL;
    if (batch < 0 || !g_dev || !out_dev || ldg < cols || ldo < cols || (g_dtype != SGCLIP_DTYPE_F32 && g_dtype != SGCLIP_DTYPE_BF16) ||
        (batch > 1 && out_batch_stride < (int64_t)(rows - 1) * ldo + cols)) {
        set_error("%s: bad matrices (batch %d, dtype %d, row strides %lld and %lld, output batch stride %lld, cols %d)", who, batch, g_dtype,
                  (long long)ldg, (long long)ldo, (long long)out_batch_stride, cols);
        return SGCLIP_EINVAL;
    }
    if (!or_workspace_ok(who, workspace_dev, workspace_bytes, batch, rows, cols)) return SGCLIP_ENOSPC;
    const size_t size = g_dtype == SGCLIP_DTYPE_F32 ? 4 : 2;
    int rc = SGCLIP_OK;
    for (int b0 = 0; b0 < batch && rc == SGCLIP_OK; b0 += OR_BATCH) {
        const int n = batch - b0 < OR_BATCH ? batch - b0 : OR_BATCH;
        OrInput in{};
        OrPointers out{};
        in.ldg = ldg;
        in.rows = rows;
        in.cols = cols;
        in.vec = cols % 4 == 0 && ldg % 4 == 0;
        for (int i = 0; i < n; i++) {
            in.g.p[i] = (char *)g_dev + (b0 + i) * batch_stride * (int64_t)size;
            out.p[i] = (char *)out_dev + (b0 + i) * out_batch_stride * 2;
            in.vec = in.vec && ((uintptr_t)in.g.p[i] & 15) == 0;
        }
        rc = g_dtype == SGCLIP_DTYPE_F32
                 ? or_run<float, false>(in, out, ldo, n, sch, eps, 1.f, 0.f, (unsigned char *)workspace_dev, (hipStream_t)stream)
                 : or_run<bf16_t, false>(in, out, ldo, n, sch, eps, 1.f, 0.f, (unsigned char *)workspace_dev, (hipStream_t)stream);
    }
    return rc;
}

int sgclip_muon_step(float *const *params, const float *const *grads, float *const *momenta, int count, int rows, int cols, float momentum,
                     int nesterov, float lr, float weight_decay, float scale, const float *coefficients, int steps, float eps,
                     void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *who = "sgclip_muon_step";
    if (count == 0) return SGCLIP_OK;
    OrSchedule sch;
    if (!or_args_ok(who, rows, cols, coefficients, steps, eps, sch)) return SGCLIP_EINVAL;
    if (count < 0 || !params || !grads || !momenta) {
        set_error("%s: bad count %d or pointer tables", who, count);
        return SGCLIP_EINVAL;
    }
    for (int i = 0; i < count; i++)
        if (!params[i] || !grads[i] || !momenta[i]) {
            set_error("%s: matrix %d has a null parameter, gradient or momentum", who, i);
            return SGCLIP_EINVAL;
        }
    if (!or_workspace_ok(who, workspace_dev, workspace_bytes, count, rows, cols)) return SGCLIP_ENOSPC;
    int rc = SGCLIP_OK;
    for (int b0 = 0; b0 < count && rc == SGCLIP_OK; b0 += OR_BATCH) {
        const int n = count - b0 < OR_BATCH ? count - b0 : OR_BATCH;
        OrInput in{};
        OrPointers out{};
        in.ldg = cols;
        in.rows = rows;
        in.cols = cols;
        in.mu = momentum;
        in.nesterov = nesterov;
        in.vec = cols % 4 == 0;
        for (int i = 0; i < n; i++) {
            in.g.p[i] = (void *)grads[b0 + i];
            in.buf.p[i] = momenta[b0 + i];
            out.p[i] = params[b0 + i];
            in.vec = in.vec && (((uintptr_t)in.g.p[i] | (uintptr_t)in.buf.p[i]) & 15) == 0;
        }
        rc = or_run<float, true>(in, out, cols, n, sch, eps, (float)(1.0 - (double)lr * weight_decay), (float)((double)lr * scale),
                                 (unsigned char *)workspace_dev, (hipStream_t)stream);
    }
    return rc;
}

}  // extern "C"
