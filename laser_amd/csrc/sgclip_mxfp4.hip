// Microscaled 4-bit floats (OCP MX: e2m1 elements, one e8m0 scale per 32 consecutive elements of a row): quantisation,
// the way back, and the linear layer  y = epilogue(x W^T + bias)  on v_mfma_scale_f32_16x16x128_f8f6f4.
//
// Storage of a [rows, cols] matrix, kp = cols rounded up to 256 (zero codes behind cols):
//   codes   u8 [rows][kp / 2], element k in byte k / 2, even k in the low nibble;
//   scales  u8 [ceil(rows / 64)][kp / 32][16][4]: the byte of (row, block) is
//           ((row / 64 * (kp / 32) + block) * 16 + row % 16) * 4 + row % 64 / 16.
// A 256-element step of a row is one 128-byte cache line, the unit of the LDS-DMA fetches below.  A lane of the 16 x 16 x 128
// instruction holds 32 consecutive elements of one row = one scale block; with this scale order the 64 lanes of a wave read
// the scales of 64 rows x 4 blocks as one contiguous 256-byte load, and the instruction picks the byte of its 16 rows itself.
#include "tile_common.h"

#include <algorithm>
#include <type_traits>

namespace sgclip {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int MX_K = 256;   // elements per stage and the padding of a row

__host__ __device__ static inline long long mx_kp(int cols) { return ((long long)cols + MX_K - 1) / MX_K * MX_K; }

__device__ __forceinline__ float mx_scale_value(unsigned byte) {   // 2^(byte - 127); 255 = NaN
    return byte == 255u ? __builtin_nanf("") : __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}

// The block's scale byte from the largest absolute bit pattern of its elements (as f32): floor(log2 max) - 2 + 127, at least
// 0; a block that holds an infinity or a NaN gets 255.  The IEEE exponent field is floor(log2) + 127 for normal numbers, and
// subnormal ones fall below the smallest scale anyway.
__device__ __forceinline__ unsigned mx_scale_byte(unsigned amax_bits) {
    const unsigned ex = amax_bits >> 23;
    return ex == 255u ? 255u : (ex > 2u ? ex - 2u : 0u);
}

// Eight elements to eight codes (element 0 in the low nibble).  x * 2^(127 - byte) is exact wherever it decides a rounding (a
// product that underflows is far below the smallest code's border), so the conversion's round-to-nearest-even is the format's.
__device__ __forceinline__ unsigned mx_codes8(const float (&v)[8], unsigned byte) {
    const float inv = byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
    unsigned r = 0;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; j++) s[j] = byte == 255u ? 0.f : v[j] * inv;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, s[0], s[1], 1.0f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, s[2], s[3], 1.0f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, s[4], s[5], 1.0f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, s[6], s[7], 1.0f, 3);
    return r;
}

// Eight elements of a row as they lie in memory.
template <typename T>
struct MxRaw {
    T v[8] __attribute__((aligned(16)));
};

// 16 bytes at any address: global memory takes accesses of four dwords without alignment
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Eight elements from column k of a row (zeros behind cols).  VEC: aligned rows of whole groups of eight.  STREAM: the elements are
// not needed again (non-temporal).
template <typename T, bool VEC, bool STREAM = false>
__device__ __forceinline__ MxRaw<T> mx_load8(const T *__restrict__ row, int k, int cols) {
    MxRaw<T> x;
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    if constexpr (VEC) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) {
            const u32x4 *p = (const u32x4 *)(row + k) + j;
            ((u32x4 *)x.v)[j] = k < cols ? (STREAM ? __builtin_nontemporal_load(p) : *p) : (u32x4){0, 0, 0, 0};
        }
    } else if (k + 8 <= cols) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) {
            const u32x4_any *p = (const u32x4_any *)(row + k) + j;
            ((u32x4 *)x.v)[j] = STREAM ? __builtin_nontemporal_load(p) : *p;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x.v[j] = k + j < cols ? row[k + j] : (T)0.f;
    }
    return x;
}

template <typename T>
__device__ __forceinline__ void mx_floats(const MxRaw<T> &x, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = (float)x.v[j];
}

// ---------------------------------------------------------------------------
// Quantisation: a workgroup takes 64 rows x 256 columns, so that the tile's scales are 512 contiguous bytes; four lanes share
// a block of 32 and find its maximum with two exchanges.  ROWS = 1, for float inputs and for few rows: eight workgroups share the
// tile and write single scale bytes (bf16 64 x 1024 2.2 us, ROWS = 8 3.7; 4096 x 1024 3.6, 4.3; 16384 x 1024 10.3, 9.0; float
// 64 x 1024 2.2, 3.8; 32768 x 4096 104, 128).  Bound by HBM: 2 (bf16) or 4 (f32) bytes read and 17 / 32 written per element;
// 73856 x 1024 bf16 in 34 us (5.7 TB/s; 46 us with ordinary loads converted at once).
// ---------------------------------------------------------------------------
template <typename T, bool VEC, int ROWS>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *__restrict__ x, long long ldx, int rows, int cols,
                                                          unsigned char *__restrict__ codes, unsigned char *__restrict__ scales) {
    __shared__ unsigned char sc[512];
    const int tid = threadIdx.x;
    const long long kp = mx_kp(cols);
    const int kt = (int)(kp / MX_K);
    constexpr int PARTS = 64 / (8 * ROWS);          // workgroups that share 64 rows
    const int kb = blockIdx.x % kt, rg = blockIdx.x / kt, rb = rg / PARTS, part = rg % PARTS;
    const int c = tid & 31, k = kb * MX_K + c * 8;
    unsigned char *tile = scales + ((long long)rb * (kp / 32) + kb * 8) * 64;
    MxRaw<T> raw[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int row = rb * 64 + (part * ROWS + i) * 8 + (tid >> 5);
        raw[i] = mx_load8<T, VEC, true>(x + min(row, rows - 1) * ldx, k, cols);
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int lr = (part * ROWS + i) * 8 + (tid >> 5), row = rb * 64 + lr;
        float v[8];
        mx_floats(raw[i], v);
        unsigned am = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) am = max(am, __float_as_uint(v[j]) & 0x7fffffffu);
        am = max(am, (unsigned)__shfl_xor((int)am, 1, 64));
        am = max(am, (unsigned)__shfl_xor((int)am, 2, 64));
        const unsigned byte = row < rows ? mx_scale_byte(am) : 0u;     // behind the last row: read with the tile, so defined
        if (row < rows) *(unsigned *)(codes + row * (kp / 2) + (k >> 1)) = mx_codes8(v, byte);
        if ((c & 3) == 0) (ROWS == 8 ? sc : tile)[(c >> 2) * 64 + (lr & 15) * 4 + (lr >> 4)] = (unsigned char)byte;
    }
    if constexpr (ROWS == 8) {
        __syncthreads();
        if (tid < 128) ((unsigned *)tile)[tid] = ((const unsigned *)sc)[tid];
    }
}

// ---------------------------------------------------------------------------
// Back to bf16, which holds every value of the format exactly.  Plain: one thread per eight elements.  Transposed: 64 x 64
// tiles through LDS, out[k][row] with zeros in columns rows .. ldo - 1 (the reduction padding of the products that follow).
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mx_values8(unsigned r, float scale, float (&v)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(r, 1.0f, 3);
    v[0] = a[0] * scale; v[1] = a[1] * scale; v[2] = b[0] * scale; v[3] = b[1] * scale;
    v[4] = c[0] * scale; v[5] = c[1] * scale; v[6] = d[0] * scale; v[7] = d[1] * scale;
}

__device__ __forceinline__ float mx_row_scale(const unsigned char *scales, long long kp, long long row, int block) {
    return mx_scale_value(scales[(((row >> 6) * (kp / 32) + block) * 16 + (row & 15)) * 4 + ((row & 63) >> 4)]);
}

__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                            int rows, int cols, bf16_t *__restrict__ out, long long ldo) {
    const long long kp = mx_kp(cols);
    const int per = (cols + 7) / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)rows * per) return;
    const long long row = i / per;
    const int k = (int)(i - row * per) * 8;
    float v[8];
    mx_values8(*(const unsigned *)(codes + row * (kp / 2) + (k >> 1)), mx_row_scale(scales, kp, row, k >> 5), v);
    bf16_t *o = out + row * ldo + k;
    if (k + 8 <= cols) {
        bf16x8 b;
#pragma unroll
        for (int j = 0; j < 8; j++) b[j] = (bf16_t)v[j];
        *(u32x4_any *)o = __builtin_bit_cast(u32x4_any, b);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k + j < cols) o[j] = (bf16_t)v[j];
    }
}

__global__ __launch_bounds__(256) void mx_dequantize_t_kernel(const unsigned char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                              int rows, int cols, bf16_t *__restrict__ out, long long ldo) {
    __shared__ bf16_t tile[64][66];
    const long long kp = mx_kp(cols);
    const int kt = (cols + 63) / 64;
    const int r0 = blockIdx.x / kt * 64, k0 = blockIdx.x % kt * 64;
    const int tid = threadIdx.x;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const int lr = (tid >> 3) + 32 * p, k = k0 + (tid & 7) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.f;
        if (r0 + lr < rows)
            mx_values8(*(const unsigned *)(codes + (long long)(r0 + lr) * (kp / 2) + (k >> 1)), mx_row_scale(scales, kp, r0 + lr, k >> 5), v);
#pragma unroll
        for (int j = 0; j < 8; j++) tile[lr][(tid & 7) * 8 + j] = (bf16_t)v[j];
    }
    __syncthreads();
    const int c = tid & 63;
#pragma unroll
    for (int p = 0; p < 16; p++) {
        const int k = (tid >> 6) + 4 * p;
        if (k0 + k < cols && r0 + c < ldo) out[(long long)(k0 + k) * ldo + r0 + c] = tile[c][k];
    }
}

// ---------------------------------------------------------------------------
// The product.  The weights are the instruction's first operand: a lane's four results are four consecutive columns of one
// row of y.
// ---------------------------------------------------------------------------
struct MxGemm {
    const unsigned char *xc, *xs, *wc, *ws;   // codes and scales of x [M, K] and w [N, K]
    const float *bias, *resid;
    void *out;
    long long ldr, ldo, kp;
    int M, N;
    int wide;    // out, bias, resid allow four columns per aligned access; 2: and the rows of out begin on cache lines
};

// x sigmoid(1.702 x) on the hardware's exp2 and reciprocal (a few 2^-24, far below the bf16 rounding that follows; with an exact
// division the large product spends 150 us more in its epilogue)
__device__ __forceinline__ float mx_gelu(float x) { return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.4554669595930156f * x)); }

enum { MX_BF16 = 0, MX_GELU = 1, MX_RESID = 2 };

// four consecutive columns n .. n + 3 of row m
template <int EPI>
__device__ __forceinline__ void mx_store4(const MxGemm &g, f32x4 v, int m, int n) {
    if (m >= g.M || n >= g.N) return;
    if (g.wide) {   // N % 4 == 0: the four columns are all inside
        if (g.bias) {
            const float4 b = *(const float4 *)(g.bias + n);
            v[0] += b.x; v[1] += b.y; v[2] += b.z; v[3] += b.w;
        }
        if constexpr (EPI == MX_RESID) {
            const float4 r = *(const float4 *)(g.resid + m * g.ldr + n);
            *(float4 *)((float *)g.out + m * g.ldo + n) = make_float4(r.x + v[0], r.y + v[1], r.z + v[2], r.w + v[3]);
        } else {
            bf16x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = (bf16_t)(EPI == MX_GELU ? mx_gelu(v[j]) : v[j]);
            *(bf16x4 *)((bf16_t *)g.out + m * g.ldo + n) = o;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (n + j >= g.N) break;
        const float t = v[j] + (g.bias ? g.bias[n + j] : 0.f);
        if constexpr (EPI == MX_RESID) ((float *)g.out)[m * g.ldo + n + j] = g.resid[m * g.ldr + n + j] + t;
        else ((bf16_t *)g.out)[m * g.ldo + n + j] = (bf16_t)(EPI == MX_GELU ? mx_gelu(t) : t);
    }
}

template <int I, int N, typename F>
__device__ __forceinline__ void static_for(F &&f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

__device__ __forceinline__ i32x8 mx_operand(i32x4 v) { return (i32x8){v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// a's lanes of rows 8 .. 15 for b's of rows 0 .. 7 (of 16): afterwards a holds both halves of rows 0 .. 7, b those of rows 8 .. 15
__device__ __forceinline__ void mx_swap8(unsigned &a, unsigned &b) {
    const unsigned t = a;
    a = __builtin_amdgcn_update_dpp(a, b, 0x128, 0xf, 0xc, false);     // row_ror:8 into lanes 8 .. 15
    b = __builtin_amdgcn_update_dpp(b, t, 0x128, 0xf, 0x3, false);     // and into lanes 0 .. 7
}

// A wave's 16 I rows (m = mw ..) x 16 J columns (n = nw ..).  Straight from the
// registers (through LDS the round trips of a 256 x 256 tile cost 2 us): for bf16 two neighbouring 16-lane rows exchange halves, after
// which a lane holds eight consecutive columns, and an instruction writes 64 bytes of each of 16 rows.  bias: that of column nw, in
// LDS (STREAM: a whole tile's) or global memory.
// STREAM: non-temporal, for results larger than the caches, where ordinary stores wait for the evictions of the previous
// tile's lines (73856 x 1024 x 4096: 267 us, non-temporal 223).
// LONG: lanes eight apart exchange too, for 128 bytes of each of eight rows: where rows do not begin on cache lines, two accesses to
// one line cost most (5000 x 200 x 5004 48 us, so 25; on lines they do not, and longer accesses to fewer rows lose: a residual of
// 73856 x 4096 576 us, so 645).
// ANY: out, bias and residual at any element, any number of columns (without: g.wide).
template <int EPI, bool STREAM, bool LONG, bool ANY, int I, int J>
__device__ __forceinline__ void mx_epilogue(const MxGemm &g, const f32x4 (&acc)[I][J], const float *bias, int mw, int nw, int lane) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const int r = lane & 15, q = lane >> 4;
    auto store = [](u32x4 v, void *at) {
        if constexpr (STREAM) __builtin_nontemporal_store(v, (u32x4_any *)at);
        else *(u32x4_any *)at = v;
    };
    f32x4 b[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int n = j * 16 + q * 4;
        b[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (!g.bias) continue;
        if constexpr (STREAM) b[j] = *(const f32x4 *)(bias + n);
        else if (nw + n + (ANY ? 4 : 1) <= g.N) b[j] = *(const f32x4_any *)(bias + n);
        else if constexpr (ANY) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (nw + n + e < g.N) b[j][e] = bias[n + e];
        }
    }
    if constexpr (EPI == MX_RESID) {
#pragma unroll
        for (int i = 0; i < I; i++)
#pragma unroll
            for (int p = 0; p < J / 2; p++) {
                unsigned v[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int e = 0; e < 4; e++) v[h][e] = __float_as_uint(acc[i][2 * p + h][e] + b[2 * p + h][e]);
                if constexpr (LONG) {
#pragma unroll
                    for (int e = 0; e < 4; e++) mx_swap8(v[0][e], v[1][e]);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int m = mw + i * 16 + (LONG ? (r & 7) + 8 * h : r), n = nw + p * 32 + (LONG ? r >> 3 : h) * 16 + q * 4;
                    if (m >= g.M) continue;
                    const float *res = g.resid + m * g.ldr + n;
                    float *o = (float *)g.out + m * g.ldo + n;
                    if (n + (ANY ? 4 : 1) <= g.N) {
                        const f32x4 sum = *(const f32x4_any *)res + __builtin_bit_cast(f32x4, (u32x4){v[h][0], v[h][1], v[h][2], v[h][3]});
                        store(__builtin_bit_cast(u32x4, sum), o);
                    } else if constexpr (ANY) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n + e < g.N) o[e] = res[e] + __uint_as_float(v[h][e]);
                    }
                }
            }
    } else {
        auto columns = [&](unsigned(&v)[4], int i, int p) {
            bf16x4 o[2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float t = acc[i][2 * p + h][e] + b[2 * p + h][e];
                    o[h][e] = (bf16_t)(EPI == MX_GELU ? mx_gelu(t) : t);
                }
            const u32x2 w0 = __builtin_bit_cast(u32x2, o[0]), w1 = __builtin_bit_cast(u32x2, o[1]);
            const u32x2 lo = __builtin_amdgcn_permlane16_swap(w0[0], w1[0], false, false), hi = __builtin_amdgcn_permlane16_swap(w0[1], w1[1], false, false);
            v[0] = lo[0];
            v[1] = hi[0];
            v[2] = lo[1];
            v[3] = hi[1];
        };
        auto put = [&](const unsigned(&v)[4], int m, int n) {
            if (m >= g.M || n >= g.N) return;
            bf16_t *o = (bf16_t *)g.out + m * g.ldo + n;
            if (n + 8 <= g.N) store((u32x4){v[0], v[1], v[2], v[3]}, o);
            else if constexpr (!ANY) *(u32x2 *)o = (u32x2){v[0], v[1]};
            else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (n + e < g.N) ((unsigned short *)o)[e] = (unsigned short)(v[e >> 1] >> (e & 1) * 16);
            }
        };
        const int n = nw + (q & 1) * 16 + (q >> 1) * 8;
        if constexpr (LONG) {
            static_assert(J == 4, "64 columns per wave");
#pragma unroll
            for (int i = 0; i < I; i++) {
                unsigned v[2][4];
                columns(v[0], i, 0);
                columns(v[1], i, 1);
#pragma unroll
                for (int e = 0; e < 4; e++) mx_swap8(v[0][e], v[1][e]);
                put(v[0], mw + i * 16 + (r & 7), n + (r >> 3) * 32);
                put(v[1], mw + i * 16 + (r & 7) + 8, n + (r >> 3) * 32);
            }
        } else {      // all rows' first halves before the second ones: a line's two stores in a row cost more (228 us, so 217)
#pragma unroll
            for (int p = 0; p < J / 2; p++)
#pragma unroll
                for (int i = 0; i < I; i++) {
                    unsigned v[4];
                    columns(v, i, p);
                    put(v, mw + i * 16 + r, n + p * 32);
                }
        }
    }
}

// Tile of 2 WT x 2 WT, four waves of WT x WT (32 or 64) each; one 256-deep stage in flight behind the one computed, its scales
// with it in registers, one barrier per stage.  Bound by the latency of a stage's fetch: 9232 x 768 x 768 9.6 us (scales loaded
// where they are used, results four columns at a time: 12.6), 1540 x 768 x 768 4.8 us, added to a residual 6.0.
template <int EPI, int WT>
__global__ __launch_bounds__(256) void mx_gemm_kernel(MxGemm g) {
    constexpr int T = 2 * WT, NT = WT / 16, OP = T * 128;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, r = lane & 15, q = lane >> 4;
    const int tiles_n = (g.N + T - 1) / T, ntiles = gridDim.x;
    const int swz = xcd_remap(blockIdx.x, ntiles);
    const int m0 = swz / tiles_n * T, n0 = swz % tiles_n * T;
    const long long ld = g.kp / 2;
    const int ns = (int)(g.kp / MX_K);

    auto fetch = [&](int s, unsigned char *slot) {
#pragma unroll
        for (int p = wave; p < T / 8; p += 4) {
            const int row = p * 8 + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
            const unsigned char *sx = g.xc + min(m0 + row, g.M - 1) * ld + s * 128 + c * 16;
            const unsigned char *sw = g.wc + min(n0 + row, g.N - 1) * ld + s * 128 + c * 16;
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(sx), LDS_PTR(slot + p * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(GLOBAL_PTR(sw), LDS_PTR(slot + OP + p * 1024), 16, 0, 0);
        }
    };
    // scale rows of this wave: group of 64 rows (the last one where the tile hangs over), first 16-row byte inside it
    const int mrow = m0 + wm * WT, nrow = n0 + wn * WT;
    const unsigned char *xs = g.xs + (long long)min(mrow >> 6, (g.M - 1) >> 6) * (g.kp / 32) * 64;
    const unsigned char *wsc = g.ws + (long long)min(nrow >> 6, (g.N - 1) >> 6) * (g.kp / 32) * 64;
    const int xsh = (mrow & 63) / 16 * 8, wsh = (nrow & 63) / 16 * 8;

    f32x4 acc[NT][NT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    unsigned na[2], nb[2];
    auto fetch_scales = [&](int s) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            na[t] = *(const unsigned *)(wsc + ((s * 8 + t * 4 + q) * 16 + r) * 4);
            nb[t] = *(const unsigned *)(xs + ((s * 8 + t * 4 + q) * 16 + r) * 4);
        }
    };
    fetch_scales(0);
    fetch(0, lds);
    for (int s = 0; s < ns; s++) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const unsigned char *cur = lds + (s & 1) * 2 * OP;
        unsigned sa[2], sb[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            sa[t] = na[t] >> wsh;
            sb[t] = nb[t] >> xsh;
        }
        if (s + 1 < ns) {
            fetch_scales(s + 1);
            fetch(s + 1, lds + ((s + 1) & 1) * 2 * OP);
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            i32x4 fx[NT], fw[NT];
#pragma unroll
            for (int i = 0; i < NT; i++) {
                fx[i] = *(const i32x4 *)(cur + lds_off(wm * WT + i * 16 + r, t * 4 + q));
                fw[i] = *(const i32x4 *)(cur + OP + lds_off(wn * WT + i * 16 + r, t * 4 + q));
            }
            static_for<0, NT>([&](auto ic) {
                static_for<0, NT>([&](auto jc) {
                    constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fw[j]), mx_operand(fx[i]), acc[i][j], 4, 4, j,
                                                                                 (int)sa[t], i, (int)sb[t]);
                });
            });
        }
    }
    if (g.wide == 2) mx_epilogue<EPI, false, false, false>(g, acc, g.bias + nrow, mrow, nrow, lane);
    else mx_epilogue<EPI, false, NT == 4, true>(g, acc, g.bias + nrow, mrow, nrow, lane);
}

// ---------------------------------------------------------------------------
// Many tiles: persistent workgroups, 256 x 256 tiles, eight waves of 128 rows x 64 columns.
// The stages of a workgroup's tiles form one stream through two LDS slots; a stage is two 128-deep sub-steps whose fragments are
// double-buffered in registers, with one barrier between them: there every wave holds all of stage g, stage g + 1 has landed,
// and the DMA of stage g + 2 (of the next tile, if need be) starts into the slot just freed.  A tile's results leave from the registers
// while the next tile's operands arrive; the barrier after them waits for the fetches only (they are older than the stores, and the
// counter retires in order).
// 73856 x 1024 x 4096 in 209 us at the least, 226 on average of ten (with GELU 241 and 250).  Of 213 us 117 are the main loop alone (1.40 a
// stage, 1.08 at the matrix rate), 25 its fetches, the rest the results, 3.7 a tile (GELU 5.4), behind which the next tile's fetches
// wait.  K = 4096: 606 us at the least, 4.1 PFLOP/s, 646 on average.
// ---------------------------------------------------------------------------
constexpr int MXP_OP = 256 * 128, MXP_SLOT = 2 * MXP_OP + 4096, MXP_BIAS = 2 * MXP_SLOT, MXP_LDS = MXP_BIAS + 4096;
static_assert(MXP_LDS <= 160 * 1024, "LDS of a CU");

struct MxFrags {
    i32x4 x[8], w[4];
    unsigned sx[2], sw;
};

__device__ __forceinline__ void mxp_read(MxFrags &f, const unsigned char *x, const unsigned char *w, const unsigned char *sx,
                                         const unsigned char *sw) {
#pragma unroll
    for (int i = 0; i < 8; i++) f.x[i] = *(const i32x4 *)(x + i * 2048);
#pragma unroll
    for (int j = 0; j < 4; j++) f.w[j] = *(const i32x4 *)(w + j * 2048);
    f.sx[0] = *(const unsigned *)sx;
    f.sx[1] = *(const unsigned *)(sx + 512);
    f.sw = *(const unsigned *)sw;
}

__device__ __forceinline__ void mxp_multiply(f32x4 (&acc)[8][4], const MxFrags &f) {
    static_for<0, 8>([&](auto ic) {
        static_for<0, 4>([&](auto jc) {
            constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(f.w[j]), mx_operand(f.x[i]), acc[i][j], 4, 4, j, (int)f.sw,
                                                                         i % 4, (int)f.sx[i / 4]);
        });
    });
#pragma unroll
    for (int p = 0; p < 15; p++) {
        __builtin_amdgcn_sched_group_barrier(SG_DS_RD, 1, 0);
        __builtin_amdgcn_sched_group_barrier(SG_MFMA, 2, 0);
    }
}

// four bytes a lane (any alignment and number of columns) to 256 consecutive bytes of LDS
__device__ __forceinline__ void mxp_dma4(const unsigned char *base, int off, unsigned lds_addr) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 1\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds_addr) : "memory");
}

// vector memory stores of a wave for a whole tile, all younger than its last fetch
template <int EPI>
constexpr int mxp_stores() {
    return EPI == MX_RESID ? 32 : 16;
}

template <int EPI, bool LONG>
__global__ __launch_bounds__(512, 2) void mx_pipe_kernel(MxGemm g, int ntiles, int tiles_n) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, r = lane & 15, q = lane >> 4;
    const int ns = (int)(g.kp / MX_K);
    const long long ld = g.kp / 2, rbs = g.kp * 2;    // bytes of a row's codes, of 64 rows' scales
    const unsigned lds0 = (unsigned)(uintptr_t)LDS_PTR(lds);

    // the fetch stream: next stage to fetch, of which tile
    const int prow = wave * 8 + (lane >> 3);
    const unsigned chunk = (unsigned)(((lane & 7) ^ ((prow >> 1) & 7)) * 16), voff = (unsigned)(prow * ld) + chunk, step = (unsigned)(64 * ld);
    const unsigned sc_lane = (lane & 31) * 16, sc_voff = (unsigned)(((wave & 1) * 2 + (lane >> 5)) * rbs) + sc_lane;
    const unsigned char *xb, *wb, *sb;
    unsigned maxx, maxw, maxs;
    int ft = blockIdx.x, fs = 0, fbias = 0, fn0 = 0, fslot = 0;
    auto origin = [&](int t, int &m0, int &n0) {
        const int swz = xcd_remap(t, ntiles), tm = swz / tiles_n;
        m0 = tm * 256;
        n0 = (swz - tm * tiles_n) * 256;
    };
    auto aim = [&]() {
        int m0, n0;
        origin(ft, m0, n0);
        fn0 = n0;
        xb = g.xc + m0 * ld;
        wb = g.wc + n0 * ld;
        maxx = (unsigned)(min(g.M - 1 - m0, 255) * ld) + chunk;
        maxw = (unsigned)(min(g.N - 1 - n0, 255) * ld) + chunk;
        const int rb0 = (wave < 2 ? m0 : n0) >> 6, last = ((wave < 2 ? g.M : g.N) - 1) >> 6;
        sb = (wave < 2 ? g.xs : g.ws) + rb0 * rbs;
        maxs = (unsigned)(min(last - rb0, 3) * rbs) + sc_lane;
    };
    auto fetch = [&]() {
        if (ft >= ntiles) return;
        const unsigned slot = lds0 + fslot * MXP_SLOT;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            p64_dma16(xb, voff, p * step, maxx, slot + (wave + 8 * p) * 1024);
            p64_dma16(wb, voff, p * step, maxw, slot + MXP_OP + (wave + 8 * p) * 1024);
        }
        if (wave < 4) p64_dma16(sb, sc_voff, 0, maxs, slot + 2 * MXP_OP + wave * 1024);
        else if (wave == 4 && fs == 0 && g.bias) {
            if constexpr (LONG) {
#pragma unroll
                for (int p = 0; p < 4; p++)
                    mxp_dma4((const unsigned char *)(g.bias + fn0), min(p * 64 + lane, g.N - 1 - fn0) * 4, lds0 + MXP_BIAS + fbias * 1024 + p * 256);
            } else p64_dma16((const unsigned char *)(g.bias + fn0), lane * 16, 0, (unsigned)(min(g.N - fn0, 256) * 4 - 16), lds0 + MXP_BIAS + fbias * 1024);
        }
        xb += 128;
        wb += 128;
        sb += 512;
        fslot ^= 1;
        if (++fs == ns) {
            fs = 0;
            fbias = (fbias + 1) & 3;
            ft += gridDim.x;
            if (ft < ntiles) aim();
        }
    };
    const int x0 = lds_off(wm * 128 + r, q), x1 = lds_off(wm * 128 + r, 4 + q);
    const int w0 = MXP_OP + lds_off(wn * 64 + r, q), w1 = MXP_OP + lds_off(wn * 64 + r, 4 + q);
    const int sx0 = 2 * MXP_OP + wm * 1024 + q * 64 + r * 4, sw0 = 2 * MXP_OP + 2048 + wn * 512 + q * 64 + r * 4;   // sub-step 1: + 256

    aim();
    fetch();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    fetch();
    f32x4 acc[8][4];
    MxFrags f0, f1;
    mxp_read(f0, lds + x0, lds + w0, lds + sx0, lds + sw0);
    int slot = 0, bias = 0;   // bias: of four, since the fetch of a tile two further on may run before this tile's epilogue
    bool stored = false;      // the last tile's stores were all issued and may still be on their way
    for (int t = blockIdx.x; t < ntiles; t += gridDim.x) {
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < ns; s++) {
            const unsigned char *cur = lds + slot * MXP_SLOT, *nxt = lds + (slot ^ 1) * MXP_SLOT;
            mxp_read(f1, cur + x1, cur + w1, cur + sx0 + 256, cur + sw0 + 256);
            mxp_multiply(acc, f0);
            if (s == 0 && stored) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(mxp_stores<EPI>()) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fetch();
            // behind the workgroup's last stage this reads what the slot held before: not used
            mxp_read(f0, nxt + x0, nxt + w0, nxt + sx0, nxt + sw0);
            mxp_multiply(acc, f1);
            slot ^= 1;
        }
        int m0, n0;
        origin(t, m0, n0);
        mx_epilogue<EPI, true, LONG, LONG>(g, acc, (const float *)(lds + MXP_BIAS + bias * 1024 + wn * 256), m0 + wm * 128, n0 + wn * 64, lane);
        bias = (bias + 1) & 3;
        stored = m0 + 256 <= g.M && n0 + 256 <= g.N;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Up to 16 rows of x, quantised on the way in: a workgroup takes 16 columns of y, its waves (one per 128 of K, at most 16)
// 128-deep slices of K in turn, and joins their sums through LDS.  A lane holds one block of 32 of one row, so the block's maximum needs no exchange.
// Bound by the weights' bytes (and, below about a megabyte of them, by the launch).
template <typename T, bool VEC, int EPI>
__global__ __launch_bounds__(1024) void mx_few_rows_kernel(const T *__restrict__ x, long long ldx, int K, MxGemm g) {
    __shared__ f32x4 part[16][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6, r = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const long long ld = g.kp / 2;
    const int nrow = min(n0 + r, g.N - 1);
    const unsigned char *wc = g.wc + nrow * ld;
    f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int steps = (K + 127) / 128;
    for (int s = wave; s < steps; s += waves) {
        const int block = s * 4 + q;
        const i32x4 fw = *(const i32x4 *)(wc + block * 16);
        const unsigned sw = g.ws[(((long long)(nrow >> 6) * (g.kp / 32) + block) * 16 + (nrow & 15)) * 4 + ((nrow & 63) >> 4)];
        i32x4 fx = (i32x4){0, 0, 0, 0};
        unsigned sx = 0;
        if (r < g.M) {
            float v[4][8];
            unsigned am = 0;
#pragma unroll
            for (int p = 0; p < 4; p++) {
                mx_floats(mx_load8<T, VEC>(x + r * ldx, block * 32 + p * 8, K), v[p]);
#pragma unroll
                for (int j = 0; j < 8; j++) am = max(am, __float_as_uint(v[p][j]) & 0x7fffffffu);
            }
            sx = mx_scale_byte(am);
#pragma unroll
            for (int p = 0; p < 4; p++) fx[p] = (int)mx_codes8(v[p], sx);
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(fw), mx_operand(fx), acc, 4, 4, 0, (int)sw, 0, (int)sx);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        for (int w = 1; w < waves; w++) acc += part[w][lane];
        mx_store4<EPI>(g, acc, r, n0 + q * 4);
    }
}

// ---------------------------------------------------------------------------
// Column sums without atomics (bias gradients): every workgroup sums a strip of rows of 512 columns (a lane eight of them, its
// waves every WAVES-th row), a second launch adds the strips in a fixed order; few rows are one strip of 16 waves, and no second
// launch.  Bound by HBM: 36928 x 4096 bf16 in 52 us (5.8 TB/s), the second launch 5 us.
// ---------------------------------------------------------------------------
constexpr int CS_COLS = 512, CS_STRIPS = 256, CS_ROWS = 32, CS_FEW = 512;

static inline int cs_strips(int M) { return M <= CS_FEW ? 1 : std::min(CS_STRIPS, (M + CS_ROWS - 1) / CS_ROWS); }

template <typename T, bool VEC, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_colsum_strip_kernel(const T *__restrict__ in, long long ld, int M, int N, float *__restrict__ parts) {
    __shared__ float sums[WAVES][CS_COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * CS_COLS + lane * 8;
    const long long per = ((long long)M + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * per, hi = min(lo + per, (long long)M);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < N) {
#pragma unroll 4
        for (long long m = lo + wave; m < hi; m += WAVES) {
            float v[8];
            mx_floats(mx_load8<T, VEC>(in + m * ld, n, N), v);
#pragma unroll
            for (int j = 0; j < 8; j++) s[j] += v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) sums[wave][lane * 8 + j] = s[j];
    __syncthreads();
    for (int c = threadIdx.x; c < CS_COLS; c += 64 * WAVES)
        if (blockIdx.x * CS_COLS + c < N) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w += 4) t += (sums[w][c] + sums[w + 1][c]) + (sums[w + 2][c] + sums[w + 3][c]);
            parts[(long long)blockIdx.y * N + blockIdx.x * CS_COLS + c] = t;
        }
}

__global__ __launch_bounds__(256) void mx_colsum_join_kernel(const float *__restrict__ parts, int strips, int N, float *__restrict__ out) {
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int i = wave; i < strips; i += 4) s += parts[(long long)i * N + n];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && n < N) out[n] = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
}

// ---------------------------------------------------------------------------
// The layer's gradients run on the bf16 products; these lay their operands out.
// ---------------------------------------------------------------------------
// [M, N] to bf16 [M, ldo] with zeros behind N; ldo a multiple of 8
template <typename T>
__global__ __launch_bounds__(256) void mx_pad_kernel(const T *__restrict__ in, long long ld, int M, int N, bf16_t *__restrict__ out, int ldo) {
    const int per = ldo / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)M * per) return;
    const long long row = i / per;
    const int k = (int)(i - row * per) * 8;
    float v[8];
    mx_floats(mx_load8<T, false>(in + row * ld, k, N), v);
    bf16x8 b;
#pragma unroll
    for (int j = 0; j < 8; j++) b[j] = (bf16_t)v[j];
    *(bf16x8 *)(out + i * 8) = b;
}

// zeros: where the weight gradient is summed, and the bias that the data gradient's product asks for
template <typename T>
__global__ __launch_bounds__(256) void mx_zero_kernel(T *__restrict__ a, long long na, T *__restrict__ b, long long nb) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < na + nb; i += (long long)gridDim.x * 256) {
        if (i < na) a[i] = (T)0.f;
        else b[i - na] = (T)0.f;
    }
}

__global__ __launch_bounds__(256) void mx_crop_kernel(const float *__restrict__ in, int ldi, int rows, int cols, float *__restrict__ out) {
    const long long n = (long long)rows * cols;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / cols;
        out[i] = in[row * ldi + (i - row * cols)];
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static bool mx_shape_ok(const char *who, int rows, int cols) {
    if (rows < 0 || rows > (1 << 30) || cols <= 0 || cols > (1 << 24)) {
        set_error("%s: bad shape rows=%d cols=%d", who, rows, cols);
        return false;
    }
    return true;
}

// a launch counts its threads in 32 bits
static bool mx_grid_ok(const char *who, long long blocks, int threads) {
    if (blocks * threads > 0xffffffffLL) {
        set_error("%s: %lld workgroups of %d threads are more than one launch holds", who, blocks, threads);
        return false;
    }
    return true;
}

static bool mx_storage_ok(const char *who, const void *codes, const void *scales) {
    if (!codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 15)) {
        set_error("%s: codes and scales must be 16-byte aligned device pointers", who);
        return false;
    }
    return true;
}

template <typename T>
static int mx_launch_quantize(const T *x, long long ldx, int rows, int cols, unsigned char *codes, unsigned char *scales, hipStream_t stream) {
    const bool vec = cols % 8 == 0 && ldx * sizeof(T) % 16 == 0 && ((uintptr_t)x & 15) == 0;
    const long long blocks = ((long long)rows + 63) / 64 * (mx_kp(cols) / MX_K);
    const bool spread = sizeof(T) == 4 || blocks < 2 * device_cus();
    if (!mx_grid_ok("sgclip_mxfp4_quantize", spread ? blocks * 8 : blocks, 256)) return SGCLIP_EINVAL;
    if (spread) {
        const dim3 grid((unsigned)(blocks * 8));
        if (vec) mx_quantize_kernel<T, true, 1><<<grid, 256, 0, stream>>>(x, ldx, rows, cols, codes, scales);
        else mx_quantize_kernel<T, false, 1><<<grid, 256, 0, stream>>>(x, ldx, rows, cols, codes, scales);
    } else if constexpr (sizeof(T) == 2) {
        const dim3 grid((unsigned)blocks);
        if (vec) mx_quantize_kernel<T, true, 8><<<grid, 256, 0, stream>>>(x, ldx, rows, cols, codes, scales);
        else mx_quantize_kernel<T, false, 8><<<grid, 256, 0, stream>>>(x, ldx, rows, cols, codes, scales);
    }
    return launch_check("sgclip_mxfp4_quantize");
}

template <int EPI>
static int mx_launch_gemm(const MxGemm &g, hipStream_t stream) {
    const long long cus = device_cus();
    const long long huge = (((long long)g.M + 255) / 256) * (((long long)g.N + 255) / 256);
    const long long big = (((long long)g.M + 127) / 128) * (((long long)g.N + 127) / 128);
    // 256 x 256 tiles where their rounds over the chip cost less: one takes as long as 2.7 of 128 x 128 tiles (K = 1024: 12.8 us for
    // one or fewer, 23 - 24 for two; 128 x 128 tiles 10.4 us for 440, 13.9 for 584, 20.7 for 1160, 25 - 29 for 1744; K = 4096: 30 and 60;
    // 23.4, 32.8, 50.9)
    if ((big + cus - 1) / cus * 10 >= (huge + cus - 1) / cus * 27 && huge < (1 << 24)) {
        const auto kernel = g.wide == 2 ? mx_pipe_kernel<EPI, false> : mx_pipe_kernel<EPI, true>;
        if (!lds_attr((const void *)kernel, MXP_LDS)) return SGCLIP_ELAUNCH;
        kernel<<<dim3((unsigned)std::min(cus, huge)), 512, MXP_LDS, stream>>>(g, (int)huge, (g.N + 255) / 256);
        return SGCLIP_OK;
    }
    // 128 x 128 tiles where they fill the chip, 64 x 64 below that (K = 1024: 6.3 against 4.6 us at 80 of the larger, 7.6 both at 224,
    // 10.4 against 11.4 at 440)
    if (!mx_grid_ok("sgclip_mxfp4_gemm", big, 256)) return SGCLIP_EINVAL;
    if (big >= cus) {
        if (!lds_attr((const void *)mx_gemm_kernel<EPI, 64>, 4 * 128 * 128)) return SGCLIP_ELAUNCH;
        mx_gemm_kernel<EPI, 64><<<dim3((unsigned)big), 256, 4 * 128 * 128, stream>>>(g);
    } else {
        const long long small = (((long long)g.M + 63) / 64) * (((long long)g.N + 63) / 64);
        mx_gemm_kernel<EPI, 32><<<dim3((unsigned)small), 256, 4 * 64 * 128, stream>>>(g);
    }
    return SGCLIP_OK;
}

template <typename T, int EPI>
static void mx_launch_few(const T *x, long long ldx, int K, const MxGemm &g, hipStream_t stream) {
    const bool vec = K % 8 == 0 && ldx * sizeof(T) % 16 == 0 && ((uintptr_t)x & 15) == 0;
    const dim3 grid((unsigned)((g.N + 15) / 16)), block(64 * std::min(16, (K + 127) / 128));
    if (vec) mx_few_rows_kernel<T, true, EPI><<<grid, block, 0, stream>>>(x, ldx, K, g);
    else mx_few_rows_kernel<T, false, EPI><<<grid, block, 0, stream>>>(x, ldx, K, g);
}

template <typename T>
static void mx_launch_colsum(const T *in, long long ld, int M, int N, int strips, float *parts, float *out, hipStream_t st) {
    const bool vec = N % 8 == 0 && ld * sizeof(T) % 16 == 0 && ((uintptr_t)in & 15) == 0;
    const dim3 grid((unsigned)ceil_div(N, CS_COLS), (unsigned)strips);
    if (strips == 1) {
        if (vec) mx_colsum_strip_kernel<T, true, 16><<<grid, 1024, 0, st>>>(in, ld, M, N, out);
        else mx_colsum_strip_kernel<T, false, 16><<<grid, 1024, 0, st>>>(in, ld, M, N, out);
        return;
    }
    if (vec) mx_colsum_strip_kernel<T, true, 4><<<grid, 256, 0, st>>>(in, ld, M, N, parts);
    else mx_colsum_strip_kernel<T, false, 4><<<grid, 256, 0, st>>>(in, ld, M, N, parts);
    mx_colsum_join_kernel<<<dim3((unsigned)((N + 63) / 64)), 256, 0, st>>>(parts, strips, N, out);
}

static inline unsigned mx_grid(long long n) { return (unsigned)std::min((n + 255) / 256, 4096LL); }     // for loops over the grid

template <typename T>
static void mx_zero(T *a, long long na, T *b, long long nb, hipStream_t st) {
    if (na + nb > 0) mx_zero_kernel<<<dim3(mx_grid(na + nb)), 256, 0, st>>>(a, na, b, nb);
}

// workspace of the layer's gradients: zeros f32 [K]; dy bf16 [M][n64], if it has to be laid out; w^T bf16 [K][n64]; x bf16 [M][k8];
// dw f32 [n8][k8], if it has to be cropped; column sums
constexpr int MX_BWD_LD = 1 << 22;     // the products count 256 rows' bytes in 32 bits

struct MxBwdPlan {
    int n8, n64, k8;
    bool pad, crop;
    size_t zeros, dy, wt, x, dw, parts, total;
};

static MxBwdPlan mx_bwd_plan(const void *dy, int dtype, long long lddy, int M, int N, int K) {
    MxBwdPlan p;
    p.n8 = (N + 7) / 8 * 8;
    p.n64 = (N + 63) / 64 * 64;
    p.k8 = (K + 7) / 8 * 8;
    p.pad = dtype == SGCLIP_DTYPE_F32 || N % 64 != 0 || lddy % 8 != 0 || lddy > MX_BWD_LD || ((uintptr_t)dy & 15);
    p.crop = p.n8 != N || p.k8 != K;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align_up(bytes, 256);
        return here;
    };
    p.zeros = take((size_t)K * 4);
    p.dy = take(p.pad ? (size_t)M * p.n64 * 2 : 0);
    p.wt = take((size_t)K * p.n64 * 2);
    p.x = take((size_t)M * p.k8 * 2);
    p.dw = take(p.crop ? (size_t)p.n8 * p.k8 * 4 : 0);
    p.parts = take(sgclip_column_sums_workspace_bytes(M, N));
    p.total = at;
    return p;
}

static int mx_epilogue(const char *who, MxGemm &g, int epilogue, const float *bias, const float *aux, int64_t ldaux, void *out, int64_t ldo,
                       int &epi) {
    switch (epilogue) {
        case SGCLIP_EPI_BIAS_BF16: epi = MX_BF16; break;
        case SGCLIP_EPI_BIAS_GELU_BF16: epi = MX_GELU; break;
        case SGCLIP_EPI_BIAS_RESID_F32: epi = MX_RESID; break;
        default: set_error("%s: epilogue %d is not one of the 4-bit product's", who, epilogue); return SGCLIP_EINVAL;
    }
    if (!out || ldo < g.N || (epi == MX_RESID && (!aux || ldaux < g.N))) {
        set_error("%s: output / residual missing or its row stride below N=%d", who, g.N);
        return SGCLIP_EINVAL;
    }
    g.bias = bias;
    g.resid = epi == MX_RESID ? aux : nullptr;
    g.ldr = ldaux;
    g.out = out;
    g.ldo = ldo;
    g.wide = g.N % 4 == 0 && ldo % 4 == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)bias & 15) == 0 &&
             (epi != MX_RESID || (ldaux % 4 == 0 && ((uintptr_t)aux & 15) == 0));
    if (g.wide && ldo * (epi == MX_RESID ? 4 : 2) % 128 == 0 && ((uintptr_t)out & 127) == 0) g.wide = 2;
    return SGCLIP_OK;
}

}  // namespace sgclip

using namespace sgclip;

extern "C" {

size_t sgclip_mxfp4_codes_bytes(int rows, int cols) { return rows <= 0 || cols <= 0 ? 0 : (size_t)rows * (size_t)(mx_kp(cols) / 2); }

size_t sgclip_mxfp4_scales_bytes(int rows, int cols) {
    return rows <= 0 || cols <= 0 ? 0 : ((size_t)rows + 63) / 64 * 64 * (size_t)(mx_kp(cols) / 32);
}

int sgclip_mxfp4_quantize(const void *x_dev, int x_dtype, int64_t ldx, int rows, int cols, void *codes_dev, void *scales_dev, void *stream) {
    if (!mx_shape_ok("sgclip_mxfp4_quantize", rows, cols)) return SGCLIP_EINVAL;
    if (rows == 0) return SGCLIP_OK;
    if (!x_dev || ldx < cols || (x_dtype != SGCLIP_DTYPE_F32 && x_dtype != SGCLIP_DTYPE_BF16)) {
        set_error("sgclip_mxfp4_quantize: bad x (dtype %d, row stride %lld, cols %d)", x_dtype, (long long)ldx, cols);
        return SGCLIP_EINVAL;
    }
    if (!mx_storage_ok("sgclip_mxfp4_quantize", codes_dev, scales_dev)) return SGCLIP_EINVAL;
    unsigned char *c = (unsigned char *)codes_dev, *s = (unsigned char *)scales_dev;
    return x_dtype == SGCLIP_DTYPE_F32 ? mx_launch_quantize((const float *)x_dev, ldx, rows, cols, c, s, (hipStream_t)stream)
                                       : mx_launch_quantize((const bf16_t *)x_dev, ldx, rows, cols, c, s, (hipStream_t)stream);
}

int sgclip_mxfp4_dequantize(const void *codes_dev, const void *scales_dev, int rows, int cols, int transpose, void *out_dev, int64_t ldo,
                            void *stream) {
    if (!mx_shape_ok("sgclip_mxfp4_dequantize", rows, cols)) return SGCLIP_EINVAL;
    if (rows == 0) return SGCLIP_OK;
    if (!out_dev || ldo < (transpose ? rows : cols) || (transpose && ldo > ((int64_t)rows + 63) / 64 * 64)) {
        set_error("sgclip_mxfp4_dequantize: bad output row stride %lld for rows=%d cols=%d transpose=%d", (long long)ldo, rows, cols, transpose);
        return SGCLIP_EINVAL;
    }
    if (!mx_storage_ok("sgclip_mxfp4_dequantize", codes_dev, scales_dev)) return SGCLIP_EINVAL;
    const unsigned char *c = (const unsigned char *)codes_dev, *s = (const unsigned char *)scales_dev;
    if (transpose) {
        const long long tiles = (((long long)rows + 63) / 64) * ((cols + 63) / 64);
        if (!mx_grid_ok("sgclip_mxfp4_dequantize", tiles, 256)) return SGCLIP_EINVAL;
        mx_dequantize_t_kernel<<<dim3((unsigned)tiles), 256, 0, (hipStream_t)stream>>>(c, s, rows, cols, (bf16_t *)out_dev, ldo);
    } else {
        const long long n = (long long)rows * ((cols + 7) / 8);
        if (!mx_grid_ok("sgclip_mxfp4_dequantize", (n + 255) / 256, 256)) return SGCLIP_EINVAL;
        mx_dequantize_kernel<<<dim3((unsigned)((n + 255) / 256)), 256, 0, (hipStream_t)stream>>>(c, s, rows, cols, (bf16_t *)out_dev, ldo);
    }
    return launch_check("sgclip_mxfp4_dequantize");
}

int sgclip_mxfp4_gemm(const void *x_codes_dev, const void *x_scales_dev, const void *w_codes_dev, const void *w_scales_dev, int M, int N,
                      int K, int epilogue, const float *bias_dev, const float *aux_dev, int64_t ldaux, void *out_dev, int64_t ldo,
                      void *stream) {
    if (!mx_shape_ok("sgclip_mxfp4_gemm", M, K) || !mx_shape_ok("sgclip_mxfp4_gemm", N, K)) return SGCLIP_EINVAL;
    if (M == 0 || N == 0) return SGCLIP_OK;
    if (!mx_storage_ok("sgclip_mxfp4_gemm", x_codes_dev, x_scales_dev) || !mx_storage_ok("sgclip_mxfp4_gemm", w_codes_dev, w_scales_dev))
        return SGCLIP_EINVAL;
    MxGemm g{};
    g.xc = (const unsigned char *)x_codes_dev;
    g.xs = (const unsigned char *)x_scales_dev;
    g.wc = (const unsigned char *)w_codes_dev;
    g.ws = (const unsigned char *)w_scales_dev;
    g.M = M;
    g.N = N;
    g.kp = mx_kp(K);
    int epi;
    int rc = mx_epilogue("sgclip_mxfp4_gemm", g, epilogue, bias_dev, aux_dev, ldaux, out_dev, ldo, epi);
    if (rc != SGCLIP_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    rc = epi == MX_BF16 ? mx_launch_gemm<MX_BF16>(g, st) : epi == MX_GELU ? mx_launch_gemm<MX_GELU>(g, st) : mx_launch_gemm<MX_RESID>(g, st);
    return rc != SGCLIP_OK ? rc : launch_check("sgclip_mxfp4_gemm");
}

size_t sgclip_mxfp4_linear_workspace_bytes(int M, int K) {
    if (M <= SGCLIP_MXFP4_FEW_ROWS) return 0;
    return align_up(sgclip_mxfp4_codes_bytes(M, K), 256) + sgclip_mxfp4_scales_bytes(M, K);
}

int sgclip_mxfp4_linear(const void *x_dev, int x_dtype, int64_t ldx, const void *w_codes_dev, const void *w_scales_dev, int M, int N, int K,
                        int epilogue, const float *bias_dev, const float *aux_dev, int64_t ldaux, void *out_dev, int64_t ldo,
                        void *workspace_dev, size_t workspace_bytes, void *stream) {
    if (!mx_shape_ok("sgclip_mxfp4_linear", M, K) || !mx_shape_ok("sgclip_mxfp4_linear", N, K)) return SGCLIP_EINVAL;
    if (M == 0 || N == 0) return SGCLIP_OK;
    if (M > SGCLIP_MXFP4_FEW_ROWS) {
        if (workspace_bytes < sgclip_mxfp4_linear_workspace_bytes(M, K) || !workspace_dev) {
            set_error("sgclip_mxfp4_linear: workspace of %zu bytes, %zu needed", workspace_bytes, sgclip_mxfp4_linear_workspace_bytes(M, K));
            return SGCLIP_ENOSPC;
        }
        unsigned char *codes = (unsigned char *)workspace_dev, *scales = codes + align_up(sgclip_mxfp4_codes_bytes(M, K), 256);
        const int rc = sgclip_mxfp4_quantize(x_dev, x_dtype, ldx, M, K, codes, scales, stream);
        if (rc != SGCLIP_OK) return rc;
        return sgclip_mxfp4_gemm(codes, scales, w_codes_dev, w_scales_dev, M, N, K, epilogue, bias_dev, aux_dev, ldaux, out_dev, ldo, stream);
    }
    if (!x_dev || ldx < K || (x_dtype != SGCLIP_DTYPE_F32 && x_dtype != SGCLIP_DTYPE_BF16)) {
        set_error("sgclip_mxfp4_linear: bad x (dtype %d, row stride %lld, K %d)", x_dtype, (long long)ldx, K);
        return SGCLIP_EINVAL;
    }
    if (!mx_storage_ok("sgclip_mxfp4_linear", w_codes_dev, w_scales_dev)) return SGCLIP_EINVAL;
    MxGemm g{};
    g.wc = (const unsigned char *)w_codes_dev;
    g.ws = (const unsigned char *)w_scales_dev;
    g.M = M;
    g.N = N;
    g.kp = mx_kp(K);
    int epi;
    const int rc = mx_epilogue("sgclip_mxfp4_linear", g, epilogue, bias_dev, aux_dev, ldaux, out_dev, ldo, epi);
    if (rc != SGCLIP_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    const bool f32 = x_dtype == SGCLIP_DTYPE_F32;
    const float *xf = (const float *)x_dev;
    const bf16_t *xb = (const bf16_t *)x_dev;
    if (epi == MX_BF16) f32 ? mx_launch_few<float, MX_BF16>(xf, ldx, K, g, st) : mx_launch_few<bf16_t, MX_BF16>(xb, ldx, K, g, st);
    else if (epi == MX_GELU) f32 ? mx_launch_few<float, MX_GELU>(xf, ldx, K, g, st) : mx_launch_few<bf16_t, MX_GELU>(xb, ldx, K, g, st);
    else f32 ? mx_launch_few<float, MX_RESID>(xf, ldx, K, g, st) : mx_launch_few<bf16_t, MX_RESID>(xb, ldx, K, g, st);
    return launch_check("sgclip_mxfp4_linear");
}

size_t sgclip_column_sums_workspace_bytes(int M, int N) {
    return M <= CS_FEW || N <= 0 ? 0 : (size_t)cs_strips(M) * (size_t)N * sizeof(float);
}

int sgclip_column_sums(const void *in_dev, int in_dtype, int64_t ld, int M, int N, float *out_dev, void *workspace_dev, size_t workspace_bytes,
                       void *stream) {
    if (N == 0) return SGCLIP_OK;
    if (M < 0 || N < 0 || (M > 0 && !in_dev) || !out_dev || ld < N || (in_dtype != SGCLIP_DTYPE_F32 && in_dtype != SGCLIP_DTYPE_BF16)) {
        set_error("sgclip_column_sums: bad arguments M=%d N=%d ld=%lld dtype=%d", M, N, (long long)ld, in_dtype);
        return SGCLIP_EINVAL;
    }
    const int strips = cs_strips(M);
    if (strips > 1 && (!workspace_dev || workspace_bytes < sgclip_column_sums_workspace_bytes(M, N))) {
        set_error("sgclip_column_sums: workspace of %zu bytes, %zu needed", workspace_dev ? workspace_bytes : (size_t)0,
                  sgclip_column_sums_workspace_bytes(M, N));
        return SGCLIP_ENOSPC;
    }
    const hipStream_t st = (hipStream_t)stream;
    if (in_dtype == SGCLIP_DTYPE_F32) mx_launch_colsum((const float *)in_dev, ld, M, N, strips, (float *)workspace_dev, out_dev, st);
    else mx_launch_colsum((const bf16_t *)in_dev, ld, M, N, strips, (float *)workspace_dev, out_dev, st);
    return launch_check("sgclip_column_sums");
}

size_t sgclip_mxfp4_linear_bwd_workspace_bytes(const void *dy_dev, int dy_dtype, int64_t lddy, int M, int N, int K) {
    return M <= 0 || N <= 0 || K <= 0 ? 0 : mx_bwd_plan(dy_dev, dy_dtype, lddy, M, N, K).total;
}

int sgclip_mxfp4_linear_bwd(const void *dy_dev, int dy_dtype, int64_t lddy, const void *x_codes_dev, const void *x_scales_dev,
                            const void *w_codes_dev, const void *w_scales_dev, int M, int N, int K, void *dx_dev, int dx_dtype, float *dw_dev,
                            float *db_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
    const char *who = "sgclip_mxfp4_linear_bwd";
    if (!mx_shape_ok(who, M, K) || !mx_shape_ok(who, N, K)) return SGCLIP_EINVAL;
    if (N > MX_BWD_LD) {
        set_error("%s: N=%d is more than %d", who, N, MX_BWD_LD);
        return SGCLIP_EINVAL;
    }
    const hipStream_t st = (hipStream_t)stream;
    if (M == 0 || N == 0) {
        if (dx_dev && dx_dtype == SGCLIP_DTYPE_F32) mx_zero((float *)dx_dev, (long long)M * K, (float *)nullptr, 0, st);
        if (dx_dev && dx_dtype == SGCLIP_DTYPE_BF16) mx_zero((bf16_t *)dx_dev, (long long)M * K, (bf16_t *)nullptr, 0, st);
        mx_zero(dw_dev, dw_dev ? (long long)N * K : 0, db_dev, db_dev ? N : 0, st);
        return launch_check(who);
    }
    if (!dy_dev || lddy < N || (dy_dtype != SGCLIP_DTYPE_F32 && dy_dtype != SGCLIP_DTYPE_BF16) ||
        (dx_dev && dx_dtype != SGCLIP_DTYPE_F32 && dx_dtype != SGCLIP_DTYPE_BF16)) {
        set_error("%s: bad dy (dtype %d, row stride %lld, N %d) or dx dtype %d", who, dy_dtype, (long long)lddy, N, dx_dtype);
        return SGCLIP_EINVAL;
    }
    if (!mx_storage_ok(who, x_codes_dev, x_scales_dev) || !mx_storage_ok(who, w_codes_dev, w_scales_dev)) return SGCLIP_EINVAL;
    const MxBwdPlan p = mx_bwd_plan(dy_dev, dy_dtype, lddy, M, N, K);
    if (!workspace_dev || workspace_bytes < p.total || ((uintptr_t)workspace_dev & 15)) {
        set_error("%s: workspace of %zu bytes, %zu needed (16-byte aligned)", who, workspace_dev ? workspace_bytes : (size_t)0, p.total);
        return SGCLIP_ENOSPC;
    }
    unsigned char *ws = (unsigned char *)workspace_dev;
    float *zeros = (float *)(ws + p.zeros), *sum = p.crop ? (float *)(ws + p.dw) : dw_dev;
    int rc = SGCLIP_OK;
    if (db_dev) rc = sgclip_column_sums(dy_dev, dy_dtype, lddy, M, N, db_dev, ws + p.parts, p.total - p.parts, stream);
    if (rc != SGCLIP_OK || (!dx_dev && !dw_dev)) return rc;
    mx_zero(sum, dw_dev ? (long long)p.n8 * p.k8 : 0, zeros, dx_dev ? K : 0, st);
    // dy as the products take it: bf16, aligned rows, whole stages of columns
    const void *dy = dy_dev;
    long long ld = lddy;
    if (p.pad) {
        const long long blocks = ((long long)M * (p.n64 / 8) + 255) / 256;
        if (!mx_grid_ok(who, blocks, 256)) return SGCLIP_EINVAL;
        bf16_t *out = (bf16_t *)(ws + p.dy);
        if (dy_dtype == SGCLIP_DTYPE_F32) mx_pad_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>((const float *)dy_dev, lddy, M, N, out, p.n64);
        else mx_pad_kernel<<<dim3((unsigned)blocks), 256, 0, st>>>((const bf16_t *)dy_dev, lddy, M, N, out, p.n64);
        dy = out;
        ld = p.n64;
    }
    if (dx_dev) {
        rc = sgclip_mxfp4_dequantize(w_codes_dev, w_scales_dev, N, K, 1, ws + p.wt, p.n64, stream);
        if (rc == SGCLIP_OK)
            rc = sgclip_gemm_bf16(dy, (int)ld, ws + p.wt, p.n64, dx_dev, K, M, K, p.n64,
                                  dx_dtype == SGCLIP_DTYPE_F32 ? SGCLIP_EPI_F32 : SGCLIP_EPI_BIAS_BF16, zeros, nullptr, 0, stream);
        if (rc != SGCLIP_OK) return rc;
    }
    if (dw_dev) {
        // the codes behind the last column are zeros, so that x reads back as one of whole groups of eight columns
        rc = sgclip_mxfp4_dequantize(x_codes_dev, x_scales_dev, M, p.k8, 0, ws + p.x, p.k8, stream);
        if (rc == SGCLIP_OK) rc = sgclip_gemm_tn_bf16(dy, (int)ld, ws + p.x, p.k8, sum, p.k8, p.n8, p.k8, M, stream);
        if (rc != SGCLIP_OK) return rc;
        if (p.crop) mx_crop_kernel<<<dim3(mx_grid((long long)N * K)), 256, 0, st>>>(sum, p.k8, N, K, dw_dev);
    }
    return launch_check(who);
}

}  // extern "C"
