// Rows to microscaled operands: the quantiser to E2M1 x E8M0 (or E4M3 x E8M0) and the residual + RMSNorm that ends in one.
//
// A group is 32 consecutive values with one E8M0 byte, value 2^(byte - 127):
//   E2M1: e = the smallest integer >= -126 with amax <= 6 * 2^e, code = x / 2^e to nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6};
//   E4M3: e = ceil(log2(max(amax, 1e-4) / 448)), code = x / 2^e to nearest even (dsv41_quant_fp8's rule).
// No value of a group saturates. A group that holds a NaN or an infinity gets byte 255 (E8M0's NaN) with codes 0 (E2M1) or 0x7F
// (E4M3's NaN), so every product with it is NaN instead of a finite number that hides the fault.
#include "common.h"
#include "mx.h"

namespace {

// eight consecutive values of a row as fp32
template <int DT>
struct Vec8 {
    float v[8];
    __device__ __forceinline__ void load(const void* base, long long i) {
        if constexpr (DT == MX_F32) {
            const v4f a = *(const v4f*)((const float*)base + i), b = *(const v4f*)((const float*)base + i + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
            const v4i w = *(const v4i*)((const uint16_t*)base + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = mx_unpack<DT>((uint32_t)w[j] & 0xFFFFu);
                v[2 * j + 1] = mx_unpack<DT>((uint32_t)w[j] >> 16);
            }
        }
    }
    __device__ __forceinline__ Raw8<MX_F32> raw() const { return Raw8<MX_F32>{v4f{v[0], v[1], v[2], v[3]}, v4f{v[4], v[5], v[6], v[7]}}; }
    __device__ __forceinline__ void store(void* base, long long i) const {
        if constexpr (DT == MX_F32) {
            *(v4f*)((float*)base + i) = v4f{v[0], v[1], v[2], v[3]};
            *(v4f*)((float*)base + i + 4) = v4f{v[4], v[5], v[6], v[7]};
        } else {
            v4i w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (int)mx_pack2<DT>(v[2 * j], v[2 * j + 1]);
            *(v4i*)((uint16_t*)base + i) = w;
        }
    }
};

}  // namespace

// ------------------------------------------------------------------------------------------ quantiser
// One lane takes eight values, four lanes a group; columns K .. Kp - 1 of the codes and scales are zero. One pass over x: the
// stream of x and of what is written bounds it (32768 x 5120 bf16 with the values written too: 126 us, 6.1 TB/s, without 74 us, 5.7; 16 x 5120: 2.8 us).
template <int DT, int FMT, int VALUES>
__global__ void __launch_bounds__(256) mx_quant_kernel(const void* __restrict__ x, long long ldx, long long rows, int K, int Kp,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint16_t* __restrict__ values) {
    const int per = Kp >> 3;                                     // units of eight values in a row
    const long long n = rows * per, step = (long long)gridDim.x * 256;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < n; u += step) {
        const long long r = u / per;
        const int c = (int)(u - r * per) * 8;
        Raw8<DT> x8;
        if (c < K) x8.load(x, r * ldx + c);
        else x8.zero();
        uint32_t w[2];
        const uint32_t b = mx_encode<FMT>(x8, w);
        if constexpr (FMT == 4) *(uint32_t*)(codes + u * 4) = w[0];
        else *(uint2*)(codes + u * 8) = make_uint2(w[0], w[1]);
        if ((u & 3) == 0) scales[u >> 2] = (uint8_t)b;
        if constexpr (VALUES) {
            v4i o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = (int)mx_bf16_pair(w[0], b, j);
            *(v4i*)(values + u * 8) = o;
        }
    }
}

extern "C" int dsv41_mx_quant(const void* x, int dtype, long long rows, int K, long long ldx, int fmt, int Kp, uint8_t* codes, uint8_t* scales,
                              uint16_t* values, void* stream) {
    const int es = dtype == MX_F32 ? 4 : 2;
    if (!x || !codes || !scales || dtype < 0 || dtype > 2 || (fmt != 4 && fmt != 8) || rows < 0 || K < 32 || (K & 31) || Kp < K || (Kp & 31) || ldx < K ||
        (values && (fmt != 4 || Kp != K)) || (ldx * es) % 16 || ((((uintptr_t)x) | ((uintptr_t)codes) | ((uintptr_t)values)) & 15))
        return DSV41_EINVAL;
    if (rows == 0) return 0;
    if (rows > (1ll << 52) / Kp) return DSV41_EINVAL;
    const long long blocks = (rows * (Kp / 8) + 255) / 256;
    const int grid = (int)(blocks < 65536 ? blocks : 65536);
    const hipStream_t st = (hipStream_t)stream;
#define MXQ(D, F, V) mx_quant_kernel<D, F, V><<<grid, 256, 0, st>>>(x, ldx, rows, K, Kp, codes, scales, values)
#define MXQ_D(D)                                   \
    case D:                                        \
        if (fmt == 8) MXQ(D, 8, 0);                \
        else if (values) MXQ(D, 4, 1);             \
        else MXQ(D, 4, 0);                         \
        break;
    switch (dtype) { MXQ_D(MX_BF16) MXQ_D(MX_F16) MXQ_D(MX_F32) }
#undef MXQ_D
#undef MXQ
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------ the tile kernels' operand
__device__ __forceinline__ void clear_words(uint32_t* zero, int zeros) {   // by the grid's first workgroup
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < zeros; i += blockDim.x) zero[i] = 0;
}

// 16 rows x 128 k per workgroup, so that the 16 rows' scale words of a tile are one 64-byte piece of [nk][M][4]. Bound by its bytes (8192 x
// 8192 bf16 to FP4: 34 us, 5.0 TB/s).
template <int DT, int FMT>
__global__ void __launch_bounds__(256) mx_operand_kernel(const void* __restrict__ x, long long ldx, int M, int K, int nk, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ scales, uint32_t* __restrict__ zero, int zeros) {
    clear_words(zero, zeros);
    const int c = threadIdx.x & 15;
    const int r = blockIdx.y * 16 + (threadIdx.x >> 4);
    const int t = blockIdx.x;
    if (r >= M) return;                                        // 16 lanes of a row together
    const int k = t * 128 + c * 8;
    Raw8<DT> v;
    if (k < K) v.load(x, (long long)r * ldx + k);
    else v.zero();
    uint32_t w[2];
    const uint32_t b = mx_encode<FMT>(v, w);
    const long long at = (long long)r * nk * 128 + k;
    if constexpr (FMT == 4) *(uint32_t*)(codes + (at >> 1)) = w[0];
    else *(uint2*)(codes + at) = make_uint2(w[0], w[1]);
    // the four groups' bytes of the row's tile as one word
    uint32_t word = (c & 3) ? 0u : b << (2 * c);
    word |= (uint32_t)__shfl_xor((int)word, 4, 16);
    word |= (uint32_t)__shfl_xor((int)word, 8, 16);
    if (c == 0) *(uint32_t*)(scales + ((long long)t * M + r) * 4) = word;
}

int mx_quant_operand(const void* x, int dtype, int M, int K, long long ldx, int fmt, int nk, uint8_t* codes, uint8_t* scales, uint32_t* zero, int zeros,
                     hipStream_t st) {
    if (M > 65535 * 16) return DSV41_EINVAL;
    const dim3 grid((unsigned)nk, (unsigned)((M + 15) / 16));
#define MXO(D)                                                                                \
    case D:                                                                                   \
        if (fmt == 4) mx_operand_kernel<D, 4><<<grid, 256, 0, st>>>(x, ldx, M, K, nk, codes, scales, zero, zeros); \
        else mx_operand_kernel<D, 8><<<grid, 256, 0, st>>>(x, ldx, M, K, nk, codes, scales, zero, zeros);          \
        break;
    switch (dtype) { MXO(MX_BF16) MXO(MX_F16) MXO(MX_F32) }
#undef MXO
    return (int)hipGetLastError();
}

typedef uint32_t u32_any __attribute__((aligned(1)));   // rows of scale bytes start anywhere

__global__ void __launch_bounds__(256) mx_turn_scales_kernel(const uint8_t* __restrict__ xs, long long ldxs, int M, int row_b, uint8_t* __restrict__ out,
                                                             uint32_t* __restrict__ zero, int zeros) {
    clear_words(zero, zeros);
    // a tile of 64 rows x up to 16 words through LDS: rows are read, and columns written, in contiguous pieces
    __shared__ uint32_t box[64][17];
    const int r0 = blockIdx.y * 64, t0 = blockIdx.x * 16, nk = (row_b + 3) / 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int i = j * 256 + threadIdx.x, r = i >> 4, t = i & 15, n = row_b - (t0 + t) * 4;   // bytes of the row from this word on
        if (r0 + r >= M || n <= 0) continue;
        const uint8_t* const p = xs + (long long)(r0 + r) * ldxs + (t0 + t) * 4;
        if (n >= 4) box[r][t] = *(const u32_any*)p;
        else box[r][t] = p[0] | (n > 1 ? (uint32_t)p[1] << 8 : 0u) | (n > 2 ? (uint32_t)p[2] << 16 : 0u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i & 63, t = i >> 6;
        if (r0 + r < M && t0 + t < nk) *(uint32_t*)(out + ((long long)(t0 + t) * M + r0 + r) * 4) = box[r][t];
    }
}

int mx_turn_scales(const uint8_t* xs, long long ldxs, int M, int K, uint8_t* out, uint32_t* zero, int zeros, hipStream_t st) {
    if (M > 65535 * 64) return DSV41_EINVAL;
    const int row_b = K / 32;
    mx_turn_scales_kernel<<<dim3((unsigned)((row_b + 63) / 64), (unsigned)((M + 63) / 64)), 256, 0, st>>>(xs, ldxs, M, row_b, out, zero, zeros);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------------------------ residual + RMSNorm
//   r = round_T(x + res)  (x itself without a residual);  v = r * (1 / sqrt(mean(r^2) + eps)) * w;  codes, scales = group(v)
// The sums are fp32, and v goes to its codes without a rounding in between (y, where asked for, is v rounded to T). r is rounded to
// the stream's type first because that is the value the next layer reads, and the statistics are of it.
// One workgroup per row, the row in registers between the two passes over it; the row's bytes bound it (16384 x 5120 bf16 to FP8: 108 us,
// 5.5 TB/s; to FP4 with y: 132 us, 5.4 TB/s; one row, 2.6 us: latency).
template <int DT, int FMT, int T, int C>
__global__ void __launch_bounds__(T) mx_norm_kernel(long long row0, const void* x, long long ldx, const void* res, long long ldr,
                                                    const void* __restrict__ g, float eps, double inv_k, int K, void* out, long long ldo, void* __restrict__ y,
                                                    uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ float part[T / 64];
    const long long row = row0 + blockIdx.x;
    const int tid = threadIdx.x;
    Vec8<DT> r[C];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int c = (i * T + tid) * 8;
        if (c < K) {
            r[i].load(x, row * ldx + c);
            if (res) {
                Vec8<DT> b;
                b.load(res, row * ldr + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) r[i].v[j] = mx_round<DT>(r[i].v[j] + b.v[j]);
                r[i].store(out, row * ldo + c);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(r[i].v[j], r[i].v[j], ss);
        }
    }
    ss = wave_reduce_sum(ss);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    // 1 / sqrt(mean + eps) in 64 bits (the instruction's estimate and one Newton step), as a sum of two floats: the factor is common to the
    // row, so its error would not average out. A mean that is no finite number above zero keeps the estimate: 0, infinity or NaN.
    double tot = 0.;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) tot += (double)part[i];
    const double m = fma(tot, inv_k, (double)eps), e0 = __builtin_amdgcn_rsq(m), e1 = fma(e0 * 0.5, fma(-m * e0, e0, 1.0), e0);
    const double inv = e1 == e1 ? e1 : e0;
    const float hi = (float)inv, lo = isfinite(hi) ? (float)(inv - (double)hi) : 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int c = (i * T + tid) * 8;
        if (c < K) {   // K % 32 == 0: the four lanes of a group take the same way
            Vec8<DT> w;
            w.load(g, c);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // r * (hi + lo) * w with the first product's rounding error carried along: v is within about half a step of fp32, and
                // fewer codes fall the other way at a rounding border (an infinite r or w keeps the plain product)
                const float p = r[i].v[j] * hi, pe = fmaf(r[i].v[j], lo, fmaf(r[i].v[j], hi, -p));
                const float v = fmaf(pe, w.v[j], p * w.v[j]), u = p * w.v[j];
                r[i].v[j] = v == v ? v : u;
            }
            if (y) r[i].store(y, row * K + c);
            uint32_t cw[2];
            const uint32_t b = mx_encode<FMT>(r[i].raw(), cw);
            const long long at = row * K + c;
            if constexpr (FMT == 4) *(uint32_t*)(codes + (at >> 1)) = cw[0];
            else *(uint2*)(codes + at) = make_uint2(cw[0], cw[1]);
            if ((tid & 3) == 0) scales[at >> 5] = (uint8_t)b;
        }
    }
}

extern "C" int dsv41_add_rmsnorm_mx(const void* x, long long ldx, const void* res, long long ldr, const void* w, float eps, int dtype, long long rows,
                                    int K, int fmt, void* out, long long ldo, void* y, uint8_t* codes, uint8_t* scales, void* stream) {
    const int es = dtype == MX_F32 ? 4 : 2;
    if (!x || !w || !codes || !scales || (res && !out) || dtype < 0 || dtype > 2 || (fmt != 4 && fmt != 8) || rows < 0 || rows > 0x7FFFFFFF || K < 32 ||
        (K & 31) || K > MX_NORM_MAX_K || !(eps >= 0.f) || ldx < K || (res && (ldr < K || ldo < K)) || (ldx * es) % 16 ||
        (res && ((ldr * es) % 16 || (ldo * es) % 16)) || ((((uintptr_t)x) | ((uintptr_t)res) | ((uintptr_t)w) | ((uintptr_t)out) | ((uintptr_t)y)) & 15) ||
        (((uintptr_t)codes) & 7))
        return DSV41_EINVAL;
    if (rows == 0) return 0;
    const hipStream_t st = (hipStream_t)stream;
    // a launch holds fewer than 2^32 threads
#define MXN(D, F, T, C)                                                                                                                        \
    for (long long r0 = 0, n; r0 < rows; r0 += n) {                                                                                            \
        n = rows - r0 < (1 << 21) ? rows - r0 : (1 << 21);                                                                                     \
        mx_norm_kernel<D, F, T, C><<<(unsigned)n, T, 0, st>>>(r0, x, ldx, res, ldr, w, eps, 1.0 / K, K, out, ldo, y, codes, scales);           \
    }
    // Many rows: 256 threads a row, so that eight rows share a CU and a thread has several pieces on the way. Few rows (or long ones): 1024
    // threads, one piece each, for the latency. bf16 to FP8, graph replays, 256 / 1024 threads: 5120 values a row, 1 row 4.7 / 4.2 us, 128 5.2 /
    // 4.5, 333 6.5 / 6.0, 512 7.2 / 6.6, 700 8.0 / 8.2, 2048 16.5 / 18.2; 7168: 1 5.4 / 4.1, 512 8.5 / 7.8, 1024 12.6 / 13.1; 2560: 333 4.8 / 4.7,
    // 1024 6.6 / 7.5, 4096 17.2 / 22.9.
#define MXN_K(D, F)                                     \
    if (K > 16384) { MXN(D, F, 1024, 4) }                  \
    else if (K > 8192) { MXN(D, F, 1024, 2) }              \
    else if (K > 2048 && rows < 512) { MXN(D, F, 1024, 1) } \
    else if (K > 6144) { MXN(D, F, 256, 4) }               \
    else if (K > 4096) { MXN(D, F, 256, 3) }               \
    else if (K > 2048) { MXN(D, F, 256, 2) }               \
    else { MXN(D, F, 256, 1) }
#define MXN_D(D) \
    case D:      \
        if (fmt == 8) { MXN_K(D, 8) } else { MXN_K(D, 4) } break;
    switch (dtype) { MXN_D(MX_BF16) MXN_D(MX_F16) MXN_D(MX_F32) }
#undef MXN_D
#undef MXN_K
#undef MXN
    return (int)hipGetLastError();
}
