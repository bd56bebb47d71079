// 8-bit integers for the linear layers: bt_quant_rows (one scale per row) and bt_linear_q8 (the product, with its epilogue).
#include "bt_common.h"
#include "bt_gelu.h"
#include "bt_quant.h"

#include <algorithm>
#include <type_traits>

namespace bt {

// Vectors at any element's address: rows of an odd length put every row but the first there.  The card takes such accesses whole
// (linear_q8 with 7707 rows of 5751 bf16 columns, K = 2560: 163 us by single elements, 107 so).
template <typename T> struct AnyVec;
template <> struct AnyVec<bf16> {
    typedef u32x4_t full __attribute__((aligned(2)));                                    // 8 elements
    typedef uint32_t four __attribute__((ext_vector_type(2), aligned(2)));               // 4
};
template <> struct AnyVec<float> {
    typedef u32x4_t full __attribute__((aligned(4)));
    typedef float four __attribute__((ext_vector_type(4), aligned(4)));
};

template <typename T>
__device__ inline void load_any(const T* p, float (&v)[Elem<T>::VEC]) {
    const u32x4_t u = *(const typename AnyVec<T>::full*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if constexpr (sizeof(T) == 2) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        else v[i] = __uint_as_float(u[i]);
}

// ---- bt_quant_rows ---------------------------------------------------------------------------------------------------------
// A row is read once into registers -- NV 16-byte pieces a lane, all loads in flight together -- and everything else happens there:
// LayerNorm statistics (two-pass, fp32), the largest magnitude, the codes.  R waves to a row: one where there are rows enough for
// the card (no barrier), four where there are not or where the row does not fit one wave's registers.  Bound by memory: x in, one
// byte a value out -- 8192 x 8192 bf16 35 us (5.7 TB/s), 4096 x 8192 22 us (4.6); with LayerNorm, 8192 x 2048 16.5 us (3.0 TB/s, six waves to
// a SIMD), 4000 x 1001 fp32 7.9 us; one row of 2048 3.0 us.
template <int R>
struct RowReduce {      // over the R waves of a row (R = 4: the workgroup)
    float* slot;
    int wave;
    __device__ inline float sum(float v) {
        v = sum64(v);
        if (R == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        return slot[0] + slot[1] + slot[2] + slot[3];
    }
    __device__ inline float max(float v) {
        v = max64(v);
        if (R == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        return fmaxf(fmaxf(slot[0], slot[1]), fmaxf(slot[2], slot[3]));
    }
};

// values c .. c + V - 1 of a row of K (zero beyond)
template <typename T>
__device__ inline void load_piece(const T* row, int c, int K, float (&v)[Elem<T>::VEC]) {
    constexpr int V = Elem<T>::VEC;
    if (c + V <= K) load_any<T>(row + c, v);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c + i < K ? Elem<T>::load(row + c + i) : 0.f;
}

template <typename T, bool LN, int NV, int R>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w,
                                                        const T* __restrict__ b, float eps, int8_t* __restrict__ codes, int64_t ldc,
                                                        float* __restrict__ scales, int64_t M, int K) {
    constexpr int V = Elem<T>::VEC;
    __shared__ float slot[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = R == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x;
    if (row >= M) return;
    const int at = R == 1 ? lane : threadIdx.x;      // piece i of this lane begins at column (i * 64 R + at) * V
    RowReduce<R> all{slot, wave};
    const T* xr = x + row * ldx;
    float v[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) load_piece<T>(xr, (i * 64 * R + at) * V, K, v[i]);
    if (LN) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[i][e];
        const float mean = all.sum(sum) / (float)K;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * R + at) * V;
            float part = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                part = fmaf(v[i][e], v[i][e], part);
            }
            if (c + V > K) {      // what lies behind the row does not count
                part = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) part = c + e < K ? fmaf(v[i][e], v[i][e], part) : part;
            }
            sq += part;
        }
        const float rstd = rsqrtf(all.sum(sq) / (float)K + eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * R + at) * V;
            float wv[V], bv[V];
            load_piece<T>(w, c, K, wv);
            load_piece<T>(b, c, K, bv);
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, wv[e], bv[e]);
            if (c + V > K) {      // (a weight of 0 does not make it 0: -mean * rstd may be infinite)
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = c + e < K ? v[i][e] : 0.f;
            }
        }
    }
    float amax = 0.f, zero = 0.f;      // (0 * v is 0 unless v is an infinity or NaN)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            amax = fmaxf(amax, fabsf(v[i][e]));
            zero = fmaf(v[i][e], 0.f, zero);
        }
    amax = all.max(zero == 0.f ? amax : INFINITY);
    const bool bad = amax == INFINITY;
    const Quantiser q(bad ? 0.f : amax);
    if (at == 0) scales[row] = bad ? __int_as_float(0x7fc00000) : q.scale;
    int8_t* cr = codes + row * ldc;
    const int Kp = (K + 15) & ~15;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * R + at) * V;
        if (c >= Kp) continue;
        uint32_t out[V / 4];
#pragma unroll
        for (int e = 0; e < V; e += 4)
            out[e / 4] = bad ? 0u : q.direct ? q.pack4(v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3])
                                             : q.pack4_exact(v[i][e], v[i][e + 1], v[i][e + 2], v[i][e + 3]);
        if constexpr (V == 8) *(uint2*)(cr + c) = uint2{out[0], out[1]};
        else *(uint32_t*)(cr + c) = out[0];
    }
}

// Rows longer than four waves' registers: a workgroup passes over the row once for each of the steps above (two, four with LayerNorm), an
// element a thread.  1000 x 20000 bf16 60 us (1.0 TB/s).
template <typename T, bool LN>
__global__ __launch_bounds__(256) void quant_long_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w,
                                                             const T* __restrict__ b, float eps, int8_t* __restrict__ codes, int64_t ldc,
                                                             float* __restrict__ scales, int64_t K) {
    __shared__ float slot[4];
    RowReduce<4> all{slot, (int)threadIdx.x >> 6};
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    float mean = 0.f, rstd = 1.f;
    if (LN) {
        float sum = 0.f, sq = 0.f;
        for (int64_t c = threadIdx.x; c < K; c += 256) sum += Elem<T>::load(xr + c);
        mean = all.sum(sum) / (float)K;
        for (int64_t c = threadIdx.x; c < K; c += 256) {
            const float d = Elem<T>::load(xr + c) - mean;
            sq = fmaf(d, d, sq);
        }
        rstd = rsqrtf(all.sum(sq) / (float)K + eps);
    }
    auto value = [&](int64_t c) {
        const float v = Elem<T>::load(xr + c);
        return LN ? fmaf((v - mean) * rstd, Elem<T>::load(w + c), Elem<T>::load(b + c)) : v;
    };
    float amax = 0.f;
    for (int64_t c = threadIdx.x; c < K; c += 256) {
        const float v = fabsf(value(c));
        amax = v < INFINITY ? fmaxf(amax, v) : INFINITY;
    }
    amax = all.max(amax);
    const bool bad = amax == INFINITY;
    const Quantiser q(bad ? 0.f : amax);
    if (threadIdx.x == 0) scales[row] = bad ? __int_as_float(0x7fc00000) : q.scale;
    int8_t* cr = codes + row * ldc;
    const int64_t Kp = (K + 15) / 16 * 16;
    for (int64_t c = threadIdx.x; c < Kp; c += 256) cr[c] = (int8_t)(c < K && !bad ? q.exact(value(c)) : 0);
}

template <typename T>
static int launch_quant_rows(int64_t M, int64_t K, const void* x, int64_t ldx, const void* w, const void* b, float eps, int8_t* codes,
                             int64_t ldc, float* scales, hipStream_t s) {
    constexpr int V = Elem<T>::VEC;
    ProfScope ps(BT_PROF_LAYERNORM, s);
    const int64_t wave_pieces = ceil_div(K, 64 * V), group_pieces = ceil_div(K, 256 * V);
    // one wave to a row from 2048 rows (8 waves to a CU) while it has at most 8 pieces a lane
    const bool one = wave_pieces <= 8 && M >= 2048;
    const int64_t pieces = one ? wave_pieces : group_pieces;
    const int64_t groups = one ? ceil_div(M, 4) : M;
    BT_CHECK_ARG(groups < (1ll << 24), "bt_quant_rows: %lld rows are too many for one launch", (long long)M);      // (2^32 threads)
    const dim3 grid((unsigned)groups);
#define BT_QR(LN_, NV_, R_)                                                                                                          \
    hipLaunchKernelGGL((quant_rows_kernel<T, LN_, NV_, R_>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, \
                       codes, ldc, scales, M, (int)K)
#define BT_QR_PIECES(LN_, R_)              \
    do {                                   \
        if (pieces <= 1) BT_QR(LN_, 1, R_); \
        else if (pieces <= 2) BT_QR(LN_, 2, R_); \
        else if (pieces <= 4) BT_QR(LN_, 4, R_); \
        else BT_QR(LN_, 8, R_);            \
    } while (0)
    if (pieces > 8) {
        if (w) hipLaunchKernelGGL((quant_long_rows_kernel<T, true>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes, ldc, scales, K);
        else hipLaunchKernelGGL((quant_long_rows_kernel<T, false>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes, ldc, scales, K);
    } else if (w) {
        if (one) BT_QR_PIECES(true, 1);
        else BT_QR_PIECES(true, 4);
    } else {
        if (one) BT_QR_PIECES(false, 1);
        else BT_QR_PIECES(false, 4);
    }
#undef BT_QR_PIECES
#undef BT_QR
    BT_LAUNCH_CHECK("bt_quant_rows launch");
    return BT_OK;
}

// ---- bt_linear_q8 ----------------------------------------------------------------------------------------------------------
typedef int i32x4 __attribute__((ext_vector_type(4)));

typedef i32x4 i32x4_any __attribute__((aligned(4)));

struct Q8Args {
    const int8_t* A;
    const int8_t* W;
    int64_t lda, ldw;
    int M, N, K;
    const float* a_scale;
    const float* w_scale;
    const void* bias;
    const void* residual;
    int64_t ldr;
    void* out;
    int64_t ldo;
    int act;
    int fours;          // w_scale and bias give four columns at a time
    int tiles_m, tiles_n;
    int slices, steps;  // K split into `slices` ranges of `steps` 64-byte steps; > 1: sums go to `slab`
    int* slab;          // [slices][M][N]
};

// act(acc * sx * sw + bias): fp32; the residual joins where the row is written.  GELU: erf for fp32, the polynomial of the other bf16
// epilogues (8.5e-6 relative) where the result is rounded to 8 bits.
template <typename T>
__device__ inline void q8_values(const i32x4& acc, float sa, const float (&sw)[4], const float (&bias)[4], int act, float (&y)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = fmaf((float)acc[r], sa * sw[r], bias[r]);
    if (act == BT_ACT_GELU) {
        if constexpr (sizeof(T) == 2) gelu4(y);
        else
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = 0.5f * y[r] * (1.0f + erff(y[r] * 0.70710678118654752440f));
    }
}

// 16 bytes per lane from base + off (unsigned) straight into LDS at lds + 16 * lane.  The waits cover an M0 write right before the load
// (1) and a base that a v_readlane may just have brought back from a spill (5): neither is padded inside an asm string.
__device__ inline void dma16(const int8_t* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds) : "memory");
}
template <int N>
__device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// Tile number `round` of this workgroup, of those that `groups` workgroups take a round at a time; false: there is none.  Workgroups of one
// XCD (ids that are equal mod 8) take neighbouring tiles, in columns of HIGH tile rows: its L2 serves them with each other's panels.
template <int HIGH>
__device__ inline bool q8_tile(const Q8Args& e, int groups, int round, int& tm, int& tn) {
    const int base = round * groups, tiles = min(e.tiles_m * e.tiles_n - base, groups), id = blockIdx.x;
    const int per = tiles >> 3, rest = tiles & 7, xcd = id & 7, local = id >> 3;
    if (tiles <= 0 || local >= per + (xcd < rest)) return false;
    const int at = base + (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + local;
    const int group = at / (HIGH * e.tiles_n), first = group * HIGH, high = min(e.tiles_m - first, HIGH), in = at - group * HIGH * e.tiles_n;
    tm = first + in % high;
    tn = in / high;
    return true;
}

constexpr int q8_pitch(int nb) { return 16 * nb * 2 + 16; }      // bytes of a row of a wave's bf16 patch: its 16 NB columns

// The sums of a wave, NI fragments of 16 rows (row0(i) is the first of fragment i) by 16 NB columns from n_w: lane (c, g) has columns
// 16 j + 4 g .. + 3 of row c.  Scales, bias, activation and residual there, then one rounding.  fp32 leaves from there, 16 bytes a lane;
// bf16 rows are put together in `patch` (16 rows, the wave's own) first.  A wave's part that is whole takes NI NB / 2 (bf16)
// or NI NB stores.
template <typename T, int NI, int NB, typename Row0>
__device__ inline void q8_write(const Q8Args& e, const i32x4 (&acc)[NI][NB], char* patch, int n_w, int lane, Row0 row0) {
    constexpr int PITCH = q8_pitch(NB);
    const int c = lane & 15, g = lane >> 4;
    // every load of scales and bias at once, and the residual's one fragment ahead: a load that is waited for costs a microsecond here
    float sa[NI], sw[NB][4], bias[NB][4];
#pragma unroll
    for (int i = 0; i < NI; ++i) sa[i] = e.a_scale[min(row0(i) + c, e.M - 1)];
    const bool fours = e.fours && n_w + 16 * NB <= e.N;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int n = n_w + j * 16 + g * 4;
        if (fours) {
            const float4 s4 = *(const float4*)(e.w_scale + n);
            sw[j][0] = s4.x, sw[j][1] = s4.y, sw[j][2] = s4.z, sw[j][3] = s4.w;
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[j][r] = 0.f;
            if (e.bias) {
                if constexpr (sizeof(T) == 2) {
                    const uint2 u = *(const uint2*)((const T*)e.bias + n);
                    bias[j][0] = __uint_as_float(u.x << 16), bias[j][1] = __uint_as_float(u.x & 0xffff0000u);
                    bias[j][2] = __uint_as_float(u.y << 16), bias[j][3] = __uint_as_float(u.y & 0xffff0000u);
                } else {
                    const float4 u = *(const float4*)((const T*)e.bias + n);
                    bias[j][0] = u.x, bias[j][1] = u.y, bias[j][2] = u.z, bias[j][3] = u.w;
                }
            }
        } else
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                sw[j][r] = e.w_scale[min(n + r, e.N - 1)];
                bias[j][r] = e.bias ? Elem<T>::load((const T*)e.bias + min(n + r, e.N - 1)) : 0.f;
            }
    }
    // whole columns go in 16-byte pieces, whole rows with no test a row; a row's address is a scalar and one lane offset
    const bool cols = n_w + 16 * NB <= e.N, whole = cols && row0(NI - 1) + 16 <= e.M;
    typedef typename AnyVec<T>::four Four;
    typedef typename AnyVec<T>::full Full;
    Four next[NB] = {};
    auto load_residual = [&](int i) {
        const int m = row0(i) + c;
        if (!e.residual || m >= e.M) return;
        const T* p = (const T*)e.residual + (int64_t)row0(i) * e.ldr + n_w + (uint32_t)(c * (int)e.ldr + g * 4);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int n = n_w + j * 16 + g * 4;
            if (cols) next[j] = *(const Four*)(p + j * 16);
            else {
                T v[4] = {};
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < e.N) v[r] = p[j * 16 + r];
                __builtin_memcpy(&next[j], v, sizeof v);
            }
        }
    };
    load_residual(0);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        Four res[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) res[j] = next[j];
        if (i + 1 < NI) load_residual(i + 1);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float y[4];
            q8_values<T>(acc[i][j], sa[i], sw[j], bias[j], e.act, y);
            if (e.residual) {
                if constexpr (sizeof(T) == 2) {
                    y[0] += __uint_as_float(res[j].x << 16), y[1] += __uint_as_float(res[j].x & 0xffff0000u);
                    y[2] += __uint_as_float(res[j].y << 16), y[3] += __uint_as_float(res[j].y & 0xffff0000u);
                } else {
                    y[0] += res[j].x, y[1] += res[j].y, y[2] += res[j].z, y[3] += res[j].w;
                }
            }
            if constexpr (sizeof(T) == 2) {
                *(uint2*)(patch + c * PITCH + (j * 16 + g * 4) * 2) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
            } else {
                T* out = (T*)e.out + (int64_t)row0(i) * e.ldo + n_w + (uint32_t)(c * (int)e.ldo + g * 4) + j * 16;
                if (whole || (cols && row0(i) + c < e.M))
                    *(Full*)out = u32x4_t{__float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3])};
                else if (!cols && row0(i) + c < e.M)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n_w + j * 16 + g * 4 + r < e.N) out[r] = y[r];
            }
        }
        if constexpr (sizeof(T) == 4) continue;
        asm volatile("" ::: "memory");      // the patch is the wave's own, and a wave's LDS accesses stay in order
        constexpr int V = Elem<T>::VEC, CH = 16 * NB / V;      // 16-byte pieces of a row
#pragma unroll
        for (int x = 0; x < 16 * CH; x += 64) {
            const int r0 = x / CH, r = lane / CH, d = (lane - r * CH) * V;      // (64 is a multiple of CH)
            const u32x4_t v = *(const u32x4_t*)(patch + (r0 + r) * PITCH + d * sizeof(T));
            T* out = (T*)e.out + (int64_t)(row0(i) + r0) * e.ldo + n_w + (uint32_t)(r * (int)e.ldo + d);
            if (whole || (cols && row0(i) + r0 + r < e.M)) *(Full*)out = v;
            else if (!cols && row0(i) + r0 + r < e.M) {
                T y[V];
                __builtin_memcpy(y, &v, sizeof v);
#pragma unroll
                for (int q = 0; q < V; ++q)
                    if (n_w + d + q < e.N) out[q] = y[q];
            }
        }
        asm volatile("" ::: "memory");
    }
}

// The tile kernel: 32 MI x 32 NB per workgroup of 2 x 2 waves, 64 bytes of K a step; of a last step that is not whole, what lies behind K
// is replaced by the step's first bytes, and A's operand is zero there.
//  * Two workgroups to a CU: while one waits at its barrier or writes its tile, the other's waves have the matrix units.  So a K step
//    needs one barrier and the epilogue no software overlap.
//  * A and W travel global -> LDS without registers, NS - 1 steps ahead, in a ring of NS stages, and LDS -> registers one step ahead: the
//    fragments of step t + 1 are read under the products of step t.  In step t a wave waits for its own loads of step t + 1 (in order: at
//    most those of the younger steps stay out), then for the others at the barrier; behind it everybody has also multiplied step t - 1,
//    whose stage takes the loads of step t + NS - 1.
//  * LDS rows are 64 bytes; the four 16-byte pieces of row r are stored in the order p ^ ((r >> 1) & 3) ^ ((r >> 3) & 1): the 16 rows that
//    a fragment read touches at once are spread over all banks.
//  * mfma(W, A): a lane gets four neighbouring columns of one row (q8_write).
// 256 x 6144 x 2048 10 .. 12 us by 64 x 64 tiles, 2048 x 2048 x 8192 45 us (1.5 POPS) by 128 x 128: bound by
// the way from L2 into a CU, as the largest kernel is, with more bytes to an operation.
template <typename T, int MI, int NB, int NS>
__global__ __launch_bounds__(256, 2) void linear_q8_tile_kernel(Q8Args e) {
    constexpr int BM = 32 * MI, BN = 32 * NB, STAGE = (BM + BN) * 64;
    constexpr int LA = BM / 64, LW = BN / 64, LOADS = LA + LW;      // 1 KiB loads of a wave and step
    constexpr int PITCH = q8_pitch(NB);
    static_assert(4 * 16 * PITCH <= NS * STAGE, "the patches take the ring's place");
    __shared__ __attribute__((aligned(16))) char smem[NS * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, c = lane & 15, g = lane >> 4;

    int m0, n0;
    q8_tile<8>(e, gridDim.x, 0, m0, n0);
    m0 *= BM;
    n0 *= BN;
    const int k0 = blockIdx.y * e.steps * 64, steps = min(e.steps, (e.K - k0 + 63) >> 6);
    const int whole = min(4, (e.K - k0 - (steps - 1) * 64) >> 4);      // 16-byte pieces of the last step
    const int cut = whole < 4 ? steps - 1 : -1;
    const int8_t* A = e.A + (int64_t)m0 * e.lda + k0;
    const int8_t* W = e.W + (int64_t)n0 * e.ldw + k0;
    uint32_t off[LOADS];
    const int row16 = lane >> 2, piece = (lane & 3) ^ ((row16 >> 1) & 3) ^ ((row16 >> 3) & 1);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        int row = i < LA ? (wave * LA + i) * 16 + row16 : (wave * LW + i - LA) * 16 + row16;
        const int last = i < LA ? e.M - 1 - m0 : e.N - 1 - n0;      // rows beyond the matrix repeat its last one
        row = row < last ? row : last;
        off[i] = (uint32_t)row * (uint32_t)(i < LA ? e.lda : e.ldw) + piece * 16;
    }
    const uint32_t back = piece >= whole ? piece * 16 : 0;
    const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)smem;
    auto load = [&](int t) {
        const uint32_t stage = ring + (t % NS) * STAGE;
        const uint32_t less = t == cut ? back : 0;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (i < LA) dma16(A + (int64_t)t * 64, off[i] - less, stage + (wave * LA + i) * 1024);
            else dma16(W + (int64_t)t * 64, off[i] - less, stage + BM * 64 + (wave * LW + i - LA) * 1024);
    };
    i32x4 acc[MI][NB];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < steps) load(t);

    const int frag = c * 64 + (g ^ ((c >> 1) & 3) ^ ((c >> 3) & 1)) * 16;
    struct Step {
        i32x4 a[MI], w[NB];
    } f[2];
    auto read = [&](int t, Step& x) {
        const char* a = smem + (t % NS) * STAGE + wm * MI * 1024 + frag;
        const char* w = smem + (t % NS) * STAGE + BM * 64 + wn * NB * 1024 + frag;
#pragma unroll
        for (int j = 0; j < NB; ++j) x.w[j] = *(const i32x4*)(w + j * 1024);
#pragma unroll
        for (int i = 0; i < MI; ++i) x.a[i] = *(const i32x4*)(a + i * 1024);
    };
    auto multiply = [&](const Step& x) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.w[j], x.a[i], acc[i][j], 0, 0, 0);
    };
    auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto step = [&](int t, const Step& now, Step& next) {      // step t of two or more, not the last
        if (t + NS - 2 < steps) wait_loads<LOADS * (NS - 3)>();
        else if (NS > 5 && t + 4 < steps) wait_loads<LOADS * 2>();      // (at most what is still out)
        else wait_loads<0>();
        barrier();
        if (t + NS - 1 < steps) load(t + NS - 1);
        read(t + 1, next);
        multiply(now);
    };
    if (steps >= NS - 1) wait_loads<LOADS * (NS - 2)>();
    else wait_loads<0>();
    barrier();
    read(0, f[0]);
    int t = 0;
    for (; t + 2 < steps; t += 2) {
        step(t, f[0], f[1]);
        step(t + 1, f[1], f[0]);
    }
    if (t + 1 < steps) {
        step(t, f[0], f[1]);
        f[0] = f[1];
    }
    if (whole < 4 && g >= whole) {
#pragma unroll
        for (int i = 0; i < MI; ++i) f[0].a[i] = i32x4{0, 0, 0, 0};
    }
    multiply(f[0]);

    const int m_w = m0 + wm * MI * 16, n_w = n0 + wn * NB * 16;
    if (e.slices > 1) {
        int* slab = e.slab + (int64_t)blockIdx.y * e.M * e.N;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int m = m_w + i * 16 + c;
            if (m >= e.M) continue;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int n = n_w + j * 16 + g * 4;
                if (n + 4 <= e.N) *(i32x4_any*)(slab + (int64_t)m * e.N + n) = acc[i][j];
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < e.N) slab[(int64_t)m * e.N + n + r] = acc[i][j][r];
            }
        }
        return;
    }
    __syncthreads();      // the ring is the patches' now
    q8_write<T, MI, NB>(e, acc, smem + wave * 16 * PITCH, n_w, lane, [&](int i) { return m_w + i * 16; });
}

// The kernel for large products: 256 x 64 NB (256 or 128) per workgroup of eight waves, 128 bytes of K a step, K % 128 == 0.  What bounds a
// large product here is the way from L2 into a CU (about 25 bytes a clock measured, and it moves whole 128-byte lines): a 256 x 256 tile
// asks for a third less than 256 x 128 does, that for a quarter less than 128 x 128, and a step of 128 bytes takes every line once.  256 x 128
// is for products that have about 256 of them.  There is room for one workgroup to a CU, so its waves take turns by themselves:
//  * The waves are two groups of four, one of each on every SIMD, half a phase apart: while one group's MFMAs run (a phase has 8 NB of them),
//    the other reads its fragments and sends loads.  Group 1 begins with one barrier more, so its first barrier of a phase meets group
//    0's second.
//  * A step has two phases, one for each half (128 rows) of A; W's fragments are read in the first and kept.  LDS holds RING steps of half
//    tiles (A0, W0, W1, A1, or A0, W, A1: in the order in which they are wanted).  Phase (t, 0) sends what follows W0 of step t + RING - 1,
//    phase (t, 1) sends A0 and W0 of step t + RING into the places that phase (t, 0) has read.
//  * A workgroup stays for all its tiles, and the loads run on from one tile into the next: when a tile's sums are finished, the next
//    one's first RING steps are on their way or there, so its products start behind the epilogue without a wait, and the epilogue's stores
//    drain under them.
//  * Waits are for all but the youngest loads (they return in order; a half tile is two).  In front of phase (t, 0) what may still be out is
//    A1 of the step, the next RING - 2 steps, and A0, W0 of the one after; in front of (t, 1), the next RING - 1 steps.  In a tile's
//    first step all of the next RING - 1 are out (they went ahead of the epilogue).  In the first RING steps of a tile the stores
//    of the one before are younger than the loads in question and are counted as well, if that tile was whole (else their number varies,
//    and the wait is for them too).  In the last RING - 1 steps of all, for everything.  Group 0 waits at the top of a phase, group 1 for the
//    next phase's before its second barrier, which is the one that opens that phase to group 0.
//  * A wave's reads have returned before its second barrier of a phase; the other group sends the loads that overwrite those places behind
//    that barrier.
//  * A tile ends with one more barrier for group 0 (group 1 has then read its last) and begins with one more for group 1, so the two
//    epilogues run side by side.
//  * A row of 128 bytes has its 16-byte pieces in the order p ^ (row & 7).
// Launch after launch in a graph: 8192 x 8192 x 2048 131 us (2.1 POPS), with GELU 141 .. 152 us by card, 8192 x 8192 x 8192
// 398 us (2.8 POPS, matrix units busy two thirds of the time at the 1.8 GHz that the card then holds); of the 131 us, 107 are the products,
// 10 the stores and 14 the rest of the epilogue.  4096 x 2048 x 8192 by 256 x 128 65 .. 72 us (2.1 POPS; by 128 x 128 77, by 256 x 256 on
// half the CUs 80).  Single launches under the profiler: 156 with GELU, 425 and 77 .. 85 us.  fp32 results: 176 us with GELU, 4096 x 2048 x
// 8192 74 us; the 256 x 256 form has six registers too few there and brings its load offsets back from scratch at a tile's start, which
// waits for every load that is out.
template <typename T, int NB>
__global__ __launch_bounds__(512, 2) void linear_q8_big_kernel(Q8Args e) {
    constexpr int HALVES = NB == 4 ? 4 : 3, RING = NB == 4 ? 2 : 3, COLS = 64 * NB;      // A0, W0, (W1,) A1
    constexpr int HALF = 128 * 128, STEP = HALVES * HALF, PITCH = q8_pitch(NB), PATCH = sizeof(T) == 2 ? 16 * PITCH : 0;
    constexpr int STORES = sizeof(T) == 2 ? 4 * NB : 8 * NB;      // of a wave and whole tile
    constexpr int LOADS = 2 * HALVES;                             // of a wave and step
    __shared__ __attribute__((aligned(16))) char smem[RING * STEP + 8 * PATCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3, c = lane & 15, g = lane >> 4;
    const bool second = wm != 0;
    const int steps = e.K >> 7;

    // the loads: step `lt` of tile number `lround`, into place `lx` of the ring
    int lm = 0, ln = 0, lt = 0, lround = 0, lx = 0;
    bool more = true;
    const int8_t *A = nullptr, *W = nullptr;
    uint32_t off[HALVES][2];      // [half tile][load]
    auto enter = [&] {
        more = q8_tile<4>(e, gridDim.x, lround, lm, ln);
        if (!more) return;
        A = e.A + (int64_t)lm * 256 * e.lda;
        W = e.W + (int64_t)ln * COLS * e.ldw;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bool a = h == 0 || h == HALVES - 1;
                int row = (h >= 2 ? 128 : 0) + wave * 16 + i * 8 + (lane >> 3);
                const int last = a ? e.M - 1 - lm * 256 : e.N - 1 - ln * COLS;      // rows beyond the matrix repeat its last one
                row = row < last ? row : last;
                off[h][i] = (uint32_t)row * (uint32_t)(a ? e.lda : e.ldw) + (uint32_t)((lane & 7) ^ (lane >> 3)) * 16;
            }
    };
    const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)smem + wave * 2048;
    auto load = [&](auto half) {
        constexpr int h = decltype(half)::value;
        if (!more) return;
        const int8_t* base = h == 0 || h == HALVES - 1 ? A : W;
        dma16(base, off[h][0], ring + lx * STEP + h * HALF);
        dma16(base, off[h][1], ring + lx * STEP + h * HALF + 1024);
    };
    using H0 = std::integral_constant<int, 0>;
    using H1 = std::integral_constant<int, 1>;
    using H2 = std::integral_constant<int, 2>;
    using H3 = std::integral_constant<int, 3>;
    auto first_half = [&] { load(H0{}); load(H1{}); };
    auto second_half = [&] {
        load(H2{});
        if constexpr (HALVES == 4) load(H3{});
        lx = lx + 1 == RING ? 0 : lx + 1;
        A += 128;
        W += 128;
        if (++lt == steps) {
            lt = 0;
            ++lround;
            if (more) enter();
        }
    };
    auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    enter();
#pragma unroll
    for (int i = 0; i < RING; ++i) {
        first_half();
        second_half();
    }

    int m0, n0, at = 0;     // the tile, and the step's place in the ring
    const int rounds = e.tiles_m * e.tiles_n / (int)gridDim.x;      // that every workgroup has a tile in; one more is some workgroups'
    int left = (rounds + q8_tile<4>(e, gridDim.x, rounds, m0, n0)) * steps;      // steps of all that are still to be done
    bool stores = false;    // the tile before has left STORES stores behind the loads of this one's first RING steps
    for (int round = 0; q8_tile<4>(e, gridDim.x, round, m0, n0); ++round) {
        m0 *= 256;
        n0 *= COLS;
        i32x4 acc[8][NB];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
        constexpr int FIRST = 2 + (RING - 2) * LOADS + 4, WHOLE = 2 + (RING - 1) * LOADS, SECOND = (RING - 1) * LOADS;
        auto wait_first = [&](int t, int left) {      // for phase (t, 0)
            if (left < RING) wait_loads<0>();
            else if (t == 0 && stores) wait_loads<WHOLE + STORES>();
            else if (t == 0) wait_loads<WHOLE>();
            else if (t < RING && stores) wait_loads<FIRST + STORES>();
            else wait_loads<FIRST>();
        };
        auto wait_second = [&](int t) {     // for phase (t, 1)
            if (left < RING) wait_loads<0>();
            else if (t < RING && stores) wait_loads<SECOND + STORES>();
            else wait_loads<SECOND>();
        };
        if (second) {
            wait_first(0, left);
            barrier();
        }
        const int p0 = (g ^ (c & 7)) * 16, p1 = ((4 + g) ^ (c & 7)) * 16;      // this lane's pieces of a row: the step's first and second 64 bytes
        i32x4 af[4][2], wf[NB][2];
        for (int t = 0; t < steps; ++t, --left, at = at + 1 == RING ? 0 : at + 1) {
            const char* step = smem + at * STEP;
            const char* a = step + (wm * 64 + c) * 128;
            const char* w = step + HALF + (wn * 16 * NB + c) * 128;
            // phase 0
            if (!second) wait_first(t, left);
            barrier();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < NB) wf[j][0] = *(const i32x4*)(w + j * 2048 + p0);
                af[j][0] = *(const i32x4*)(a + j * 2048 + p0);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j < NB) wf[j][1] = *(const i32x4*)(w + j * 2048 + p1);
                af[j][1] = *(const i32x4*)(a + j * 2048 + p1);
            }
            if (t > 0) second_half();
            if (second) wait_second(t);
            __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
            barrier();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][k], af[i][k], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
            // phase 1
            if (!second) wait_second(t);
            barrier();
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) af[i][k] = *(const i32x4*)(a + (HALVES - 1) * HALF + i * 2048 + (k ? p1 : p0));
            first_half();
            if (second && t + 1 < steps) wait_first(t + 1, left - 1);
            __builtin_amdgcn_s_waitcnt(0xc07f);
            barrier();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[4 + i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j][k], af[i][k], acc[4 + i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!second) barrier();      // group 1 has read its last fragments
        second_half();
        int hide = lane;
        asm volatile("" : "+v"(hide));      // the epilogue's addresses are not to be kept in registers through the products
        q8_write<T, 8, NB>(e, acc, smem + RING * STEP + wave * PATCH, n0 + wn * 16 * NB, hide, [&](int i) { return m0 + (i >> 2) * 128 + wm * 64 + (i & 3) * 16; });
        stores = m0 + 256 <= e.M && n0 + COLS <= e.N;
    }
}

// Few rows: 16 MB rows by 16 columns per workgroup, its eight waves dividing K among themselves.  W is read once, straight into the operand
// registers of the matrix instruction (a lane holds 16 bytes of a row: nothing to rearrange, no LDS, no barrier in the loop), with
// every load of four (MB = 2: two) 128-byte units out at once: a problem of this size is a few microseconds of latency, not of bandwidth.
// A comes the same way, from the caches.  The partial sums meet in LDS; being integers, they do not depend on the number of waves.  One
// row: 6144 x 2048 5.4 us (2.3 TB/s of weights), 8192 x 2048 5.6 us (3.0 TB/s), 2048 x 8192 7.4 us (128 workgroups: half the CUs).
template <typename T, int MB>
__global__ __launch_bounds__(512) void linear_q8_rows_kernel(Q8Args e) {
    constexpr int NW = 8, U = MB == 1 ? 4 : 2;      // waves, units of a round
    __shared__ i32x4 part[NW][MB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MB;
    const int8_t* ap[MB];
    const int8_t* wp = e.W + (int64_t)min(n0 + c, e.N - 1) * e.ldw + 16 * g;
#pragma unroll
    for (int i = 0; i < MB; ++i) ap[i] = e.A + (int64_t)min(m0 + 16 * i + c, e.M - 1) * e.lda + 16 * g;
    i32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = i32x4{0, 0, 0, 0};
    const i32x4 zero{0, 0, 0, 0};
    for (int k = wave * 128; k < e.K; k += NW * 128 * U) {
        i32x4 a[U][2][MB], w[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = k + u * NW * 128 + h * 64;
                const bool in = at + 16 * g < e.K;      // K is a whole number of 16-byte pieces
                w[u][h] = in ? *(const i32x4*)(wp + at) : zero;
#pragma unroll
                for (int i = 0; i < MB; ++i) a[u][h][i] = in ? *(const i32x4*)(ap[i] + at) : zero;
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MB; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u][h], a[u][h][i], acc[i], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    // lane (c, g) of fragment f: row c, columns 4 g .. 4 g + 3
    for (int x = threadIdx.x; x < MB * 64; x += NW * 64) {
        const int f = x >> 6, l = x & 63;
        i32x4 sum = part[0][f][l];
#pragma unroll
        for (int w = 1; w < NW; ++w) sum += part[w][f][l];
        const int m = m0 + f * 16 + (l & 15), n = n0 + (l >> 4) * 4;
        if (m >= e.M || n >= e.N) continue;
        float sw[4], bias[4], y[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sw[r] = e.w_scale[min(n + r, e.N - 1)];
            bias[r] = e.bias ? Elem<T>::load((const T*)e.bias + min(n + r, e.N - 1)) : 0.f;
        }
        q8_values<T>(sum, e.a_scale[m], sw, bias, e.act, y);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= e.N) continue;
            if (e.residual) y[r] += Elem<T>::load((const T*)e.residual + (int64_t)m * e.ldr + n + r);
            Elem<T>::store((T*)e.out + (int64_t)m * e.ldo + n + r, y[r]);
        }
    }
}

// Joins K slices: sums them (integers: in any order) and finishes as the tile kernel does.  Four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void linear_q8_join_kernel(Q8Args e) {
    const int quads = (e.N + 3) >> 2;
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (x >= (int64_t)e.M * quads) return;
    const int m = (int)(x / quads), n = (int)(x - (int64_t)m * quads) * 4;
    const int64_t slice = (int64_t)e.M * e.N;
    const int* p = e.slab + (int64_t)m * e.N + n;
    const bool four = n + 4 <= e.N;
    i32x4 sum{0, 0, 0, 0};
    for (int s = 0; s < e.slices; ++s, p += slice) {
        if (four) sum += *(const i32x4_any*)p;
        else
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n + r < e.N) sum[r] += p[r];
    }
    float sw[4], bias[4], y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        sw[r] = e.w_scale[min(n + r, e.N - 1)];
        bias[r] = e.bias ? Elem<T>::load((const T*)e.bias + min(n + r, e.N - 1)) : 0.f;
    }
    q8_values<T>(sum, e.a_scale[m], sw, bias, e.act, y);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= e.N) continue;
        if (e.residual) y[r] += Elem<T>::load((const T*)e.residual + (int64_t)m * e.ldr + n + r);
        Elem<T>::store((T*)e.out + (int64_t)m * e.ldo + n + r, y[r]);
    }
}

// What runs a product, from its sizes alone: the cheapest by a model of the time in microseconds, fitted to graph-replayed launches of
// M = 64 .. 8192 by N = 512 .. 8192 by K = 256 .. 8192, odd ones among them (half of them within 8 % of it, nine in ten within 22 %; its
// choice is 1.4 % above the best of them on average, 29 % at most).
//   64 x 64 tiles    3.5 + 0.8 times their number t to a CU + 0.15 a step, or 0.12 t    (256 x 6144 x 2048: 10.6; 128 x 128 tiles 14.0)
//   128 x 128 tiles  4.5 + 1.5 t + 0.28 a step, 0.5 where some CUs have two, or 0.3 t   (2048 x 2048 x 2048: 15.1; 256 x 128 tiles 20.5)
//   256 x 128 tiles  5.5 + 3 a round + 0.44 a step, 0.38 where few CUs have one         (4096 x 2048 x 8192: 64.7; 128 x 128 tiles 77,
//                                                                                        256 x 256 80)
//   256 x 256 tiles  5 + 5 a round + 0.73 a step, 0.53 up to half the CUs               (8192 x 2048 x 2048: 33.5; 256 x 128 tiles 44)
//   K in slices      3 for the second launch, and the sums once out and in at 4 TB/s    (128 x 2048 x 8192 in 4: 13.9; whole 22.1)
// Up to 32 rows the rows kernel, which reads W as fast as it comes (32 x 6144 x 2048: 8.2; 64 rows by tiles 7.9, by rows 9.5).
struct Q8Plan {
    enum Kind { ROWS, TILE64, TILE128, TALL, BIG } kind;
    int slices;      // of K (TILE64 and TILE128)
};

static Q8Plan q8_plan(int64_t M, int64_t N, int64_t K) {
    if (M <= 32) return {Q8Plan::ROWS, 1};
    const int64_t steps = ceil_div(K, 64);
    const double t64 = (double)(ceil_div(M, 64) * ceil_div(N, 64)) / 256, t128 = (double)(ceil_div(M, 128) * ceil_div(N, 128)) / 256;
    Q8Plan best{Q8Plan::TILE64, 1};
    double least = 1e30;
    for (int s = 1; s <= 8 && (s == 1 || steps / s >= 4); s *= 2) {
        const double part = (double)ceil_div(steps, s), join = s == 1 ? 0 : 3 + (double)s * (double)M * (double)N * 8 / 4e6;
        const double a = 3.5 + 0.8 * t64 + part * std::max(0.15, 0.12 * t64 * s) + join;
        const double b = 4.5 + 1.5 * t128 + part * std::max(t128 * s > 1 ? 0.5 : 0.28, 0.3 * t128 * s) + join;
        if (a < least) least = a, best = {Q8Plan::TILE64, s};
        if (b < least) least = b, best = {Q8Plan::TILE128, s};
    }
    if (K % 128) return best;
    auto rounds = [&](int64_t tiles, double each, auto last) {      // of 256 tiles; the last may be for some of the CUs
        const double rest = (double)(tiles % 256) / 256;
        return each * (double)ceil_div(tiles, 256) + (double)steps * (last(1.0) * (double)(tiles / 256) + (rest > 0 ? last(rest) : 0));
    };
    const double tall = 5.5 + rounds(ceil_div(M, 256) * ceil_div(N, 128), 3, [](double part) { return 0.38 + 0.06 * part; });
    const double big = 5 + rounds(ceil_div(M, 256) * ceil_div(N, 256), 5, [](double part) { return 0.53 + 0.4 * std::max(0.0, part - 0.5); });
    if (tall < least) least = tall, best = {Q8Plan::TALL, 1};
    if (big < least) best = {Q8Plan::BIG, 1};
    return best;
}

template <typename T, int MI, int NB, int NS>
static void launch_tile(Q8Args& e, int slices, hipStream_t s) {
    e.tiles_m = (int)ceil_div(e.M, 32 * MI);
    e.tiles_n = (int)ceil_div(e.N, 32 * NB);
    e.steps = (int)ceil_div(ceil_div(e.K, 64), slices);
    e.slices = (int)ceil_div(ceil_div(e.K, 64), e.steps);
    hipLaunchKernelGGL((linear_q8_tile_kernel<T, MI, NB, NS>), dim3((unsigned)(e.tiles_m * e.tiles_n), (unsigned)e.slices), dim3(256), 0, s, e);
    if (e.slices > 1)
        hipLaunchKernelGGL((linear_q8_join_kernel<T>), dim3((unsigned)ceil_div((int64_t)e.M * ((e.N + 3) / 4), 256)), dim3(256), 0, s, e);
}

template <typename T, int MB>
static void launch_rows(const Q8Args& e, hipStream_t s) {
    hipLaunchKernelGGL((linear_q8_rows_kernel<T, MB>), dim3((unsigned)ceil_div(e.N, 16), (unsigned)ceil_div(e.M, 16 * MB)), dim3(512), 0, s, e);
}

template <typename T>
static int launch_linear_q8(Q8Args& e, int64_t scratch_bytes, hipStream_t s) {
    ProfScope ps(BT_PROF_LINEAR_MFMA, s);
    Q8Plan p = q8_plan(e.M, e.N, e.K);
    if (p.slices > 1 && scratch_bytes < (int64_t)p.slices * e.M * e.N * (int64_t)sizeof(int)) p.slices = 1;
    if (e.lda >= (1 << 23) || e.ldw >= (1 << 23)) p.kind = Q8Plan::ROWS;      // a tile's rows would not be within 32 bits
    BT_CHECK_ARG(p.kind != Q8Plan::ROWS || e.M < (1 << 21), "bt_linear_q8: M=%d is too many rows for codes so far apart", e.M);      // (grid.y)
    switch (p.kind) {
        case Q8Plan::ROWS:
            if (e.M <= 16) launch_rows<T, 1>(e, s);
            else launch_rows<T, 2>(e, s);
            break;
        case Q8Plan::TILE64: launch_tile<T, 2, 2, 8>(e, p.slices, s); break;
        case Q8Plan::TILE128: launch_tile<T, 4, 4, 4>(e, p.slices, s); break;
        case Q8Plan::BIG:
            e.tiles_m = (int)ceil_div(e.M, 256);
            e.tiles_n = (int)ceil_div(e.N, 256);
            hipLaunchKernelGGL((linear_q8_big_kernel<T, 4>), dim3((unsigned)std::min(e.tiles_m * e.tiles_n, 256)), dim3(512), 0, s, e);
            break;
        case Q8Plan::TALL:
            e.tiles_m = (int)ceil_div(e.M, 256);
            e.tiles_n = (int)ceil_div(e.N, 128);
            hipLaunchKernelGGL((linear_q8_big_kernel<T, 2>), dim3((unsigned)std::min(e.tiles_m * e.tiles_n, 256)), dim3(512), 0, s, e);
            break;
    }
    BT_LAUNCH_CHECK("bt_linear_q8 launch");
    return BT_OK;
}

}  // namespace bt

using namespace bt;

extern "C" int bt_quant_rows(int dtype, int64_t M, int64_t K, const void* x, int64_t ldx, const void* ln_w, const void* ln_b, float eps,
                             int8_t* codes, int64_t ldc, float* scales, bt_stream stream) {
    BT_CHECK_ARG(dtype == BT_F32 || dtype == BT_BF16, "bt_quant_rows: bad dtype %d", dtype);
    BT_CHECK_ARG(M >= 0 && M < (1ll << 31) && K > 0 && K < (1ll << 31), "bt_quant_rows: bad shape M=%lld K=%lld", (long long)M, (long long)K);
    if (M == 0) return BT_OK;      // (an empty tensor has no pointer)
    BT_CHECK_ARG(x && codes && scales, "bt_quant_rows: null pointer");
    BT_CHECK_ARG((ln_w != nullptr) == (ln_b != nullptr), "bt_quant_rows: LayerNorm needs ln_w and ln_b");
    BT_CHECK_ARG(ldx >= K || M <= 1, "bt_quant_rows: row stride smaller than row");
    BT_CHECK_ARG(ldc >= ceil_div(K, 16) * 16 && ldc % 16 == 0 && aligned16(codes),
                 "bt_quant_rows: codes need a row stride of round_up(K, 16) or more, in 16-byte units");
    if (dtype == BT_BF16)
        return launch_quant_rows<bf16>(M, K, x, ldx, ln_w, ln_b, eps, codes, ldc, scales, (hipStream_t)stream);
    return launch_quant_rows<float>(M, K, x, ldx, ln_w, ln_b, eps, codes, ldc, scales, (hipStream_t)stream);
}

extern "C" int64_t bt_linear_q8_scratch_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const Q8Plan p = q8_plan(M, N, K);
    return p.slices > 1 ? (int64_t)p.slices * M * N * (int64_t)sizeof(int) : 0;
}

extern "C" int bt_linear_q8(int dtype, int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t lda, const float* a_scale,
                            const int8_t* W, int64_t ldw, const float* w_scale, const void* bias, const void* residual, int64_t ldr,
                            void* out, int64_t ldo, int act, void* scratch, int64_t scratch_bytes, bt_stream stream) {
    BT_CHECK_ARG(dtype == BT_F32 || dtype == BT_BF16, "bt_linear_q8: bad dtype %d", dtype);
    BT_CHECK_ARG(M >= 0 && N > 0 && K > 0 && M < (1ll << 22) && N < (1ll << 22), "bt_linear_q8: bad shape M=%lld N=%lld K=%lld",
                 (long long)M, (long long)N, (long long)K);
    BT_CHECK_ARG(K % 16 == 0 && K <= 131056, "bt_linear_q8: K = %lld is not a multiple of 16 up to 131056", (long long)K);
    if (M == 0) return BT_OK;      // (an empty tensor has no pointer)
    BT_CHECK_ARG(A && W && a_scale && w_scale && out, "bt_linear_q8: null pointer");
    BT_CHECK_ARG(lda >= K && ldw >= K && lda % 16 == 0 && ldw % 16 == 0 && aligned16(A) && aligned16(W),
                 "bt_linear_q8: rows of codes must be 16-byte granular");
    BT_CHECK_ARG(ldo >= N && (!residual || ldr >= N), "bt_linear_q8: row stride smaller than row");
    BT_CHECK_ARG(ldo < (1 << 26) && ldr < (1 << 26), "bt_linear_q8: row stride too large");      // (16 rows within 32 bits)
    BT_CHECK_ARG(act == BT_ACT_NONE || act == BT_ACT_GELU, "bt_linear_q8: bad act %d", act);
    BT_CHECK_ARG(!scratch || (scratch_bytes >= 0 && aligned16(scratch)), "bt_linear_q8: scratch must be 16-byte aligned");
    Q8Args e{};
    e.A = A;
    e.W = W;
    e.lda = lda;
    e.ldw = ldw;
    e.M = (int)M;
    e.N = (int)N;
    e.K = (int)K;
    e.a_scale = a_scale;
    e.w_scale = w_scale;
    e.bias = bias;
    e.residual = residual;
    e.ldr = ldr;
    e.out = out;
    e.ldo = ldo;
    e.act = act;
    e.fours = aligned16(w_scale) && aligned16(bias);
    e.slab = (int*)scratch;
    if (!scratch) scratch_bytes = 0;
    return dtype == BT_BF16 ? launch_linear_q8<bf16>(e, scratch_bytes, (hipStream_t)stream)
                            : launch_linear_q8<float>(e, scratch_bytes, (hipStream_t)stream);
}
