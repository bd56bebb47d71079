// 8-bit integers for the linear layers: bt_quant_rows (one scale per row) and bt_linear_q8 (the product, with its epilogue).
#include "bt_common.h"
#include "bt_quant.h"

namespace bt {

// ---- bt_quant_rows ---------------------------------------------------------------------------------------------------------
// A row is read once into registers -- NV 16-byte pieces a lane, all loads in flight together -- and everything else happens there:
// LayerNorm statistics (two-pass, fp32), the largest magnitude, the codes.  R waves to a row: one where there are rows enough for
// the card (no barrier), four where there are not or where the row does not fit one wave's registers.  Bound by memory: x in, one
// byte a value out.
template <int R>
struct RowReduce {      // over the R waves of a row (R = 4: the workgroup)
    float* slot;
    int wave;
    __device__ inline float sum(float v) {
        v = wave_sum(v);
        if (R == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        return slot[0] + slot[1] + slot[2] + slot[3];
    }
    __device__ inline float max(float v) {
        v = wave_max(v);
        if (R == 1) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        return fmaxf(fmaxf(slot[0], slot[1]), fmaxf(slot[2], slot[3]));
    }
};

// values c .. c + V - 1 of a row of K (zero beyond); VEC: the row is 16-byte aligned
template <typename T, bool VEC>
__device__ inline void load_piece(const T* row, int c, int K, float (&v)[Elem<T>::VEC]) {
    constexpr int V = Elem<T>::VEC;
    if (VEC && c + V <= K) load_vec<T>(row + c, v);
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c + i < K ? Elem<T>::load(row + c + i) : 0.f;
}

template <typename T, bool LN, bool VEC, int NV, int R>
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
    for (int i = 0; i < NV; ++i) load_piece<T, VEC>(xr, (i * 64 * R + at) * V, K, v[i]);
    if (LN) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[i][e];
        const float mean = all.sum(sum) / (float)K;
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[i][e] -= mean;
                if ((i * 64 * R + at) * V + e < K) sq = fmaf(v[i][e], v[i][e], sq);
            }
        const float rstd = rsqrtf(all.sum(sq) / (float)K + eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * R + at) * V;
            float wv[V], bv[V];
            load_piece<T, VEC>(w, c, K, wv);
            load_piece<T, VEC>(b, c, K, bv);
#pragma unroll
            for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, wv[e], bv[e]);      // 0 beyond K, as wv and bv are
        }
    }
    float amax = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (LN && v[i][e] != v[i][e] && (i * 64 * R + at) * V + e >= K) v[i][e] = 0.f;      // (0 * an infinite rstd)
            amax = fmaxf(amax, fabsf(v[i][e]));
            odd |= !(fabsf(v[i][e]) < INFINITY);
        }
    amax = all.max(odd ? INFINITY : amax);
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

// Rows longer than four waves' registers: a workgroup passes over the row once for each of the steps above.
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
    const bool vec = aligned16(x) && (ldx % V == 0 || M == 1) && (!w || (aligned16(w) && aligned16(b)));
    const int64_t wave_pieces = ceil_div(K, 64 * V), group_pieces = ceil_div(K, 256 * V);
    // one wave to a row from 2048 rows (8 waves to a CU) while it has at most 8 pieces a lane
    const bool one = wave_pieces <= 8 && M >= 2048;
    const int64_t pieces = one ? wave_pieces : group_pieces;
    const dim3 grid((unsigned)(one ? ceil_div(M, 4) : M));
#define BT_QR(LN_, VEC_, NV_, R_)                                                                                                    \
    hipLaunchKernelGGL((quant_rows_kernel<T, LN_, VEC_, NV_, R_>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, \
                       codes, ldc, scales, M, (int)K)
#define BT_QR_PIECES(LN_, VEC_, R_)              \
    do {                                         \
        if (pieces <= 1) BT_QR(LN_, VEC_, 1, R_); \
        else if (pieces <= 2) BT_QR(LN_, VEC_, 2, R_); \
        else if (pieces <= 4) BT_QR(LN_, VEC_, 4, R_); \
        else BT_QR(LN_, VEC_, 8, R_);            \
    } while (0)
#define BT_QR_ROW(LN_, VEC_)                     \
    do {                                         \
        if (one) BT_QR_PIECES(LN_, VEC_, 1);     \
        else BT_QR_PIECES(LN_, VEC_, 4);         \
    } while (0)
    if (pieces > 8) {
        if (w) hipLaunchKernelGGL((quant_long_rows_kernel<T, true>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes, ldc, scales, K);
        else hipLaunchKernelGGL((quant_long_rows_kernel<T, false>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes, ldc, scales, K);
    } else if (w) {
        if (vec) BT_QR_ROW(true, true);
        else BT_QR_ROW(true, false);
    } else {
        if (vec) BT_QR_ROW(false, true);
        else BT_QR_ROW(false, false);
    }
#undef BT_QR_ROW
#undef BT_QR_PIECES
#undef BT_QR
    BT_LAUNCH_CHECK("bt_quant_rows launch");
    return BT_OK;
}

// ---- bt_linear_q8 ----------------------------------------------------------------------------------------------------------
typedef int i32x4 __attribute__((ext_vector_type(4)));

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
    int wide;           // out (and residual) take 16-byte accesses
    int tiles_m, tiles_n;
    int slices, steps;  // K split into `slices` ranges of `steps` 64-byte steps; > 1: sums go to `slab`
    int* slab;          // [slices][M][N]
};

// act(acc * sx * sw + bias): fp32; the residual joins where the row is written
__device__ inline float q8_value(int acc, float sa, float sw, float bias, int act) {
    const float y = fmaf((float)acc, sa * sw, bias);
    return act == BT_ACT_GELU ? 0.5f * y * (1.0f + erff(y * 0.70710678118654752440f)) : y;
}

template <typename T>
__device__ inline void q8_store(const Q8Args& e, int m, int n, int acc) {
    float y = q8_value(acc, e.a_scale[m], e.w_scale[n], e.bias ? Elem<T>::load((const T*)e.bias + n) : 0.f, e.act);
    if (e.residual) y += Elem<T>::load((const T*)e.residual + (int64_t)m * e.ldr + n);
    Elem<T>::store((T*)e.out + (int64_t)m * e.ldo + n, y);
}

// Any K % 16 == 0: 64 x 64 tile per workgroup, 64 bytes of K at a time through LDS, four products per v_dot4.
template <typename T>
__global__ __launch_bounds__(256) void linear_q8_dot_kernel(Q8Args e) {
    __shared__ int4 sa[64][5], sw[64][5];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    const int r = threadIdx.x >> 2, c = threadIdx.x & 3;
    const int tm = (threadIdx.x >> 4) * 4, tn = (threadIdx.x & 15) * 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < e.K; k0 += 64) {
        const int k = k0 + c * 16;
        int4 a{0, 0, 0, 0}, w{0, 0, 0, 0};
        if (k < e.K && m0 + r < e.M) a = *(const int4*)(e.A + (m0 + r) * e.lda + k);
        if (k < e.K && n0 + r < e.N) w = *(const int4*)(e.W + (n0 + r) * e.ldw + k);
        __syncthreads();
        sa[r][c] = a;
        sw[r][c] = w;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            int4 av[4], wv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                av[i] = sa[tm + i][q];
                wv[i] = sw[tn + i][q];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = __builtin_amdgcn_sdot4(av[i].x, wv[j].x, acc[i][j], false);
                    acc[i][j] = __builtin_amdgcn_sdot4(av[i].y, wv[j].y, acc[i][j], false);
                    acc[i][j] = __builtin_amdgcn_sdot4(av[i].z, wv[j].z, acc[i][j], false);
                    acc[i][j] = __builtin_amdgcn_sdot4(av[i].w, wv[j].w, acc[i][j], false);
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m0 + tm + i < e.M && n0 + tn + j < e.N) q8_store<T>(e, m0 + tm + i, n0 + tn + j, acc[i][j]);
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

// The tile kernel: 32 MI x 32 NB per workgroup of 2 x 2 waves, 64 bytes of K a step, K % 64 == 0.
//  * Two workgroups to a CU: while one waits at its barrier or writes its tile, the other's waves have the matrix units.  So a K step
//    needs one barrier and the epilogue no software overlap.
//  * A and W travel global -> LDS without registers, NS - 1 steps ahead, in a ring of NS stages.  A wave waits for its own loads of step t
//    (in order: at most those of the younger steps stay out), then for the others at the barrier; behind it everybody has also consumed
//    step t - 1, whose stage takes the loads of step t + NS - 1.
//  * LDS rows are 64 bytes; the four 16-byte pieces of row r are stored in the order p ^ ((r >> 1) & 3) ^ ((r >> 3) & 1): the 16 rows that
//    a fragment read touches at once are spread over all banks.
//  * mfma(W, A): a lane gets four neighbouring columns of one row; rows are put together in LDS and leave as 16-byte pieces.
template <typename T, int MI, int NB, int NS>
__global__ __launch_bounds__(256, 2) void linear_q8_tile_kernel(Q8Args e) {
    constexpr int BM = 32 * MI, BN = 32 * NB, STAGE = (BM + BN) * 64;
    constexpr int LA = BM / 64, LW = BN / 64, LOADS = LA + LW;      // 1 KiB loads of a wave and step
    constexpr int PITCH = 16 * NB * sizeof(T) + 16;                 // a row of the wave's patch: its 16 NB columns
    constexpr int RING = NS * STAGE, PATCH = 4 * 16 * PITCH;
    __shared__ __attribute__((aligned(16))) char smem[RING > PATCH ? RING : PATCH];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, c = lane & 15, g = lane >> 4;

    // workgroups of one XCD (ids that are equal mod 8) take neighbouring tiles, in columns of 8 tile rows: its L2 serves them with each
    // other's panels
    const int tiles = e.tiles_m * e.tiles_n, id = blockIdx.x;
    const int per = tiles >> 3, rest = tiles & 7, xcd = id & 7, local = id >> 3;
    const int at = (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + local;
    const int group = at / (8 * e.tiles_n), first = group * 8, high = min(e.tiles_m - first, 8), in = at - group * 8 * e.tiles_n;
    const int m0 = (first + in % high) * BM, n0 = (in / high) * BN;

    const int k0 = blockIdx.y * e.steps * 64, steps = min(e.steps, (e.K - k0) >> 6);
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
    const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)smem;
    auto load = [&](int t) {
        const uint32_t stage = ring + (t % NS) * STAGE;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            if (i < LA) dma16(A + (int64_t)t * 64, off[i], stage + (wave * LA + i) * 1024);
            else dma16(W + (int64_t)t * 64, off[i], stage + BM * 64 + (wave * LW + i - LA) * 1024);
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
    int stage = 0;
    for (int t = 0; t < steps; ++t) {
        if (t + NS - 2 < steps) wait_loads<LOADS * (NS - 2)>();
        else if (NS > 3 && t + 1 < steps) wait_loads<LOADS>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (t + NS - 1 < steps) load(t + NS - 1);
        const char* a = smem + stage * STAGE + wm * MI * 1024 + frag;
        const char* w = smem + stage * STAGE + BM * 64 + wn * NB * 1024 + frag;
        i32x4 af[MI], wf[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) wf[j] = *(const i32x4*)(w + j * 1024);
#pragma unroll
        for (int i = 0; i < MI; ++i) af[i] = *(const i32x4*)(a + i * 1024);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], af[i], acc[i][j], 0, 0, 0);
        stage = stage + 1 == NS ? 0 : stage + 1;
    }

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
                if (n + 4 <= e.N && (e.N & 3) == 0) *(i32x4*)(slab + (int64_t)m * e.N + n) = acc[i][j];
                else
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < e.N) slab[(int64_t)m * e.N + n + r] = acc[i][j][r];
            }
        }
        return;
    }
    float sw[NB][4], bias[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int n = n_w + j * 16 + g * 4 + r < e.N ? n_w + j * 16 + g * 4 + r : e.N - 1;
            sw[j][r] = e.w_scale[n];
            bias[j][r] = e.bias ? Elem<T>::load((const T*)e.bias + n) : 0.f;
        }
    __syncthreads();      // the ring is the patches' now
    char* patch = smem + wave * 16 * PITCH;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = m_w + i * 16 + c;
        const float sa = e.a_scale[m < e.M ? m : e.M - 1];
        float res[NB][4] = {};      // joins before the one rounding
        if (e.residual && m < e.M) {
            const T* p = (const T*)e.residual + (int64_t)m * e.ldr + n_w + g * 4;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int n = n_w + j * 16 + g * 4;
                if (e.wide && n + 4 <= e.N) {
                    if constexpr (sizeof(T) == 2) {
                        const uint2 u = *(const uint2*)(p + j * 16);
                        res[j][0] = __uint_as_float(u.x << 16), res[j][1] = __uint_as_float(u.x & 0xffff0000u);
                        res[j][2] = __uint_as_float(u.y << 16), res[j][3] = __uint_as_float(u.y & 0xffff0000u);
                    } else {
                        const float4 u = *(const float4*)(p + j * 16);
                        res[j][0] = u.x, res[j][1] = u.y, res[j][2] = u.z, res[j][3] = u.w;
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < e.N) res[j][r] = Elem<T>::load(p + j * 16 + r);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) y[r] = q8_value(acc[i][j][r], sa, sw[j][r], bias[j][r], e.act) + res[j][r];
            if constexpr (sizeof(T) == 2) *(uint2*)(patch + c * PITCH + (j * 16 + g * 4) * 2) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
            else *(float4*)(patch + c * PITCH + (j * 16 + g * 4) * 4) = float4{y[0], y[1], y[2], y[3]};
        }
        asm volatile("" ::: "memory");      // the patch is the wave's own, and a wave's LDS accesses stay in order
        constexpr int V = Elem<T>::VEC, CH = 16 * NB / V;      // 16-byte pieces of a row
#pragma unroll
        for (int x = 0; x < 16 * CH; x += 64) {
            const int r = (x + lane) / CH, d = ((x + lane) - r * CH) * V, mm = m_w + i * 16 + r, n = n_w + d;
            if (mm >= e.M || n >= e.N) continue;
            float y[V];
            load_vec<T>((const T*)(patch + r * PITCH) + d, y);
            T* out = (T*)e.out + (int64_t)mm * e.ldo + n;
            if (e.wide && n + V <= e.N) store_vec<T>(out, y);
            else
#pragma unroll
                for (int q = 0; q < V; ++q)
                    if (n + q < e.N) Elem<T>::store(out + q, y[q]);
        }
        asm volatile("" ::: "memory");
    }
}

template <typename T, int MI, int NB, int NS>
static void launch_tile(Q8Args& e, hipStream_t s) {
    e.tiles_m = (int)ceil_div(e.M, 32 * MI);
    e.tiles_n = (int)ceil_div(e.N, 32 * NB);
    e.slices = 1;
    e.steps = e.K / 64;
    hipLaunchKernelGGL((linear_q8_tile_kernel<T, MI, NB, NS>), dim3((unsigned)(e.tiles_m * e.tiles_n), 1), dim3(256), 0, s, e);
}

template <typename T>
static int launch_linear_q8(Q8Args& e, hipStream_t s) {
    ProfScope ps(BT_PROF_LINEAR_MFMA, s);
    if (e.K % 64 == 0 && e.lda < (1 << 23) && e.ldw < (1 << 23)) {
        const int64_t big = ceil_div(e.M, 256) * ceil_div(e.N, 128);
        if (big >= 512) launch_tile<T, 8, 4, 3>(e, s);
        else if (ceil_div(e.M, 128) * ceil_div(e.N, 128) >= 256) launch_tile<T, 4, 4, 4>(e, s);
        else launch_tile<T, 2, 2, 4>(e, s);
    } else
        hipLaunchKernelGGL((linear_q8_dot_kernel<T>), dim3((unsigned)ceil_div(e.N, 64), (unsigned)ceil_div(e.M, 64)), dim3(256), 0, s, e);
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
    (void)M; (void)N; (void)K;
    return 0;
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
    const int V = dtype == BT_BF16 ? 8 : 4;
    e.wide = aligned16(out) && ldo % V == 0 && (!residual || (aligned16(residual) && ldr % V == 0));
    return dtype == BT_BF16 ? launch_linear_q8<bf16>(e, (hipStream_t)stream) : launch_linear_q8<float>(e, (hipStream_t)stream);
}
