// 8-bit integers for the linear layers: bt_quant_rows (one scale per row) and bt_linear_q8 (the product, with its epilogue).
#include "bt_common.h"
#include "bt_quant.h"

namespace bt {

// ---- bt_quant_rows ---------------------------------------------------------------------------------------------------------
// One wave per row, 4 rows per workgroup: LayerNorm statistics (two-pass, as bt_layernorm), the largest magnitude, the codes.
template <typename T, bool LN>
__global__ __launch_bounds__(256) void quant_rows_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w,
                                                        const T* __restrict__ b, float eps, int8_t* __restrict__ codes, int64_t ldc,
                                                        float* __restrict__ scales, int64_t M, int64_t K) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    const T* xr = x + row * ldx;
    float mean = 0.f, rstd = 1.f;
    if (LN) {
        float sum = 0.f;
        for (int64_t c = lane; c < K; c += 64) sum += Elem<T>::load(xr + c);
        mean = wave_sum(sum) / (float)K;
        float sq = 0.f;
        for (int64_t c = lane; c < K; c += 64) {
            const float d = Elem<T>::load(xr + c) - mean;
            sq = fmaf(d, d, sq);
        }
        rstd = rsqrtf(wave_sum(sq) / (float)K + eps);
    }
    float amax = 0.f;
    bool bad = false;
    for (int64_t c = lane; c < K; c += 64) {
        float v = Elem<T>::load(xr + c);
        if (LN) v = fmaf((v - mean) * rstd, Elem<T>::load(w + c), Elem<T>::load(b + c));
        amax = fmaxf(amax, fabsf(v));
        bad |= !(fabsf(v) < INFINITY);
    }
    amax = wave_max(amax);
    bad = __any(bad);
    const Quantiser q(bad ? 0.f : amax);
    if (lane == 0) scales[row] = bad ? __int_as_float(0x7fc00000) : q.scale;
    int8_t* cr = codes + row * ldc;
    const int64_t Kp = (K + 15) / 16 * 16;
    for (int64_t c = lane; c < Kp; c += 64) {
        int code = 0;
        if (c < K && !bad) {
            float v = Elem<T>::load(xr + c);
            if (LN) v = fmaf((v - mean) * rstd, Elem<T>::load(w + c), Elem<T>::load(b + c));
            code = q.code(v);
        }
        cr[c] = (int8_t)code;
    }
}

template <typename T>
static int launch_quant_rows(int64_t M, int64_t K, const void* x, int64_t ldx, const void* w, const void* b, float eps, int8_t* codes,
                             int64_t ldc, float* scales, hipStream_t s) {
    ProfScope ps(BT_PROF_LAYERNORM, s);
    const dim3 grid((unsigned)ceil_div(M, 4));
    if (w)
        hipLaunchKernelGGL((quant_rows_kernel<T, true>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes,
                           ldc, scales, M, K);
    else
        hipLaunchKernelGGL((quant_rows_kernel<T, false>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)w, (const T*)b, eps, codes,
                           ldc, scales, M, K);
    BT_LAUNCH_CHECK("bt_quant_rows launch");
    return BT_OK;
}

// ---- bt_linear_q8 ----------------------------------------------------------------------------------------------------------
struct Q8Epi {
    const float* a_scale;
    const float* w_scale;
    const void* bias;
    const void* residual;
    int64_t ldr;
    void* out;
    int64_t ldo;
    int act;
};

template <typename T>
__device__ inline void q8_store(const Q8Epi& e, int64_t m, int64_t n, int acc) {
    float y = (float)acc * (e.a_scale[m] * e.w_scale[n]);
    if (e.bias) y += Elem<T>::load((const T*)e.bias + n);
    if (e.act == BT_ACT_GELU) y = 0.5f * y * (1.0f + erff(y * 0.70710678118654752440f));
    if (e.residual) y += Elem<T>::load((const T*)e.residual + m * e.ldr + n);
    Elem<T>::store((T*)e.out + m * e.ldo + n, y);
}

// 64 x 64 tile per workgroup, 64 bytes of K at a time through LDS, four products per v_dot4.
template <typename T>
__global__ __launch_bounds__(256) void linear_q8_kernel(const int8_t* __restrict__ A, int64_t lda, const int8_t* __restrict__ W,
                                                       int64_t ldw, int64_t M, int64_t N, int64_t K, Q8Epi e) {
    __shared__ int4 sa[64][5], sw[64][5];
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int r = threadIdx.x >> 2, c = threadIdx.x & 3;
    const int tm = (threadIdx.x >> 4) * 4, tn = (threadIdx.x & 15) * 4;
    int acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 64) {
        const int64_t k = k0 + c * 16;
        int4 a{0, 0, 0, 0}, w{0, 0, 0, 0};
        if (k < K && m0 + r < M) a = *(const int4*)(A + (m0 + r) * lda + k);
        if (k < K && n0 + r < N) w = *(const int4*)(W + (n0 + r) * ldw + k);
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
            if (m0 + tm + i < M && n0 + tn + j < N) q8_store<T>(e, m0 + tm + i, n0 + tn + j, acc[i][j]);
}

template <typename T>
static int launch_linear_q8(int64_t M, int64_t N, int64_t K, const int8_t* A, int64_t lda, const int8_t* W, int64_t ldw, const Q8Epi& e,
                            hipStream_t s) {
    ProfScope ps(BT_PROF_LINEAR_MFMA, s);
    hipLaunchKernelGGL((linear_q8_kernel<T>), dim3((unsigned)ceil_div(N, 64), (unsigned)ceil_div(M, 64)), dim3(256), 0, s, A, lda, W, ldw,
                       M, N, K, e);
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
    BT_CHECK_ARG(M >= 0 && N > 0 && K > 0 && M < (1ll << 22) && N < (1ll << 31), "bt_linear_q8: bad shape M=%lld N=%lld K=%lld",
                 (long long)M, (long long)N, (long long)K);
    BT_CHECK_ARG(K % 16 == 0 && K <= 131056, "bt_linear_q8: K = %lld is not a multiple of 16 up to 131056", (long long)K);
    if (M == 0) return BT_OK;      // (an empty tensor has no pointer)
    BT_CHECK_ARG(A && W && a_scale && w_scale && out, "bt_linear_q8: null pointer");
    BT_CHECK_ARG(lda >= K && ldw >= K && lda % 16 == 0 && ldw % 16 == 0 && aligned16(A) && aligned16(W),
                 "bt_linear_q8: rows of codes must be 16-byte granular");
    BT_CHECK_ARG(ldo >= N && (!residual || ldr >= N), "bt_linear_q8: row stride smaller than row");
    BT_CHECK_ARG(act == BT_ACT_NONE || act == BT_ACT_GELU, "bt_linear_q8: bad act %d", act);
    BT_CHECK_ARG(!scratch || (scratch_bytes >= 0 && aligned16(scratch)), "bt_linear_q8: scratch must be 16-byte aligned");
    const Q8Epi e{a_scale, w_scale, bias, residual, ldr, out, ldo, act};
    if (dtype == BT_BF16) return launch_linear_q8<bf16>(M, N, K, A, lda, W, ldw, e, (hipStream_t)stream);
    return launch_linear_q8<float>(M, N, K, A, lda, W, ldw, e, (hipStream_t)stream);
}
