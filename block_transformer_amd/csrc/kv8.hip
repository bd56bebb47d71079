// A KV cache in 8 bits with one scale per block of rows and head (layout and rules: bt_kv8_cache in bt_hip.h): append with RoPE, read
// back, and attention over it.
#include "bt_common.h"
#include "bt_quant.h"

namespace bt {

struct Rows {      // bt_kv8_rows on the device
    char* p;
    int64_t b, t, h;
};

// ---- bt_kv8_append ---------------------------------------------------------------------------------------------------------
struct AppendArgs {
    bt_kv8_cache c;
    Rows q, q_out, k, v;
    int64_t kv_items;      // waves for keys and values: batch * kv_heads * blocks
    int blocks;            // blocks that q_len rows can touch
    int q_len, heads, rot, pos0_host, shift;
    const int32_t* pos0_dev;
    const int32_t* pos_table;
    const float* cos_tab;
    const float* sin_tab;
    int64_t max_pos;
};

template <typename T>
__device__ inline float rotated(const T* row, int e, int rot, int64_t angle, const float* cos_tab, const float* sin_tab) {
    const float x = Elem<T>::load(row + e);
    const int half = rot >> 1;
    if (e >= 2 * half) return x;
    const int j = e < half ? e : e - half;
    const double c = cos_tab[angle * half + j], s = sin_tab[angle * half + j];
    const double o = Elem<T>::load(row + (e < half ? e + half : e - half));
    return (float)(e < half ? (double)x * c - o * s : (double)x * c + o * s);
}

__device__ inline int64_t angle_of(const AppendArgs& a, int pos) {
    int64_t r = a.pos_table ? a.pos_table[pos] : pos;
    r = r < 0 ? 0 : r;
    return r < a.max_pos ? r : a.max_pos - 1;
}

// One wave per (sequence, head, block) that the new rows touch; the waves behind them rotate q, one (row, head) each.
template <typename T>
__global__ __launch_bounds__(64) void kv8_append_kernel(AppendArgs a) {
    const int D = a.c.head_dim, bl = a.c.block, lane = threadIdx.x;
    const int pos0 = a.pos0_dev ? *a.pos0_dev : a.pos0_host;
    if (pos0 < 0) return;
    if (blockIdx.x >= a.kv_items) {
        const int64_t i = blockIdx.x - a.kv_items;
        const int64_t b = i / ((int64_t)a.q_len * a.heads);
        const int th = (int)(i - b * a.q_len * a.heads), t = th / a.heads, h = th - t * a.heads;
        const T* src = (const T*)a.q.p + b * a.q.b + t * a.q.t + h * a.q.h;
        T* dst = (T*)a.q_out.p + b * a.q_out.b + t * a.q_out.t + h * a.q_out.h;
        const int64_t ang = angle_of(a, pos0 + t);
        float y[2];
        for (int i2 = 0; i2 < 2; ++i2)
            if (lane + 64 * i2 < D) y[i2] = rotated<T>(src, lane + 64 * i2, a.rot, ang, a.cos_tab, a.sin_tab);
        __syncthreads();
        for (int i2 = 0; i2 < 2; ++i2)
            if (lane + 64 * i2 < D) Elem<T>::store(dst + lane + 64 * i2, y[i2]);
        return;
    }
    const int64_t bh = blockIdx.x / a.blocks;
    const int item = (int)(blockIdx.x - bh * a.blocks);
    const int64_t b = bh / a.c.kv_heads;
    const int h = (int)(bh - b * a.c.kv_heads);
    const int64_t end = pos0 + (int64_t)a.q_len < a.c.n_max ? pos0 + (int64_t)a.q_len : a.c.n_max;
    const int first = pos0 >> a.shift;
    const T* ksrc = (const T*)a.k.p + b * a.k.b + h * a.k.h;
    const T* vsrc = (const T*)a.v.p + b * a.v.b + h * a.v.h;
    T* kt = (T*)a.c.k_tail + bh * bl * D;
    T* vt = (T*)a.c.v_tail + bh * bl * D;
    const int64_t n_blk = a.c.n_max >> a.shift;
    const int last = (int)(end >> a.shift);      // the block that stays open
    // the open block's rows take the places that the first block's old rows leave: the same wave does both, in that order
    for (int pass = 0; pass < 2; ++pass) {
        const int blk = pass == 0 ? first + item : last;
        if (pass == 1 && (item != 0 || last == first)) return;
        if (pass == 0 && blk > first && blk >= last) return;
        const int64_t row0 = (int64_t)blk * bl;
        if (row0 >= end) continue;
        if (row0 + bl <= end) {
            float ka = 0.f, va = 0.f;
            for (int e = lane; e < bl * D; e += 64) {
                const int t = e / D, d = e - t * D;
                const int64_t at = row0 + t - pos0;
                const float k = at < 0 ? Elem<T>::load(kt + t * D + d)
                                       : rotated<T>(ksrc + at * a.k.t, d, a.rot, angle_of(a, pos0 + (int)at), a.cos_tab, a.sin_tab);
                const float v = at < 0 ? Elem<T>::load(vt + d * bl + t) : Elem<T>::load(vsrc + at * a.v.t + d);
                T kr;
                Elem<T>::store(&kr, k);
                const float kf = Elem<T>::load(&kr);
                if (fabsf(kf) < INFINITY) ka = fmaxf(ka, fabsf(kf));
                if (fabsf(v) < INFINITY) va = fmaxf(va, fabsf(v));
            }
            const Quantiser qk(wave_max(ka)), qv(wave_max(va));
            if (lane == 0) {
                a.c.k_scale[bh * n_blk + blk] = qk.scale;
                a.c.v_scale[bh * n_blk + blk] = qv.scale;
            }
            for (int e = lane; e < bl * D; e += 64) {
                const int t = e / D, d = e - t * D;
                const int64_t at = row0 + t - pos0;
                const float k = at < 0 ? Elem<T>::load(kt + t * D + d)
                                       : rotated<T>(ksrc + at * a.k.t, d, a.rot, angle_of(a, pos0 + (int)at), a.cos_tab, a.sin_tab);
                const float v = at < 0 ? Elem<T>::load(vt + d * bl + t) : Elem<T>::load(vsrc + at * a.v.t + d);
                T kr;
                Elem<T>::store(&kr, k);
                a.c.k_codes[(bh * a.c.n_max + row0 + t) * D + d] = (int8_t)qk.code(Elem<T>::load(&kr));
                a.c.v_codes[((bh * n_blk + blk) * D + d) * bl + t] = (int8_t)qv.code(v);
            }
        } else {
            for (int e = lane; e < bl * D; e += 64) {
                const int t = e / D, d = e - t * D;
                const int64_t at = row0 + t - pos0;
                if (at < 0 || row0 + t >= end) continue;
                Elem<T>::store(kt + t * D + d, rotated<T>(ksrc + at * a.k.t, d, a.rot, angle_of(a, pos0 + (int)at), a.cos_tab, a.sin_tab));
                Elem<T>::store(vt + d * bl + t, Elem<T>::load(vsrc + at * a.v.t + d));
            }
        }
    }
}

// ---- bt_kv8_read -----------------------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void kv8_read_kernel(bt_kv8_cache c, int shift, int64_t n, int64_t first, int64_t count,
                                                      T* __restrict__ ko, T* __restrict__ vo) {
    const int D = c.head_dim, bl = c.block;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= c.batch * c.kv_heads * count * D) return;
    const int d = (int)(i % D);
    const int64_t bh = i / D / count, row = first + i / D - bh * count;
    const int64_t blk = row >> shift, n_blk = c.n_max >> shift;
    const int t = (int)(row & (bl - 1));
    if (blk < n >> shift) {
        if (ko) Elem<T>::store(ko + i, (float)c.k_codes[(bh * c.n_max + row) * D + d] * c.k_scale[bh * n_blk + blk]);
        if (vo) Elem<T>::store(vo + i, (float)c.v_codes[((bh * n_blk + blk) * D + d) * bl + t] * c.v_scale[bh * n_blk + blk]);
    } else {
        if (ko) ko[i] = ((const T*)c.k_tail)[(bh * bl + t) * D + d];
        if (vo) vo[i] = ((const T*)c.v_tail)[(bh * D + d) * bl + t];
    }
}

// ---- bt_attention_kv8 ------------------------------------------------------------------------------------------------------
struct AttnArgs {
    bt_kv8_cache c;
    Rows q;
    int q_len, heads, pos0_host, shift;
    const int32_t* pos0_dev;
    const uint8_t* mask;
    int64_t mask_ld;
    void* out;
    int64_t ldo;
    float scale;      // log2(e) / sqrt(head_dim)
};

// One wave per (sequence, row, head): a lane scores one cached row of 64, then owns head_dim / 64 columns of the output.
template <typename T>
__global__ __launch_bounds__(64) void attention_kv8_kernel(AttnArgs a) {
    __shared__ float qs[128], ps[64];
    const int D = a.c.head_dim, bl = a.c.block, lane = threadIdx.x;
    const int64_t i = blockIdx.x;
    const int h = (int)(i % a.heads);
    const int64_t row = i / a.heads;
    const int64_t b = row / a.q_len;
    const int t = (int)(row - b * a.q_len);
    const int pos0 = a.pos0_dev ? *a.pos0_dev : a.pos0_host;
    const int64_t n = pos0 + (int64_t)a.q_len < a.c.n_max ? pos0 + (int64_t)a.q_len : a.c.n_max;
    const int64_t lim = pos0 + t + 1 < n ? pos0 + t + 1 : n;
    const int64_t bh = b * a.c.kv_heads + h / (a.heads / a.c.kv_heads);
    const int64_t n_blk = a.c.n_max >> a.shift, full = n >> a.shift;
    const T* q = (const T*)a.q.p + b * a.q.b + t * a.q.t + h * a.q.h;
    for (int d = lane; d < D; d += 64) qs[d] = Elem<T>::load(q + d);
    float m = -1e30f, l = 0.f, o[2] = {0.f, 0.f};
    for (int64_t j0 = 0; j0 < lim; j0 += 64) {
        const int64_t j = j0 + lane;
        const bool on = j < lim && !(a.mask && a.mask[b * a.mask_ld + j] == 0);
        float s = -INFINITY;
        __syncthreads();
        if (on) {
            const int64_t blk = j >> a.shift;
            s = 0.f;
            if (blk < full) {
                const int8_t* k = a.c.k_codes + (bh * a.c.n_max + j) * D;
                for (int d = 0; d < D; ++d) s = fmaf(qs[d], (float)k[d], s);
                s *= a.c.k_scale[bh * n_blk + blk];
            } else {
                const T* k = (const T*)a.c.k_tail + (bh * bl + (j & (bl - 1))) * D;
                for (int d = 0; d < D; ++d) s = fmaf(qs[d], Elem<T>::load(k + d), s);
            }
            s *= a.scale;
        }
        const bool nan = __any(s != s);
        const float mn = fmaxf(m, wave_max(s));
        const float p = nan ? __int_as_float(0x7fc00000) : __builtin_amdgcn_exp2f(s - mn), al = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l = l * al + p;
        ps[lane] = p;
        __syncthreads();
        for (int i2 = 0; i2 < 2; ++i2) {
            const int d = lane + 64 * i2;
            if (d >= D) break;
            float acc = o[i2] * al;
            for (int jj = 0; jj < 64 && j0 + jj < lim; ++jj) {
                const float pj = ps[jj];
                if (pj == 0.f) continue;
                const int64_t blk = (j0 + jj) >> a.shift;
                const int tt = (int)((j0 + jj) & (bl - 1));
                const float v = blk < full ? (float)a.c.v_codes[((bh * n_blk + blk) * D + d) * bl + tt] * a.c.v_scale[bh * n_blk + blk]
                                           : Elem<T>::load((const T*)a.c.v_tail + (bh * D + d) * bl + tt);
                acc = fmaf(pj, v, acc);
            }
            o[i2] = acc;
        }
    }
    l = wave_sum(l);
    for (int i2 = 0; i2 < 2; ++i2)
        if (lane + 64 * i2 < D) Elem<T>::store((T*)a.out + row * a.ldo + h * D + lane + 64 * i2, l == 0.f ? 0.f : o[i2] / l);
}

static int check_cache(const char* who, int dtype, const bt_kv8_cache* c, int* shift) {
    BT_CHECK_ARG(dtype == BT_F32 || dtype == BT_BF16, "%s: bad dtype %d", who, dtype);
    BT_CHECK_ARG(c, "%s: null cache", who);
    BT_CHECK_ARG(c->struct_size == sizeof(bt_kv8_cache), "%s: bt_kv8_cache.struct_size %u, this library expects %zu", who, c->struct_size,
                 sizeof(bt_kv8_cache));
    BT_CHECK_ARG(c->block == 16 || c->block == 32 || c->block == 64, "%s: block %d is not 16, 32 or 64", who, c->block);
    BT_CHECK_ARG(c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d not instantiated", who, c->head_dim);
    BT_CHECK_ARG(c->batch >= 0 && c->kv_heads > 0 && c->batch * c->kv_heads < (1ll << 31), "%s: bad batch or kv_heads", who);
    BT_CHECK_ARG(c->n_max > 0 && c->n_max % c->block == 0 && c->n_max < (1ll << 30), "%s: n_max %lld is not a multiple of the block", who,
                 (long long)c->n_max);
    *shift = c->block == 16 ? 4 : c->block == 32 ? 5 : 6;
    if (c->batch == 0) return BT_OK;      // (an empty tensor has no pointer)
    BT_CHECK_ARG(c->k_codes && c->v_codes && c->k_scale && c->v_scale && c->k_tail && c->v_tail, "%s: null cache pointer", who);
    BT_CHECK_ARG(aligned16(c->k_codes) && aligned16(c->v_codes) && aligned16(c->k_tail) && aligned16(c->v_tail),
                 "%s: cache pointers must be 16-byte aligned", who);
    return BT_OK;
}

static int check_rows(const char* who, const char* name, int dtype, const bt_kv8_rows* r) {
    BT_CHECK_ARG(r && r->p, "%s: null %s", who, name);
    const int V = dtype == BT_BF16 ? 8 : 4;
    BT_CHECK_ARG(aligned16(r->p) && r->b_stride % V == 0 && r->t_stride % V == 0 && r->h_stride % V == 0,
                 "%s: %s must be 16-byte granular", who, name);
    return BT_OK;
}

static Rows rows_of(const bt_kv8_rows* r) { return r ? Rows{(char*)r->p, r->b_stride, r->t_stride, r->h_stride} : Rows{nullptr, 0, 0, 0}; }

}  // namespace bt

using namespace bt;

extern "C" int bt_kv8_append(int dtype, const bt_kv8_cache* cache, int32_t q_len, int32_t heads, const bt_kv8_rows* q,
                             const bt_kv8_rows* q_out, const bt_kv8_rows* k, const bt_kv8_rows* v, const int32_t* pos0_dev,
                             int32_t pos0_host, const int32_t* pos_table, int32_t rot, const float* cos_tab, const float* sin_tab,
                             int64_t max_pos, bt_stream stream) {
    AppendArgs a{};
    BT_TRY(check_cache("bt_kv8_append", dtype, cache, &a.shift));
    BT_CHECK_ARG(q_len > 0, "bt_kv8_append: bad q_len %d", q_len);
    if (cache->batch == 0) return BT_OK;
    BT_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= cache->head_dim, "bt_kv8_append: bad rotary_ndims %d", rot);
    BT_CHECK_ARG(rot == 0 || (cos_tab && sin_tab && max_pos > 0), "bt_kv8_append: rotation needs cos and sin tables");
    BT_CHECK_ARG(rot > 0 || !q, "bt_kv8_append: q given, but nothing to rotate it by");
    BT_CHECK_ARG(!q == !q_out && (!q || heads > 0), "bt_kv8_append: q needs q_out and heads");
    if (q) {
        BT_TRY(check_rows("bt_kv8_append", "q", dtype, q));
        BT_TRY(check_rows("bt_kv8_append", "q_out", dtype, q_out));
    }
    BT_TRY(check_rows("bt_kv8_append", "k", dtype, k));
    BT_TRY(check_rows("bt_kv8_append", "v", dtype, v));
    BT_CHECK_ARG(pos0_dev || (pos0_host >= 0 && (int64_t)pos0_host + q_len <= cache->n_max), "bt_kv8_append: cache overflow");
    BT_CHECK_ARG(pos0_dev || pos_table || rot == 0 || (int64_t)pos0_host + q_len <= max_pos, "bt_kv8_append: positions beyond the tables");
    a.c = *cache;
    a.q = rows_of(q);
    a.q_out = rows_of(q_out);
    a.k = rows_of(k);
    a.v = rows_of(v);
    a.blocks = pos0_dev ? (q_len + cache->block - 2) / cache->block + 1
                        : (int)(((int64_t)pos0_host + q_len - 1) / cache->block - pos0_host / cache->block) + 1;
    a.kv_items = cache->batch * cache->kv_heads * a.blocks;
    a.q_len = q_len;
    a.heads = heads;
    a.rot = rot;
    a.pos0_host = pos0_host;
    a.pos0_dev = pos0_dev;
    a.pos_table = pos_table;
    a.cos_tab = cos_tab;
    a.sin_tab = sin_tab;
    a.max_pos = max_pos;
    const int64_t grid = a.kv_items + (q ? cache->batch * q_len * heads : 0);
    BT_CHECK_ARG(grid < (1ll << 31), "bt_kv8_append: grid too large");
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ROPE, s);
    if (dtype == BT_BF16)
        hipLaunchKernelGGL(kv8_append_kernel<bf16>, dim3((unsigned)grid), dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL(kv8_append_kernel<float>, dim3((unsigned)grid), dim3(64), 0, s, a);
    BT_LAUNCH_CHECK("bt_kv8_append launch");
    return BT_OK;
}

extern "C" int bt_kv8_read(int dtype, const bt_kv8_cache* cache, int64_t n, int64_t first, int64_t count, void* k_out, void* v_out,
                           bt_stream stream) {
    int shift;
    BT_TRY(check_cache("bt_kv8_read", dtype, cache, &shift));
    BT_CHECK_ARG(n >= 0 && n <= cache->n_max && first >= 0 && count >= 0 && first + count <= n, "bt_kv8_read: rows out of range");
    BT_CHECK_ARG((!k_out || aligned16(k_out)) && (!v_out || aligned16(v_out)), "bt_kv8_read: outputs must be 16-byte aligned");
    if (cache->batch == 0 || count == 0 || (!k_out && !v_out)) return BT_OK;
    const int64_t grid = ceil_div(cache->batch * cache->kv_heads * count * cache->head_dim, 256);
    BT_CHECK_ARG(grid < (1ll << 31), "bt_kv8_read: grid too large");
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ROPE, s);
    if (dtype == BT_BF16)
        hipLaunchKernelGGL(kv8_read_kernel<bf16>, dim3((unsigned)grid), dim3(256), 0, s, *cache, shift, n, first, count, (bf16*)k_out,
                           (bf16*)v_out);
    else
        hipLaunchKernelGGL(kv8_read_kernel<float>, dim3((unsigned)grid), dim3(256), 0, s, *cache, shift, n, first, count, (float*)k_out,
                           (float*)v_out);
    BT_LAUNCH_CHECK("bt_kv8_read launch");
    return BT_OK;
}

extern "C" int32_t bt_attention_kv8_split_count(int64_t batch, int32_t kv_heads, int32_t group, int32_t q_len, int64_t n) {
    (void)batch; (void)kv_heads; (void)group; (void)q_len; (void)n;
    return 1;
}

extern "C" int64_t bt_attention_kv8_workspace_bytes(int64_t batch, int32_t q_len, int32_t heads, int32_t head_dim, int32_t n_split) {
    return n_split <= 1 ? 0 : batch * q_len * heads * n_split * (head_dim + 2) * (int64_t)sizeof(float);
}

extern "C" int bt_attention_kv8(int dtype, const bt_kv8_cache* cache, int32_t q_len, int32_t heads, const bt_kv8_rows* q,
                                const int32_t* pos0_dev, int32_t pos0_host, const uint8_t* mask, int64_t mask_ld, void* out, int64_t ldo,
                                int32_t n_split, void* ws, int64_t ws_bytes, bt_stream stream) {
    AttnArgs a{};
    BT_TRY(check_cache("bt_attention_kv8", dtype, cache, &a.shift));
    BT_CHECK_ARG(q_len > 0, "bt_attention_kv8: bad q_len %d", q_len);
    BT_CHECK_ARG(heads > 0 && heads % cache->kv_heads == 0, "bt_attention_kv8: %d heads cannot share %d", heads, cache->kv_heads);
    if (cache->batch == 0) return BT_OK;
    BT_TRY(check_rows("bt_attention_kv8", "q", dtype, q));
    const int V = dtype == BT_BF16 ? 8 : 4;
    BT_CHECK_ARG(out && aligned16(out) && ldo % V == 0 && ldo >= (int64_t)heads * cache->head_dim,
                 "bt_attention_kv8: output rows must be 16-byte granular and hold heads * head_dim");
    BT_CHECK_ARG(pos0_dev || (pos0_host >= 0 && (int64_t)pos0_host + q_len <= cache->n_max), "bt_attention_kv8: cache overflow");
    BT_CHECK_ARG(!mask || mask_ld >= (pos0_dev ? cache->n_max : (int64_t)pos0_host + q_len), "bt_attention_kv8: mask row too short");
    BT_CHECK_ARG(n_split >= 1, "bt_attention_kv8: bad n_split %d", n_split);
    const int64_t need = bt_attention_kv8_workspace_bytes(cache->batch, q_len, heads, cache->head_dim, n_split);
    if (need > 0 && (!ws || ws_bytes < need || !aligned16(ws))) {
        set_error("bt_attention_kv8: split workspace too small or unaligned (%lld < %lld bytes)", (long long)ws_bytes, (long long)need);
        return BT_ERR_WORKSPACE;
    }
    const int64_t grid = cache->batch * q_len * heads;
    BT_CHECK_ARG(grid < (1ll << 31), "bt_attention_kv8: grid too large");
    a.c = *cache;
    a.q = rows_of(q);
    a.q_len = q_len;
    a.heads = heads;
    a.pos0_host = pos0_host;
    a.pos0_dev = pos0_dev;
    a.mask = mask;
    a.mask_ld = mask_ld;
    a.out = out;
    a.ldo = ldo;
    a.scale = 1.4426950408889634f / sqrtf((float)cache->head_dim);
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ATTN_ROWS, s);
    if (dtype == BT_BF16)
        hipLaunchKernelGGL(attention_kv8_kernel<bf16>, dim3((unsigned)grid), dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL(attention_kv8_kernel<float>, dim3((unsigned)grid), dim3(64), 0, s, a);
    BT_LAUNCH_CHECK("bt_attention_kv8 launch");
    return BT_OK;
}
