// A KV cache in 8 bits with one scale per block of rows and head (layout and rules: bt_kv8_cache in bt_hip.h): append with RoPE, read
// back, and attention over it.
#include "bt_common.h"
#include "bt_quant.h"

#include <algorithm>
#include <type_traits>

namespace bt {

struct Rows {      // bt_kv8_rows on the device
    char* p;
    int64_t b, t, h;
};

// ---- bt_kv8_append ---------------------------------------------------------------------------------------------------------
struct AppendArgs {
    bt_kv8_cache c;
    Rows q, q_out, k, v;
    uint32_t kv_items;     // waves for keys and values: batch * kv_heads * blocks << split
    uint32_t q_rows;       // batch * q_len * heads
    int blocks;            // blocks that q_len rows can touch
    int split;             // keys and values of a block by a wave each (1), by one (0)
    int q_len, heads, rot, pos0_host;
    bool vec_rope;
    const int32_t* pos0_dev;
    const int32_t* pos_table;
    const float* cos_tab;
    const float* sin_tab;
    int64_t max_pos;
};

// The entry of the position table for row t of a call at `pos0`, which the device may have read from anywhere: rows behind the cache's end
// are dropped, but their queries are rotated all the same, by the table's last entry and not by what lies behind it.  (64 bits: pos0 + t
// leaves an int.)
__host__ __device__ constexpr int64_t table_entry(int64_t pos, int64_t n_max) { return pos < 0 ? 0 : pos < n_max ? pos : n_max - 1; }
static_assert(table_entry((int64_t)INT32_MAX + 1, 64) == 63 && table_entry((int64_t)INT32_MAX + (1 << 30), 64) == 63);
static_assert(table_entry(63, 64) == 63 && table_entry(64, 64) == 63 && table_entry(0, 64) == 0 && table_entry(INT32_MIN, 64) == 0);

__device__ inline int64_t angle_of(const AppendArgs& a, int64_t pos) {
    int64_t r = a.pos_table ? a.pos_table[table_entry(pos, a.c.n_max)] : pos;
    r = r < 0 ? 0 : r;
    return r < a.max_pos ? r : a.max_pos - 1;
}

// Dims e0 .. e0 + V - 1 of a row, rotated.  The two products of 24-bit numbers are exact in fp64, so the result is their sum rounded to
// fp64 and from there to fp32 (and, where the row is written in bf16, from fp32 to bf16, as torch converts): codes, and so what is compared
// bit for bit, do not depend on how a sum was fused.  Costs nothing here: memory is the bound.
template <typename T>
__device__ inline void rotated_piece(const AppendArgs& a, const T* row, int e0, int64_t angle, float (&v)[Elem<T>::VEC]) {
    constexpr int V = Elem<T>::VEC;
    load_vec<T>(row + e0, v);
    if (e0 >= a.rot) return;
    const int half = a.rot >> 1;
    if (a.vec_rope) {      // half is a multiple of V: the other halves are one piece too
        const bool low = e0 < half;
        const int j = low ? e0 : e0 - half;
        float o[V];
        load_vec<T>(row + (low ? e0 + half : j), o);
        const float* c = a.cos_tab + angle * half + j;
        const float* s = a.sin_tab + angle * half + j;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 cc = *(const float4*)(c + i), ss = *(const float4*)(s + i);
            const float cs[4] = {cc.x, cc.y, cc.z, cc.w}, sn[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double p = (double)o[i + k] * (low ? -sn[k] : sn[k]);
                v[i + k] = (float)fma((double)v[i + k], (double)cs[k], p);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = e0 + i;
            if (e >= a.rot) break;
            const int j = e < half ? e : e - half;
            const double o = Elem<T>::load(row + (e < half ? e + half : j)), c = a.cos_tab[angle * half + j], s = a.sin_tab[angle * half + j];
            v[i] = (float)fma((double)v[i], c, e < half ? -o * s : o * s);
        }
    }
}

// v as `T` holds it
template <typename T>
__device__ inline void round_piece(float (&v)[Elem<T>::VEC]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint32_t two = pack_bf16x2(v[i], v[i + 1]);
            v[i] = __uint_as_float(two << 16);
            v[i + 1] = __uint_as_float(two & 0xffff0000u);
        }
    }
}

// The scale of a block: the largest finite magnitude.  Two instructions a value; `odd` (a NaN or infinity: 0 * v is not 0) is rare, and
// then the largest is looked for again without those.
struct BlockMax {
    float amax = 0.f, zero = 0.f;
    __device__ inline void see(float v) {
        amax = fmaxf(amax, fabsf(v));
        zero = fmaf(v, 0.f, zero);
    }
    __device__ inline bool odd() const { return __any(zero != 0.f); }      // (NaN != 0)
    template <int N>
    __device__ static inline float finite(const float (&v)[N]) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.f);
        return max64(m);
    }
};

// One wave per (sequence, head, block) that the new rows touch, or one for its K and one for its V (`split`); the waves behind them rotate q.
//   K, q: a lane has 16-byte pieces of rows, four to a row, a quarter row apart: the rotary dims are then the same piece of every lane, and
//         the fp64 work of the others is skipped.
//   V: a lane has columns 2 x, 2 x + 1 of 16 rows, that is two 16-byte runs of v_codes: rows are read 256 bytes a wave and instruction,
//      and no transpose is needed.  Rows of the open block come in runs from v_tail, which is transposed already.
// K and V are held in registers between the search for the scale and the codes.  Bound by memory and the chain load -> scale -> codes:
// 32 sequences x 509 rows x 16 heads of 128 (333 MB) in blocks of 16 88 .. 93 us by card (3.6 .. 3.8 TB/s; 79 registers, six waves to a
// SIMD), in blocks of 32 166 .. 173 us (85, five), of 64 242 .. 256 us (162, three); fp32 (600 MB) in blocks of 16 149 us (4.0 TB/s).  The
// straight-line code for a block is 54, 90 and 156 KB, so from 32 rows on more than an instruction cache holds.  A step that fills 4096
// blocks of 16 rows 16 us, one that fills none 8 us.
template <typename T, int D, int BL>
__global__ __launch_bounds__(256, D * BL <= 2048 ? 5 : D * BL <= 4096 ? 4 : 2) void kv8_append_kernel(AppendArgs a) {
    constexpr int V = Elem<T>::VEC, RP = D / V, LR = RP / 4;      // pieces of a row, lanes to a row
    const int lane = threadIdx.x & 63;
    const int pos0 = a.pos0_dev ? *a.pos0_dev : a.pos0_host;
    if (pos0 < 0) return;
    const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e_lane = lane % LR * V;      // piece k of this lane: dims e_lane + k D / 4
    if (item >= a.kv_items) {
        // A row (b, t, h) of q to LR lanes.  The last workgroup has waves too many, without q all of these are.
        const uint32_t i0 = (item - a.kv_items) * (64 / LR);
        if (i0 >= a.q_rows) return;
        uint32_t i = i0 + lane / LR;
        const bool there = i < a.q_rows;
        i = there ? i : a.q_rows - 1;
        const uint32_t bt = i / (uint32_t)a.heads, b = bt / (uint32_t)a.q_len;
        const int h = (int)(i - bt * a.heads), t = (int)(bt - b * a.q_len);
        const T* src = (const T*)a.q.p + b * a.q.b + t * a.q.t + h * a.q.h;
        T* dst = (T*)a.q_out.p + b * a.q_out.b + t * a.q_out.t + h * a.q_out.h;
        const int64_t pos = (int64_t)pos0 + t;
        float v[4][V];
#pragma unroll
        for (int k = 0; k < 4; ++k) load_vec<T>(src + e_lane + k * (D / 4), v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e_lane + k * (D / 4) < a.rot) rotated_piece<T>(a, src, e_lane + k * (D / 4), angle_of(a, pos), v[k]);
        asm volatile("" ::: "memory");      // q_out may be q: every lane of the row has read before one writes
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (there) store_vec<T>(dst + e_lane + k * (D / 4), v[k]);
        return;
    }
    // neighbouring waves take neighbouring heads: of a fused projection's rows they read one piece of memory
    const uint32_t row = item / (uint32_t)a.c.kv_heads, bn = row >> a.split, b = bn / (uint32_t)a.blocks;
    const bool values = !a.split || (row & 1), keys = !a.split || !(row & 1);
    const int h = (int)(item - row * a.c.kv_heads), nth = (int)(bn - b * a.blocks);
    const uint32_t bh = b * a.c.kv_heads + h;
    const int64_t end = pos0 + (int64_t)a.q_len < a.c.n_max ? pos0 + (int64_t)a.q_len : a.c.n_max;
    const T* ksrc = (const T*)a.k.p + b * a.k.b + h * a.k.h;
    const T* vsrc = (const T*)a.v.p + b * a.v.b + h * a.v.h;
    T* kt = (T*)a.c.k_tail + (int64_t)bh * BL * D;
    T* vt = (T*)a.c.v_tail + (int64_t)bh * BL * D;
    const int64_t n_blk = a.c.n_max / BL;
    const int first = pos0 / BL, last = (int)(end / BL);      // `last` stays open
    if (nth > 0 && first + nth >= last) return;
    const int64_t blk = first + nth, row0 = blk * BL;
    if (row0 >= end) return;
    const int old = nth == 0 ? pos0 - (int)row0 : 0;          // rows of the block that stand in the tail
    if (row0 + BL <= end) {
        if (keys) {
            constexpr int NR = BL * LR / 64 > 0 ? BL * LR / 64 : 1;      // rows of a lane
            float x[NR][4][V];
            BlockMax top;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int t = (i * 64 + lane) / LR;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int e0 = e_lane + k * (D / 4);
#pragma unroll
                    for (int e = 0; e < V; ++e) x[i][k][e] = 0.f;
                    if (t >= BL) continue;
                    if (t < old) load_vec<T>(kt + t * D + e0, x[i][k]);
                    else load_vec<T>(ksrc + (row0 + t - pos0) * a.k.t + e0, x[i][k]);
                }
            }
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int t = (i * 64 + lane) / LR;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int e0 = e_lane + k * (D / 4);
                    if (t < BL && t >= old && e0 < a.rot) {
                        const int at = (int)(row0 + t - pos0);
                        rotated_piece<T>(a, ksrc + at * a.k.t, e0, angle_of(a, (int64_t)pos0 + at), x[i][k]);
                        round_piece<T>(x[i][k]);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) top.see(x[i][k][e]);
                }
            }
            const bool odd = top.odd();
            float amax = max64(top.amax);
            if (odd) {
                amax = 0.f;
#pragma unroll
                for (int i = 0; i < NR; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) amax = fmaxf(amax, BlockMax::finite(x[i][k]));
            }
            const Quantiser q(amax);
            const bool quick = q.direct && !odd;
            if (lane == 0) a.c.k_scale[bh * n_blk + blk] = q.scale;
            int8_t* out = a.c.k_codes + (bh * a.c.n_max + row0) * D;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const int t = (i * 64 + lane) / LR;
                if (t >= BL) continue;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float* y = x[i][k];
                    uint32_t w[V / 4];
#pragma unroll
                    for (int e = 0; e < V; e += 4)
                        w[e / 4] = quick ? q.pack4(y[e], y[e + 1], y[e + 2], y[e + 3]) : q.pack4_exact(y[e], y[e + 1], y[e + 2], y[e + 3]);
                    int8_t* o = out + t * D + e_lane + k * (D / 4);
                    if constexpr (V == 8) *(uint2*)o = uint2{w[0], w[1]};
                    else *(uint32_t*)o = w[0];
                }
            }
        }
        if (values) {
            constexpr int UNITS = D / 2 * (BL / 16), NU = (UNITS + 63) / 64;      // V: (pair of columns, run of 16 rows)
            typedef typename std::conditional<sizeof(T) == 2, uint32_t, float2>::type Pair;
            Pair raw[NU][16];
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int idx = u * 64 + lane, d = (idx % (D / 2)) * 2, t0 = idx / (D / 2) * 16;
                const T* p = vsrc + (row0 - pos0 + t0) * a.v.t + d;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    raw[u][e] = Pair{};
                    if (idx < UNITS && t0 + e >= old) raw[u][e] = *(const Pair*)(p + e * a.v.t);
                }
            }
            float x[NU][2][16];
            BlockMax top;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int idx = u * 64 + lane, d = (idx % (D / 2)) * 2, t0 = idx / (D / 2) * 16;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (sizeof(T) == 2) {
                        x[u][0][e] = __uint_as_float(raw[u][e] << 16);
                        x[u][1][e] = __uint_as_float(raw[u][e] & 0xffff0000u);
                    } else {
                        x[u][0][e] = raw[u][e].x;
                        x[u][1][e] = raw[u][e].y;
                    }
                }
                if (idx < UNITS && t0 < old) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int e = 0; e < 16; e += V) {
                            float v[V];
                            load_vec<T>(vt + (d + c) * BL + t0 + e, v);
#pragma unroll
                            for (int k = 0; k < V; ++k) x[u][c][e + k] = t0 + e + k < old ? v[k] : x[u][c][e + k];
                        }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    top.see(x[u][0][e]);
                    top.see(x[u][1][e]);
                }
            }
            const bool odd = top.odd();
            float amax = max64(top.amax);
            if (odd) {
                amax = 0.f;
#pragma unroll
                for (int u = 0; u < NU; ++u) amax = fmaxf(amax, fmaxf(BlockMax::finite(x[u][0]), BlockMax::finite(x[u][1])));
            }
            const Quantiser q(amax);
            const bool quick = q.direct && !odd;
            if (lane == 0) a.c.v_scale[bh * n_blk + blk] = q.scale;
            int8_t* out = a.c.v_codes + (bh * n_blk + blk) * D * BL;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int idx = u * 64 + lane, d = (idx % (D / 2)) * 2, t0 = idx / (D / 2) * 16;
                if (idx >= UNITS) continue;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float* y = x[u][c];
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = quick ? q.pack4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3])
                                     : q.pack4_exact(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
                    *(uint4*)(out + (d + c) * BL + t0) = uint4{w[0], w[1], w[2], w[3]};
                }
            }
        }
    }
    // The open block's rows take the places that the first block's old rows leave, so the first wave writes them, after it has read those.
    if (nth != 0) return;
    const int64_t open0 = (int64_t)last * BL;
    const int from = open0 > pos0 ? 0 : (int)(pos0 - open0), to = (int)(end - open0);
    for (int idx = from * RP + lane; keys && idx < to * RP; idx += 64) {
        const int t = idx / RP, e0 = (idx & (RP - 1)) * V;
        const int at = (int)(open0 + t - pos0);
        float v[V];
        rotated_piece<T>(a, ksrc + at * a.k.t, e0, a.rot ? angle_of(a, (int64_t)pos0 + at) : 0, v);
        store_vec<T>(kt + t * D + e0, v);
    }
    if (values && to - from == 1) {
        const T* p = vsrc + (open0 + from - pos0) * a.v.t;
        for (int d = lane; d < D; d += 64) vt[d * BL + from] = p[d];
    } else if (values && lane * 2 < D) {
        // 16 rows in flight together
        typedef typename std::conditional<sizeof(T) == 2, uint32_t, float2>::type Pair;
        const int d = lane * 2;
        for (int t0 = from & ~15; t0 < to; t0 += 16) {
            const T* p = vsrc + (open0 + t0 - pos0) * a.v.t + d;
            Pair raw[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (t0 + e >= from && t0 + e < to) raw[e] = *(const Pair*)(p + e * a.v.t);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (t0 + e >= from && t0 + e < to) {
                    T two[2];
                    __builtin_memcpy(two, &raw[e], sizeof two);
                    vt[d * BL + t0 + e] = two[0];
                    vt[(d + 1) * BL + t0 + e] = two[1];
                }
        }
    }
}

// ---- bt_kv8_read -----------------------------------------------------------------------------------------------------------
// One wave per (sequence, head, block): K by pieces of 16 codes, V by pairs of columns and runs of 16 rows, as append has them.  Bound by
// memory: 32 x 509 rows x 16 heads of 128 (200 MB) 31 .. 37 us by card (5.4 .. 6.4 TB/s, part of it from the caches); in blocks of 32 44 us,
// of 64 52 us.
template <typename T, int D, int BL>
__global__ __launch_bounds__(256) void kv8_read_kernel(bt_kv8_cache c, int64_t n, int64_t first, int64_t count, int blocks,
                                                      T* __restrict__ ko, T* __restrict__ vo) {
    constexpr int V = Elem<T>::VEC;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= c.batch * c.kv_heads * blocks) return;
    const int64_t bh = item / blocks, n_blk = c.n_max / BL, blk = first / BL + (item - bh * blocks);
    const int64_t out0 = (bh * count + blk * BL - first) * D;      // where row 0 of the block would go
    const int from = first > blk * BL ? (int)(first - blk * BL) : 0;
    const int to = first + count < (blk + 1) * BL ? (int)(first + count - blk * BL) : BL;
    const bool open = blk >= n / BL;
    if (ko) {
        const float s = open ? 0.f : c.k_scale[bh * n_blk + blk];
        const int8_t* kc = c.k_codes + (bh * c.n_max + blk * BL) * D;
        const T* kt = (const T*)c.k_tail + bh * BL * D;
#pragma unroll
        for (int i = 0; i < (BL * D / 16 + 63) / 64; ++i) {
            const int idx = i * 64 + lane, t = idx / (D / 16), e0 = idx % (D / 16) * 16;
            if (t < from || t >= to) continue;
            T* o = ko + out0 + t * D + e0;
            if (open) {
#pragma unroll
                for (int e = 0; e < 16; e += V) *(uint4*)(o + e) = *(const uint4*)(kt + t * D + e0 + e);
            } else {
                const int4 w = *(const int4*)(kc + t * D + e0);
                const int words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 16; e += V) {
                    float v[V];
#pragma unroll
                    for (int k = 0; k < V; ++k) v[k] = (float)(int8_t)(words[(e + k) >> 2] >> (8 * (k & 3))) * s;
                    store_vec<T>(o + e, v);
                }
            }
        }
    }
    if (vo) {
        const float s = open ? 0.f : c.v_scale[bh * n_blk + blk];
        const int8_t* vc = c.v_codes + (bh * n_blk + blk) * D * BL;
        const T* vt = (const T*)c.v_tail + bh * BL * D;
        constexpr int UNITS = D / 2 * (BL / 16);
#pragma unroll
        for (int u = 0; u < (UNITS + 63) / 64; ++u) {
            const int idx = u * 64 + lane, d = (idx % (D / 2)) * 2, t0 = idx / (D / 2) * 16;
            if (idx >= UNITS) continue;
            float x[2][16];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (open) {
#pragma unroll
                    for (int e = 0; e < 16; e += V) {
                        float v[V];
                        load_vec<T>(vt + (d + k) * BL + t0 + e, v);
#pragma unroll
                        for (int y = 0; y < V; ++y) x[k][e + y] = v[y];
                    }
                } else {
                    const int4 w = *(const int4*)(vc + (d + k) * BL + t0);
                    const int words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[k][e] = (float)(int8_t)(words[e >> 2] >> (8 * (e & 3))) * s;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (t0 + e < from || t0 + e >= to) continue;
                T* o = vo + out0 + (t0 + e) * D + d;
                if constexpr (sizeof(T) == 2) *(uint32_t*)o = pack_bf16x2(x[0][e], x[1][e]);
                else *(float2*)o = float2{x[0][e], x[1][e]};
            }
        }
    }
}

// ---- bt_attention_kv8 ------------------------------------------------------------------------------------------------------
// The arithmetic of an fp32 attention on the bf16 matrix instructions.  A code is an exact bf16, q and the probabilities (times their rows' V
// scales) enter as the one or three bf16 whose sum they are, so products are exact and sums fp32: small probabilities beside a large one,
// blocks of different scales and queries with outliers keep all their bits.  (Digits of a fixed point for a tile do not: a row of
// e^-17 of the largest weight was lost.)
//
// A wave works on 16 query rows (rows x heads that share a KV head) and 64 cached rows at a time:
//   S^T = K Q^T   A = K: lane (m = lane & 15, g = lane >> 4) holds 16 bytes (8 of 32 dims) of row tok(i, m) = 16 (m >> 2) + 4 i + (m & 3),
//                 i = 0 .. 3; 8 of them are one operand of v_mfma_f32_16x16x32_bf16 (its k-range 8 g .. 8 g + 7: the dims that q has there).
//                 In the result lane (query c = lane & 15, g) holds rows 16 g + 4 i + r, r = 0 .. 3: 16 consecutive rows, one block's
//                 scale, one 16-byte piece of the mask.
//   O^T = V^T P^T B = P: the lane's own 16 rows are two operands: nothing moves between lanes.
//                 A = V^T: lane m holds the same 16 consecutive rows of dim 16 j + m, one 16-byte load from v_codes.
// Softmax: a running (max, sum, output) in fp32.  The open block is one more tile, its rows as they stand (fp32: v_mfma_f32_16x16x4_f32).
// Bound by reading the cache where there is enough of it: 1024 sequences x 16 heads of 128 x 543 rows 401 .. 429 us by card (5.5 .. 5.9 TB/s;
// the card reads 6.0), 256 sequences 111 .. 120 us (4.9 .. 5.3), 4 sequences x 32773 rows, 8 heads to a KV head, 30 us with the join (4.5),
// fp32, 128 sequences, 61 .. 68 us (4.2 .. 4.7).  A tile costs about 710 vector instructions (over half of them turn codes into bf16) and 64
// matrix instructions for its 16 KB, under half of what would bound it; with one wave to a SIMD that shows: 8 sequences x 24608 rows x 2 heads
// of 64, 20 query rows each, 24 us, where a fixed point for a tile took 20.5.  One sequence of 21 rows: 6.2 us, three round trips to memory.
// 32 prompts of 512 rows 222 us: every 16 query rows read K and V for themselves.
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct AttnArgs {
    bt_kv8_cache c;
    Rows q;
    int q_len, heads, share, rows, row_groups, n_split, pos0_host, shift;
    const int32_t* pos0_dev;
    const uint8_t* mask;
    int64_t mask_ld;
    void* out;
    int64_t ldo;
    float* part;      // [batch][kv_heads][rows][n_split][head_dim + 2]: output, max, sum; nullptr: one split
    float scale;      // log2(e) / sqrt(head_dim)
};

// "no score yet": the lowest finite number, so that a difference of two of them is 0 and no score of a row that is seen lies below
constexpr float M_FLOOR = -3.402823466e38f;

// The numbers of a pair of floats as NP bf16 each, largest first: what the first has cut off goes to the next, so three are exact.
template <int NP>
__device__ inline void cut_bf16x2(float x0, float x1, uint32_t (&out)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        out[p] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302);
        x0 -= __uint_as_float(__float_as_uint(x0) & 0xffff0000u);
        x1 -= __uint_as_float(__float_as_uint(x1) & 0xffff0000u);
    }
}

// eight codes as bf16
__device__ inline bf16x8 codes_bf16(int w0, int w1) {
    union { uint32_t u[4]; bf16x8 f; } r;
    const int w[2] = {w0, w1};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = w[i >> 1], at = 16 * (i & 1);
        r.u[i] = __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)(x >> (at + 8))), __float_as_uint((float)(int8_t)(x >> at)), 0x07060302);
    }
    return r.f;
}

template <typename T, int D>
struct Attend {
    static constexpr int NQ = sizeof(T) == 2 ? 1 : 3;       // bf16 numbers to an element of q
    static constexpr int NC = (D + 63) / 64;                // 64-dim pieces of a row of K
    static constexpr int NH = D >= 64 ? 2 : 1;              // operands of a lane's part of a piece, 8 dims each
    static constexpr int NJ = D / 16;                       // 16-dim pieces of the output
    typedef typename std::conditional<D >= 64, i32x4, i32x2>::type KPart;
    union Operand {
        uint32_t u[4];
        bf16x8 f;
    };

    const AttnArgs& a;
    const int lane, c, g;
    int64_t bh, n_full, full, n_blk;
    const int8_t *kc, *vc;
    const float *ks, *vs;
    const uint8_t* mask;
    const T* q;
    int64_t lim;              // rows that this lane's query sees
    int up = 0;               // q is held times 2^-up, so that its products with codes stay in fp32
    float poison = 0.f;       // NaN where q has an infinity or NaN, else 0
    Operand qf[NQ][NC][NH];
    float m = M_FLOOR, l = 0.f;
    f32x4 o[NJ];

    __device__ Attend(const AttnArgs& a_) : a(a_), lane(threadIdx.x & 63), c(lane & 15), g(lane >> 4) {}

    __device__ inline void load_query(bool real) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        float x[NC][8 * NH];
        float amax = 0.f, bad = 0.f;
#pragma unroll
        for (int k = 0; k < NC; ++k) {
#pragma unroll
            for (int e = 0; e < 8 * NH; e += Elem<T>::VEC) {
                float v[Elem<T>::VEC] = {};
                if (real) load_vec<T>(q + 64 * k + 8 * NH * g + e, v);
#pragma unroll
                for (int i = 0; i < Elem<T>::VEC; ++i) {
                    x[k][e + i] = v[i];
                    amax = fmaxf(amax, fabsf(v[i]));
                    bad = fabsf(v[i]) < INFINITY ? bad : 1.f;
                }
            }
        }
        amax = max_over_groups(amax);
        bad = max_over_groups(bad);
        poison = bad != 0.f ? __int_as_float(0x7fc00000) : 0.f;
        up = bad != 0.f ? 0 : __builtin_amdgcn_frexp_expf(amax);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int e = 0; e < 8 * NH; e += 2) {
                uint32_t two[NQ];
                cut_bf16x2<NQ>(bad != 0.f ? poison : ldexpf(x[k][e], -up), bad != 0.f ? poison : ldexpf(x[k][e + 1], -up), two);
#pragma unroll
                for (int p = 0; p < NQ; ++p) qf[p][k][e >> 3].u[(e & 7) >> 1] = two[p];
            }
    }

    __device__ inline void load_k(int64_t tile, KPart (&k)[4][NC]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int64_t tok = tile * 64 + 16 * (c >> 2) + 4 * i + (c & 3);
            tok = tok < a.c.n_max ? tok : a.c.n_max - 1;
            const int8_t* p = kc + tok * D + 8 * NH * g;
#pragma unroll
            for (int n = 0; n < NC; ++n) k[i][n] = *(const KPart*)(p + 64 * n);
        }
    }
    // the scales and the mask of this lane's 16 rows of a tile
    struct Side {
        float sk, sv;
        uint4 mask;
    };
    __device__ inline Side load_side(int64_t tile) const {
        const int64_t tok = tile * 64 + 16 * g;
        int64_t blk = tok >> a.shift;
        blk = blk < full ? blk : full - 1;      // (a tile has a full block; what lies behind the last is hidden)
        Side x{ks[blk], vs[blk], uint4{0, 0, 0, 0}};
        if (mask && tok + 16 <= n_full) __builtin_memcpy(&x.mask, mask + tok, 16);      // wherever they lie
        return x;
    }
    __device__ inline void load_v(int64_t tile, i32x4 (&v)[NJ]) const {
        const int64_t tok = tile * 64 + 16 * g;
        int64_t blk = tok >> a.shift;
        blk = blk < n_blk ? blk : n_blk - 1;
        const int8_t* p = vc + (blk * D + c) * a.c.block + (tok & (a.c.block - 1));
#pragma unroll
        for (int j = 0; j < NJ; ++j) v[j] = *(const i32x4*)(p + (int64_t)16 * j * a.c.block);
    }
    // bit e: byte e is not 0
    __device__ static inline uint32_t set_bytes(const uint4& u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t on = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t set = ((((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) >> 7) & 0x01010101u;
            on |= ((set * 0x10204080u) >> 28) << (4 * i);      // the first byte's to bit 28, the last one's to bit 31
        }
        return on;
    }
    // bits 0 .. count - 1: rows tok0 .. that are before `end` and before this lane's query's limit
    __device__ inline uint32_t reached(int64_t tok0, int count, int64_t end) const {
        const int64_t left = (end < lim ? end : lim) - tok0;
        const int most = left < count ? (left < 0 ? 0 : (int)left) : count;
        return (1u << most) - 1u;
    }

    // enters a tile with its largest score: the factor for what is there already
    __device__ inline float enter(float mt) {
        const float mn = fmaxf(m, mt), alpha = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        return alpha;
    }

    // One tile.  `k` and `v` hold it; MORE: the next tile's take their places as soon as they have been used, K under the softmax and
    // the second product, V under the next tile's first.
    template <bool MORE>
    __device__ inline void tile(int64_t at, int64_t then, KPart (&k)[4][NC], i32x4 (&v)[NJ], Side& side, bool cut) {
        const int64_t tok0 = at * 64 + 16 * g;
        const Side now = side;
        if (MORE) side = load_side(then);
        const float mul = ldexpf(a.scale * now.sk, up);
        float sv = now.sv;
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const bf16x8 kf = codes_bf16(k[i][n][2 * h], k[i][n][2 * h + 1]);
#pragma unroll
                    for (int p = NQ - 1; p >= 0; --p) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[p][n][h].f, acc, 0, 0, 0);
                }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = acc[r] * mul;
        }
        if (MORE) load_k(then, k);
        if (cut) {
            uint32_t on = reached(tok0, 16, n_full);
            if (mask) on &= set_bytes(now.mask);
            sv = on ? sv : 0.f;      // of a block that nobody sees not even the scale counts: it may be anything
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][r] = (on >> (4 * i + r)) & 1 ? s[i][r] : -INFINITY;
        }
        float mt = M_FLOOR;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[i][r]);
        const float alpha = enter(max_over_groups(mt));
        float sum = 0.f;
        Operand p[3][2];      // rows 8 h .. 8 h + 7 of the lane's 16
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float e0 = __builtin_amdgcn_exp2f(s[e >> 2][e & 3] - m), e1 = __builtin_amdgcn_exp2f(s[e >> 2][(e & 3) + 1] - m);
            sum += e0;
            sum += e1;
            uint32_t two[3];
            cut_bf16x2<3>(e0 * sv, e1 * sv, two);
#pragma unroll
            for (int x = 0; x < 3; ++x) p[x][e >> 3].u[(e & 7) >> 1] = two[x];
        }
        l = fmaf(l, alpha, sum);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bf16x8 vf = codes_bf16(v[j][2 * h], v[j][2 * h + 1]);
#pragma unroll
                for (int x = 2; x >= 0; --x) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, p[x][h].f, acc, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][r] = fmaf(o[j][r], alpha, acc[r]);
        }
        if (MORE) load_v(then, v);
    }

    // The open block: rows n_full .. end - 1, row 4 nI g + 4 i + r of it with lane g's (i, r), nI = block / 16.
    __device__ void tail(int64_t end) {
        const int bl = a.c.block, nI = bl >> 4, per = bl >> 2;
        const T* kt = (const T*)a.c.k_tail + bh * bl * D;
        const T* vt = (const T*)a.c.v_tail + bh * bl * D;
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= nI) {
#pragma unroll
                for (int r = 0; r < 4; ++r) s[i][r] = -INFINITY;
                continue;
            }
            const T* kr = kt + (per * (c >> 2) + 4 * i + (c & 3)) * D;
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int n = 0; n < D / 32; ++n) {
                    const bf16x8 kf = *(const bf16x8*)(kr + 32 * n + 8 * g), qf = *(const bf16x8*)(q + 32 * n + 8 * g);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf, acc, 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int n = 0; n < D / 4; n += 4) {
                    const f32x4 kf = *(const f32x4*)(kr + D / 4 * g + n), qf = *(const f32x4*)(q + D / 4 * g + n);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[e], acc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = fmaf(acc[r], a.scale, poison);
        }
        const int64_t tok0 = n_full + per * g;
        const int there = end - tok0 < per ? (end > tok0 ? (int)(end - tok0) : 0) : per;
        uint32_t some = (1u << there) - 1u;      // rows that any query may see
        if (mask)
            for (int e = 0; e < there; ++e) some &= mask[tok0 + e] != 0 ? ~0u : ~(1u << e);
        const uint32_t on = reached(tok0, per, end) & some;
        float mt = M_FLOOR;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[i][r] = (on >> (4 * i + r)) & 1 ? s[i][r] : -INFINITY;
                mt = fmaxf(mt, s[i][r]);
            }
        const float alpha = enter(max_over_groups(mt));
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - m);
                sum += s[i][r];
            }
        l = fmaf(l, alpha, sum);
        // P V.  Rows that nobody may see are taken as zero: they may hold anything.
        f32x4 before[NJ];
        uint32_t keep[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) keep[e] = (some >> e) & 1 ? ~0u : 0u;
        Operand p[3][2];      // bf16: the probabilities in three pieces, rows 8 h .. 8 h + 7 of the lane's
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                uint32_t two[3];
                cut_bf16x2<3>(s[e >> 2][e & 3], s[e >> 2][(e & 3) + 1], two);
#pragma unroll
                for (int x = 0; x < 3; ++x) p[x][e >> 3].u[(e & 7) >> 1] = two[x];
            }
        }
        float zero = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            before[j] = o[j] *= alpha;
            const T* vr = vt + (16 * j + c) * bl + per * g;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (8 * h >= per) continue;      // per is 4, 8 or 16
                    Operand vf;
                    const uint2 low = *(const uint2*)(vr + 8 * h), high = per > 4 ? *(const uint2*)(vr + 8 * h + 4) : uint2{0, 0};
                    const uint32_t four[4] = {low.x, low.y, high.x, high.y};
#pragma unroll
                    for (int e = 0; e < 4; ++e) vf.u[e] = four[e] & __builtin_amdgcn_perm(keep[8 * h + 2 * e + 1], keep[8 * h + 2 * e], 0x05040100);
#pragma unroll
                    for (int x = 2; x >= 0; --x) o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf.f, p[x][h].f, o[j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 16; h += 4) {
                    if (h >= per) continue;
                    const f32x4 v = *(const f32x4*)(vr + h);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(__float_as_uint(v[e]) & keep[h + e]), s[h >> 2][e], o[j], 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) zero = fmaf(o[j][r], 0.f, zero);
        }
        // An infinity or NaN in a row that some queries see and others do not: the product has given it to all of them.  Once more, by hand.
        if (__any(zero != 0.f)) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) o[j] = before[j];
#pragma unroll 1
            for (int x = 0; x < bl; ++x) {
                const int gg = x / per, e = x - gg * per;
                float p = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) p = i == e ? s[i >> 2][i & 3] : p;
                p = __shfl(p, gg * 16 + c, 64);
                const bool seen = (__shfl((int)on, gg * 16 + c, 64) >> e) & 1;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float y = Elem<T>::load(vt + (16 * j + 4 * g + r) * bl + x);
                        o[j][r] = seen ? fmaf(p, y, o[j][r]) : o[j][r];
                    }
            }
        }
    }
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attention_kv8_kernel(AttnArgs a) {
    using A = Attend<T, D>;
    __shared__ float merged[NW > 1 ? NW : 1][NW > 1 ? 16 : 1][D + 4];
    const int wave = NW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    A w(a);
    const uint32_t part = blockIdx.x / (uint32_t)a.n_split, head = part / (uint32_t)a.row_groups;
    const int split = (int)(blockIdx.x - part * (uint32_t)a.n_split), rg = (int)(part - head * (uint32_t)a.row_groups);
    w.bh = head;
    const int64_t b = head / (uint32_t)a.c.kv_heads;
    const int h0 = (int)(w.bh - b * a.c.kv_heads) * a.share;
    const int pos0 = a.pos0_dev ? *a.pos0_dev : a.pos0_host;
    const int row = rg * 16 + w.c;
    const bool real = row < a.rows;
    const int t = real ? row / a.share : 0, h = h0 + (real ? row - t * a.share : 0);
    int64_t n = pos0 + (int64_t)a.q_len;
    n = n < 0 ? 0 : n < a.c.n_max ? n : a.c.n_max;
    const int last_row = rg * 16 + 15 < a.rows ? rg * 16 + 15 : a.rows - 1;
    int64_t end = pos0 + (int64_t)last_row / a.share + 1;      // no row of this group sees further
    end = end < 0 ? 0 : end < n ? end : n;
    int64_t least = pos0 + (int64_t)(rg * 16) / a.share + 1;   // every row of it sees as far as this
    w.full = n >> a.shift;
    w.n_full = w.full << a.shift;
    w.n_blk = a.c.n_max >> a.shift;
    w.lim = pos0 + (int64_t)t + 1 < n ? pos0 + (int64_t)t + 1 : n;
    w.kc = a.c.k_codes + w.bh * a.c.n_max * D;
    w.vc = a.c.v_codes + w.bh * a.c.n_max * D;
    w.ks = a.c.k_scale + w.bh * w.n_blk;
    w.vs = a.c.v_scale + w.bh * w.n_blk;
    w.mask = a.mask ? a.mask + b * a.mask_ld : nullptr;
    w.q = (const T*)a.q.p + b * a.q.b + t * a.q.t + h * a.q.h;
    const int64_t closed = w.n_full < end ? w.n_full : end;      // rows of full blocks that somebody sees
    const int64_t tiles = (closed + 63) >> 6, all = tiles + (end > w.n_full ? 1 : 0);
    const int64_t per = (all + a.n_split - 1) / a.n_split;
    int64_t at = split * per + wave;
    const int64_t stop = (split + 1) * per < all ? (split + 1) * per : all, closed_stop = stop < tiles ? stop : tiles;
    if (at < closed_stop) {
        typename A::KPart k[4][A::NC];
        i32x4 v[A::NJ];
        typename A::Side side = w.load_side(at);
        w.load_k(at, k);
        w.load_v(at, v);
        w.load_query(real);      // (its wait covers them too)
        auto cut = [&](int64_t t) { return w.mask || t * 64 + 64 > w.n_full || t * 64 + 64 > least; };
        for (; at + NW < closed_stop; at += NW) w.template tile<true>(at, at + NW, k, v, side, cut(at));
        w.template tile<false>(at, 0, k, v, side, cut(at));
        at += NW;
    } else
        w.load_query(real);
    if (at < stop) w.tail(end);
    w.l = sum_over_groups(w.l);

    if constexpr (NW > 1) {
        if (real) {
#pragma unroll
            for (int j = 0; j < A::NJ; ++j) *(f32x4*)&merged[wave][w.c][16 * j + 4 * w.g] = w.o[j];
            if (w.g == 0) {
                merged[wave][w.c][D] = w.m;
                merged[wave][w.c][D + 1] = w.l;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 4); i += NW * 64) {
            const int cc = i / (D / 4), d = (i - cc * (D / 4)) * 4, rr = rg * 16 + cc;
            if (rr >= a.rows) break;
            float m = M_FLOOR, l = 0.f;
            f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < NW; ++x) m = fmaxf(m, merged[x][cc][D]);
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float f = __builtin_amdgcn_exp2f(merged[x][cc][D] - m);
                l = fmaf(merged[x][cc][D + 1], f, l);
                o += *(const f32x4*)&merged[x][cc][d] * f;
            }
            if (a.part) {
                float* p = a.part + ((w.bh * a.rows + rr) * a.n_split + split) * (D + 2);
#pragma unroll
                for (int r = 0; r < 4; ++r) p[d + r] = o[r];
                if (d == 0) {
                    p[D] = m;
                    p[D + 1] = l;
                }
            } else {
                const int tt = rr / a.share;
                T* y = (T*)a.out + (b * a.q_len + tt) * a.ldo + (int64_t)(h0 + rr - tt * a.share) * D + d;
                const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
                for (int r = 0; r < 4; ++r) Elem<T>::store(y + r, o[r] * inv);
            }
        }
    } else if (real) {
        if (a.part) {
            float* p = a.part + ((w.bh * a.rows + row) * a.n_split + split) * (D + 2);
#pragma unroll
            for (int j = 0; j < A::NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) p[16 * j + 4 * w.g + r] = w.o[j][r];
            if (w.g == 0) {
                p[D] = w.m;
                p[D + 1] = w.l;
            }
        } else {
            T* y = (T*)a.out + (b * a.q_len + t) * a.ldo + (int64_t)h * D;
            const float inv = w.l == 0.f ? 0.f : 1.0f / w.l;
#pragma unroll
            for (int j = 0; j < A::NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) Elem<T>::store(y + 16 * j + 4 * w.g + r, w.o[j][r] * inv);
        }
    }
}

// Joins the splits of one row: a workgroup each.  Thread x sums column x % D of every (256 / D)-th split, so that the loads of a row are
// 256 / D splits abreast and independent of each other; the 256 / D partial sums meet in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_kv8_join_kernel(AttnArgs a) {
    constexpr int G = 256 / D;
    __shared__ float part[G][D + 1], most[4];
    const int tid = threadIdx.x, d = tid % D, sub = tid / D;
    const int64_t bh = blockIdx.x / a.rows;
    const int row = (int)(blockIdx.x - bh * a.rows);
    const float* p = a.part + (int64_t)blockIdx.x * a.n_split * (D + 2);
    float m = M_FLOOR;
    for (int s = tid; s < a.n_split; s += 256) m = fmaxf(m, p[(int64_t)s * (D + 2) + D]);
    m = max64(m);
    if ((tid & 63) == 0) most[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    float l = 0.f, o = 0.f;
#pragma unroll 4
    for (int s = sub; s < a.n_split; s += G) {
        const float* ps = p + (int64_t)s * (D + 2);
        const float f = __builtin_amdgcn_exp2f(ps[D] - m);
        l = fmaf(ps[D + 1], f, l);
        o = fmaf(ps[d], f, o);
    }
    part[sub][d] = o;
    if (d == 0) part[sub][D] = l;
    __syncthreads();
    if (tid >= D) return;
    l = o = 0.f;
#pragma unroll
    for (int x = 0; x < G; ++x) {
        o += part[x][d];
        l += part[x][D];
    }
    const int64_t b = bh / a.c.kv_heads;
    const int t = row / a.share, h = (int)(bh - b * a.c.kv_heads) * a.share + row - t * a.share;
    Elem<T>::store((T*)a.out + (b * a.q_len + t) * a.ldo + (int64_t)h * D + d, l == 0.f ? 0.f : o / l);
}

template <typename T, int D>
static void launch_attention(const AttnArgs& a, int64_t groups, hipStream_t s) {
    const int64_t grid = groups * a.n_split;
    // Four waves to a head's rows where heads are few, one where there would be more workgroups of four than the card holds at a time
    // (two to a CU): 512 heads x 543 rows 19.0 against 22.5 us, 768 heads 31.6 against 25.9, 2048 heads 70.9 against 54.7.
    if (grid > 512)
        hipLaunchKernelGGL((attention_kv8_kernel<T, D, 1>), dim3((unsigned)grid), dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL((attention_kv8_kernel<T, D, 4>), dim3((unsigned)grid), dim3(256), 0, s, a);
    if (a.n_split > 1)
        hipLaunchKernelGGL((attention_kv8_join_kernel<T, D>), dim3((unsigned)(a.c.batch * a.c.kv_heads * a.rows)), dim3(256), 0, s, a);
}

static int check_cache(const char* who, int dtype, const bt_kv8_cache* c, int* shift) {
    BT_CHECK_ARG(dtype == BT_F32 || dtype == BT_BF16, "%s: bad dtype %d", who, dtype);
    BT_CHECK_ARG(c, "%s: null cache", who);
    BT_CHECK_ARG(c->struct_size == sizeof(bt_kv8_cache), "%s: bt_kv8_cache.struct_size %u, this library expects %zu", who, c->struct_size,
                 sizeof(bt_kv8_cache));
    BT_CHECK_ARG(c->block == 16 || c->block == 32 || c->block == 64, "%s: block %d is not 16, 32 or 64", who, c->block);
    BT_CHECK_ARG(c->head_dim == 32 || c->head_dim == 64 || c->head_dim == 128, "%s: head_dim %d not instantiated", who, c->head_dim);
    BT_CHECK_ARG(c->batch >= 0 && c->kv_heads > 0 && c->batch < (1ll << 31) && c->batch * c->kv_heads < (1ll << 31),
                 "%s: bad batch or kv_heads", who);
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

// BT_KV8(type, head_dim, block) for the cache's
#define BT_KV8_BLOCK(T, D_, block) ((block) == 16 ? (void)(BT_KV8(T, D_, 16)) : (block) == 32 ? (void)(BT_KV8(T, D_, 32)) : (void)(BT_KV8(T, D_, 64)))
#define BT_KV8_DIM(T, d, block) ((d) == 32 ? BT_KV8_BLOCK(T, 32, block) : (d) == 64 ? BT_KV8_BLOCK(T, 64, block) : BT_KV8_BLOCK(T, 128, block))
#define BT_KV8_DISPATCH(dtype, d, block) ((dtype) == BT_BF16 ? BT_KV8_DIM(bf16, d, block) : BT_KV8_DIM(float, d, block))

static Rows rows_of(const bt_kv8_rows* r) { return r ? Rows{(char*)r->p, r->b_stride, r->t_stride, r->h_stride} : Rows{nullptr, 0, 0, 0}; }

}  // namespace bt

using namespace bt;

extern "C" int bt_kv8_append(int dtype, const bt_kv8_cache* cache, int32_t q_len, int32_t heads, const bt_kv8_rows* q,
                             const bt_kv8_rows* q_out, const bt_kv8_rows* k, const bt_kv8_rows* v, const int32_t* pos0_dev,
                             int32_t pos0_host, const int32_t* pos_table, int32_t rot, const float* cos_tab, const float* sin_tab,
                             int64_t max_pos, bt_stream stream) {
    AppendArgs a{};
    int shift;
    BT_TRY(check_cache("bt_kv8_append", dtype, cache, &shift));
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
    a.blocks = pos0_dev ? (int)(((int64_t)q_len + cache->block - 2) / cache->block) + 1
                        : (int)(((int64_t)pos0_host + q_len - 1) / cache->block - pos0_host / cache->block) + 1;
    // Blocks that fill up have a wave for K and one for V, steps that fill none (or may: the device knows) one for both: 32 x 509 rows 88 us
    // and 97, 8 x 100 9.8 and 14.9; a step of 256 sequences that fills no block 9.8 and 7.5, and of a step whose position the device
    // reads, one row at a time, at most one in 16 fills its blocks.
    a.split = pos0_dev ? q_len > 1 : ((int64_t)pos0_host + q_len) / cache->block > pos0_host / cache->block;
    const int64_t kv_items = (cache->batch * cache->kv_heads * a.blocks) << a.split;
    BT_CHECK_ARG(!q || (double)cache->batch * q_len * heads < (double)(1 << 30), "bt_kv8_append: too many rows for one call");
    const int64_t q_rows = q ? cache->batch * q_len * heads : 0;
    const int V = dtype == BT_BF16 ? 8 : 4;
    BT_CHECK_ARG(kv_items < (1ll << 25) && ceil_div(q_rows * cache->head_dim, 256 * V) < (1ll << 25),
                 "bt_kv8_append: too many rows for one call");      // (2^32 threads)
    a.kv_items = (uint32_t)kv_items;
    a.q_rows = (uint32_t)q_rows;
    a.q_len = q_len;
    a.heads = heads;
    a.rot = rot;
    a.pos0_host = pos0_host;
    a.pos0_dev = pos0_dev;
    a.pos_table = pos_table;
    a.cos_tab = cos_tab;
    a.sin_tab = sin_tab;
    a.max_pos = max_pos;
    a.vec_rope = (rot / 2) % V == 0 && aligned16(cos_tab) && aligned16(sin_tab);
    const int64_t waves = kv_items + ceil_div(q_rows * cache->head_dim, 256 * V);
    const dim3 grid((unsigned)ceil_div(waves, 4));
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ROPE, s);
#define BT_KV8(T, D_, BL_) kv8_append_kernel<T, D_, BL_><<<grid, dim3(256), 0, s>>>(a)
    BT_KV8_DISPATCH(dtype, cache->head_dim, cache->block);
#undef BT_KV8
    BT_LAUNCH_CHECK("bt_kv8_append launch");
    return BT_OK;
}

extern "C" int bt_kv8_read(int dtype, const bt_kv8_cache* cache, int64_t n, int64_t first, int64_t count, void* k_out, void* v_out,
                           bt_stream stream) {
    int shift;
    BT_TRY(check_cache("bt_kv8_read", dtype, cache, &shift));
    BT_CHECK_ARG(n >= 0 && n <= cache->n_max && first >= 0 && count >= 0 && first <= n && count <= n - first,
                 "bt_kv8_read: rows out of range");
    BT_CHECK_ARG((!k_out || aligned16(k_out)) && (!v_out || aligned16(v_out)), "bt_kv8_read: outputs must be 16-byte aligned");
    if (cache->batch == 0 || count == 0 || (!k_out && !v_out)) return BT_OK;
    const int blocks = (int)((first + count - 1) / cache->block - first / cache->block) + 1;
    const int64_t waves = cache->batch * cache->kv_heads * blocks;
    BT_CHECK_ARG(waves < (1ll << 26), "bt_kv8_read: grid too large");      // (2^32 threads)
    const dim3 grid((unsigned)ceil_div(waves, 4));
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ROPE, s);
#define BT_KV8(T, D_, BL_) kv8_read_kernel<T, D_, BL_><<<grid, dim3(256), 0, s>>>(*cache, n, first, count, blocks, (T*)k_out, (T*)v_out)
    BT_KV8_DISPATCH(dtype, cache->head_dim, cache->block);
#undef BT_KV8
    BT_LAUNCH_CHECK("bt_kv8_read launch");
    return BT_OK;
}

// One workgroup to a CU, none with less than two 64-row tiles, 64 splits at most; fewer than three are not worth the second launch of 4 us.
// Measured at 16 heads of one sequence: 543 rows 10.7 us whole, 9.2 in 4; 2000 rows 15.9 and 9.2 in 16; 32768 rows 163 and 27.6 in 16 (32: 27.7);
// at 128 heads 543 rows 11.0 whole, 11.8 in 2.
extern "C" int32_t bt_attention_kv8_split_count(int64_t batch, int32_t kv_heads, int32_t group, int32_t q_len, int64_t n) {
    const int64_t groups = batch * kv_heads * ceil_div((int64_t)group * q_len, 16), tiles = ceil_div(n, 64);
    if (groups <= 0) return 1;
    const int64_t s = std::min<int64_t>(std::min(256 / groups, tiles / 2), 64);
    return s < 3 ? 1 : (int32_t)s;
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
    BT_CHECK_ARG(!mask || mask_ld == 0 || mask_ld >= (pos0_dev ? cache->n_max : (int64_t)pos0_host + q_len),
                 "bt_attention_kv8: mask row too short");      // (0: one row for all sequences)
    BT_CHECK_ARG(n_split >= 1, "bt_attention_kv8: bad n_split %d", n_split);
    const int64_t need = bt_attention_kv8_workspace_bytes(cache->batch, q_len, heads, cache->head_dim, n_split);
    if (need > 0 && (!ws || ws_bytes < need || !aligned16(ws))) {
        set_error("bt_attention_kv8: split workspace too small or unaligned (%lld < %lld bytes)", (long long)ws_bytes, (long long)need);
        return BT_ERR_WORKSPACE;
    }
    a.c = *cache;
    a.q = rows_of(q);
    a.q_len = q_len;
    a.heads = heads;
    a.share = heads / cache->kv_heads;
    BT_CHECK_ARG((int64_t)q_len * a.share < (1ll << 30), "bt_attention_kv8: too many rows");
    a.rows = q_len * a.share;
    a.row_groups = (a.rows + 15) / 16;
    a.n_split = n_split;
    a.part = n_split > 1 ? (float*)ws : nullptr;
    const int64_t groups = cache->batch * cache->kv_heads * a.row_groups;
    BT_CHECK_ARG(groups < (1ll << 26) && groups * n_split < (1ll << 26) && (n_split == 1 || cache->batch * cache->kv_heads * a.rows < (1ll << 24)),
                 "bt_attention_kv8: grid too large");      // (2^32 threads)
    a.pos0_host = pos0_host;
    a.pos0_dev = pos0_dev;
    a.mask = mask;
    a.mask_ld = mask_ld;
    a.out = out;
    a.ldo = ldo;
    a.scale = 1.4426950408889634f / sqrtf((float)cache->head_dim);
    hipStream_t s = (hipStream_t)stream;
    ProfScope ps(BT_PROF_ATTN_ROWS, s);
#define BT_ATT8(D_) (dtype == BT_BF16 ? launch_attention<bf16, D_>(a, groups, s) : launch_attention<float, D_>(a, groups, s))
    switch (cache->head_dim) {
        case 32: BT_ATT8(32); break;
        case 64: BT_ATT8(64); break;
        default: BT_ATT8(128);
    }
#undef BT_ATT8
    BT_LAUNCH_CHECK("bt_attention_kv8 launch");
    return BT_OK;
}
