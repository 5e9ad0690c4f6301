// Attention with a learned relative position bias by buckets, fused, and its gradients:
//   s_ij = scale q_i . k_j + table[map[clip(j - p_i, -R, R) + R]][h]   for j < klen_b (causal: and j <= p_i),   p_i = qstart_b + i
//   P = softmax(s), o = P v, lse_i = log sum_j e^s_ij;   a row without keys: o = 0, lse = -inf, no gradient
//   dS = P (dO v^T - D), D_i = sum_c dO_ic o_ic;  dq = scale dS k;  dk = scale dS^T q;  dv = P^T dO;  dtable[n][h] = sum of dS where map = n
// The bias is never materialised: a head's 2R + 1 values lie in LDS (padded so that a tile near the diagonal indexes them without a clamp), and a
// tile farther than R from the diagonal sees one value.  All products run on 16x16 matrix instructions (K = 32 for sixteen-bit elements, four
// K = 4 steps for fp32), softmax statistics and sums in fp32.  The matrix unit takes both operands in one type, so P (before P v and P^T dO) and dS (before
// dS k and dS^T q) are rounded to the tensors' sixteen-bit type, relative to the largest of their column: off by half a step of each, which averages out
// over the keys - the output is then off by 1.3 to 1.5 times its own rounding.  Two numbers of the type instead of one cost another product each: free where
// the kernel waits for memory (few queries, which does that), a third of the products in the others.  The softmax's sum, D and the table's
// gradient take P and dS unrounded.  Every product is arranged so that its result's columns are the axis the
// wave owns (queries in the forward and dq passes, keys in the dk / dv pass): scores come out with a query's keys in one lane's registers, and go
// straight back in as the next product's right operand - P and dS never pass through LDS.  Their key order inside a K = 32 step
// (16 (j / 4) + 4 (lane / 16) + j % 4) is matched by reading the other operand transposed from its row-major tile.
// dk / dv and dq are two passes (S and dP computed twice: 14 ch operations a pair of query and key instead of 10): dq stays in registers, nothing is
// added by atomics from several workgroups, the bits are the same in every run.
#pragma once
#include <atomic>
#include "elem.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int RMAX = 1024;
constexpr int NWAVE = 4, NTHR = 64 * NWAVE;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

// A fragment covers KSTEP of the summed axis: 32 sixteen-bit elements (8 a lane), 16 fp32 ones (4 a lane).
template <typename T> struct Frag;
template <> struct Frag<float> { typedef f32x4 type; static constexpr int N = 4; };
template <> struct Frag<bf16_t> { typedef bf16x8 type; static constexpr int N = 8; };
template <> struct Frag<f16_t> { typedef f16x8 type; static constexpr int N = 8; };

// D[16 x 16] += A[16 x 4N] B[4N x 16]: lane l holds A[l % 16][N (l / 16) + j], B[N (l / 16) + j][l % 16], D[4 (l / 16) + r][l % 16].  fp32: four
// K = 4 instructions, the j-th over the lanes' j-th elements - the order of the summed axis is free as long as A and B agree.
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
constexpr f32x4 ZERO4 = {0.f, 0.f, 0.f, 0.f};

struct AttP {
    const void *q, *k, *v, *table, *out, *dout, *olo_in;
    void *o, *olo, *dq, *dk, *dv, *dtable;
    long qb, qr, kb, kr, vb, vr, ob, orow, db, dr, dqb, dqr, dkb, dkr, dvb, dvr;      // batch and row strides, elements
    const int32_t *map, *klen, *qstart;
    float *lse, *dsum, *diag, *part, *part_ml, *kv_part;
    int B, Tq, Tk, H, Hk, ch, R, nb, causal, table_dtype, splits, qsplits, nblk, swz;
    float scale;
};

// Shapes of the tiles of a type and a padded head width (a multiple of 16).
template <typename T, int CHP> struct Shape {
    static constexpr bool F32 = sizeof(T) == 4;
    // fp16 ends at 2^-24 and 65504: the backward passes take P and dS times powers of two there (P_SHIFT, in_range); bf16 and fp32 hold them as they are
    static constexpr bool NARROW = __is_same(T, f16_t);
    static constexpr float P_SHIFT = NARROW ? 14.f : 0.f;   // log2
    static constexpr int KSTEP = 4 * Frag<T>::N, NP = KSTEP / 16;   // summed elements of one product; result tiles that feed one
    static constexpr int KW = (CHP + KSTEP - 1) / KSTEP * KSTEP, KS = KW / KSTEP, CT = CHP / 16;
    static constexpr int KT = F32 ? 32 : 64;              // rows of a staged tile
    static constexpr int NQ = F32 ? 1 : 2;                // 16-query column tiles of a wave: each fragment read from LDS feeds NQ products
    static constexpr int NK = F32 || CHP > 64 ? 1 : 2;    // 16-key column tiles of a wave in the dk / dv pass (its accumulators are twice as many)
    static constexpr int QB = 16 * NQ * NWAVE, KB = 16 * NK * NWAVE;
    static constexpr int PITCH = KW + 16 / (int)sizeof(T);   // elements: 16 rows' 16-byte pieces fall on distinct banks
    static constexpr int PAD = KT + 16 * NQ;                // bias values beyond +-R that a tile near the diagonal can index
    static constexpr size_t TILE = (size_t)KT * PITCH * sizeof(T);
};

// Workgroup -> (batch, kv head, query head, block): the blocks of one kv head stay on one of the eight XCDs (consecutive workgroups go
// round them), so its keys and values are fetched into one L2 - where there are enough kv heads to fill all eight.
struct Where { int b, h, hk, blk; };
__device__ __forceinline__ Where place(const AttP& p, int heads_inner, unsigned id) {
    const unsigned inner = (unsigned)heads_inner * p.nblk;
    unsigned unit, in;
    if (p.swz) {
        const unsigned x = id & 7, i = id >> 3;
        unit = x + 8 * (i / inner);
        in = i % inner;
    } else {
        unit = id / inner;
        in = id % inner;
    }
    Where w;
    w.b = (int)(unit / p.Hk);
    w.hk = (int)(unit % p.Hk);
    w.h = w.hk * (p.H / p.Hk) + (int)(in / p.nblk);
    w.blk = (int)(in % p.nblk);
    return w;
}

__device__ __forceinline__ int keys_of(const AttP& p, int b) { return p.klen ? min(max(p.klen[b], 0), p.Tk) : p.Tk; }
__device__ __forceinline__ int start_of(const AttP& p, int b) { return p.qstart ? min(max(p.qstart[b], -(1 << 30)), 1 << 30) : 0; }

// Bias of head h at clipped distance index i in [0, 2R], in log2 units; a map entry outside [0, nb) adds nothing, a value below -1e30 (a mask of the
// type's lowest value) is -inf: in log2 units it would leave fp32's range.  Finite values are taken as between -BIAS_MAX and BIAS_MAX, the range of fp16:
// beside -1e9 a score, the row's maximum and lse have no digits left, P as the gradients compute it again would be 2^(+-64), and what such a bias says -
// not to be seen beside any other key - -BIAS_MAX says as well.
constexpr float BIAS_MAX = 65504.f;
__device__ __forceinline__ float bias_at(const AttP& p, int h, int i) {
    const int m = p.map[i];
    if (m < 0 || m >= p.nb) return 0.f;
    const long at = (long)m * p.H + h;
    const float v = p.table_dtype == DUA_DTYPE_F32 ? ((const float*)p.table)[at]
                                                   : (p.table_dtype == DUA_DTYPE_BF16 ? (float)((const bf16_t*)p.table)[at] : (float)((const f16_t*)p.table)[at]);
    if (v < -1e30f) return -INFINITY;
    return LOG2E * (v < -BIAS_MAX ? -BIAS_MAX : (v > BIAS_MAX && v < INFINITY ? BIAS_MAX : v));       // (+inf and NaN stay)
}
// lut[rel + R + pad], rel clipped to [-R, R]
__device__ __forceinline__ void load_lut(const AttP& p, int h, int pad, float* lut) {
    const int n = 2 * (p.R + pad) + 1;
    for (int i = threadIdx.x; i < n; i += NTHR) lut[i] = bias_at(p, h, min(max(i - pad, 0), 2 * p.R));
}

template <typename T> using Vec16 = typename VecOf<T, Elem<T>::VEC>::type;

template <typename T>
__device__ __forceinline__ Vec16<T> zero16() {
    Vec16<T> r;
#pragma unroll
    for (int j = 0; j < Elem<T>::VEC; ++j) r[j] = (T)0.f;
    return r;
}
// 16 bytes of a row from column c on, zeros at and past ch (a multiple of 16 bytes): the load is unconditional, from the row's own elements where
// there are none, and what does not count is zeroed when it is used.  (Loads behind lanes' conditions are waited for at once: the zeros
// go to their registers.)
template <typename T>
__device__ __forceinline__ Vec16<T> load16(const T* row, int c, int ch) { return *(const typename MemVec<T, Elem<T>::VEC>::type*)(row + min(c, ch - Elem<T>::VEC)); }
template <typename T>
__device__ __forceinline__ Vec16<T> keep16(Vec16<T> x, int c, int ch, bool there) { return there && c < ch ? x : zero16<T>(); }

// A lane's part of a fragment from global memory (16 bytes); a row that is not there (`row` may be any that is) reads as zeros
template <typename T>
__device__ __forceinline__ typename Frag<T>::type row_frag_global(const T* row, int c, int ch, bool there) {
    static_assert(Frag<T>::N == Elem<T>::VEC, "a lane's part of a fragment is 16 bytes");
    return keep16<T>(load16<T>(row, c, ch), c, ch, there);
}

// A tile of ROWS rows on its way from global memory through registers to LDS: the loads of the next tile are in flight while the present one
// is multiplied.  Rows at and past n (n > 0) and the columns past ch are zeros.
template <typename T, int CHP, int ROWS, int THREADS = NTHR> struct Carrier {
    static constexpr int V = Elem<T>::VEC, C = Shape<T, CHP>::KW / V, P = Shape<T, CHP>::PITCH, N = (ROWS * C + THREADS - 1) / THREADS;
    static constexpr bool EVEN = ROWS * C % THREADS == 0;
    Vec16<T> x[N];
    unsigned off[N];                                         // bytes from a tile's first row (row strides are below 2^24 elements)
    int rows;
    __device__ __forceinline__ Carrier(long stride, int ch, int tid) {
#pragma unroll
        for (int u = 0; u < N; ++u) off[u] = at(u, ROWS, stride, ch, tid);
    }
    __device__ static __forceinline__ unsigned at(int u, int n, long stride, int ch, int tid) {
        const int i = tid + u * THREADS, r = i / C, c = i % C * V;
        return ((unsigned)min(r, n - 1) * (unsigned)stride + (unsigned)min(c, ch - V)) * (unsigned)sizeof(T);
    }
    __device__ __forceinline__ void fetch(const T* src, long stride, int n, int ch, int tid) {
        rows = n;
        const char* s = (const char*)src;
        if (n >= ROWS) {
#pragma unroll
            for (int u = 0; u < N; ++u) x[u] = *(const typename MemVec<T, V>::type*)(s + off[u]);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) x[u] = *(const typename MemVec<T, V>::type*)(s + at(u, n, stride, ch, tid));
        }
    }
    __device__ __forceinline__ void put(T* tile, int ch, int tid) const {
        if (rows >= ROWS && ch == Shape<T, CHP>::KW) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = tid + u * THREADS, r = i / C, c = i % C * V;
                if (EVEN || r < ROWS) *(Vec16<T>*)(tile + r * P + c) = x[u];
            }
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = tid + u * THREADS, r = i / C, c = i % C * V;
                if (EVEN || r < ROWS) *(Vec16<T>*)(tile + r * P + c) = keep16<T>(x[u], c, ch, r < rows);
            }
        }
    }
};

// Fragment of a row-major tile: lane -> row row0 + l % 16, its part of columns c .. c + KSTEP - 1
template <typename T>
__device__ __forceinline__ typename Frag<T>::type row_frag(const T* tile, int pitch, int row0, int c, int lane) {
    return *(const typename Frag<T>::type*)(tile + (row0 + (lane & 15)) * pitch + c + Frag<T>::N * (lane >> 4));
}
// The same tile transposed: lane -> column c0 + l % 16, element j -> row row0 + 16 (j / 4) + 4 (l / 16) + j % 4.  Sixteen-bit elements by two
// transposing LDS reads (each 16-lane group reads a block of 4 rows x 16 columns, a lane gets its column's 4 rows).
template <typename T>
__device__ __forceinline__ typename Frag<T>::type col_frag(const T* tile, int pitch, int row0, int c0, int lane) {
    typename Frag<T>::type f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = tile[(row0 + 4 * (lane >> 4) + j) * pitch + c0 + (lane & 15)];
    } else {
        typedef short s4 __attribute__((__vector_size__(8)));
        const T* a = tile + (row0 + 4 * (lane >> 4) + ((lane & 15) >> 2)) * pitch + c0 + 4 * (lane & 3);
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)a);
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(a + 16 * pitch));
        struct { s4 lo, hi; } pr{x, y};
        __builtin_memcpy(&f, &pr, 16);
    }
    return f;
}
// NP result tiles as the right operand of the next product
template <typename T>
__device__ __forceinline__ typename Frag<T>::type acc_frag(const f32x4* a) {
    if constexpr (sizeof(T) == 4) {
        return a[0];
    } else {
        typename Frag<T>::type f;
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = (T)a[0][j]; f[4 + j] = (T)a[1][j]; }
        return f;
    }
}

// four consecutive channels of a row
template <typename T>
__device__ __forceinline__ void store4(T* row, int c, int ch, f32x4 v) {
    if (c >= ch) return;
    typename VecOf<T, 4>::type x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (T)v[j];
    *(typename MemVec<T, 4>::type*)(row + c) = x;
}
// what the rounding to T left of v
template <typename T>
__device__ __forceinline__ f32x4 rest4(f32x4 v) {
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = v[j] - (float)(T)v[j];
    return r;
}

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// max / sum over the four lanes that share a column
__device__ __forceinline__ float col_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float col_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// dS as fp16 operands.  Its size is the incoming gradient's, from 1e-9 (a mean over many tokens) to past 65504 (loss scaling), so it is multiplied by a
// power of two f of the result column's own (a query of dq, a key of dk), whose accumulators carry the same factor until they are stored: exact, and every
// operand is rounded relative to the column's largest one (to 2^-11 of its own size down to 2^-21 of that, to 2^-32 of the largest below).  f falls when a
// value would pass 2^15, to where the largest is in [2^7, 2^8): with the first values that count, then hardly ever.  Rounded unscaled, a dO of 1e-5 lost
// half of dq.
constexpr float F_START = 0x1p100f;
__device__ __forceinline__ float pow2_inverse(float f) { return __int_as_float(0x7F000000 - __float_as_int(f)); }
template <int NP, int CT>
__device__ __forceinline__ void in_range(f32x4* e, float& f, f32x4* acc) {
    float mx = 0.f;
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(e[n][r]));
    if (__any(mx * f > 32768.f)) {
        const float top = col_max(mx);
        if (top * f > 32768.f) {                                            // (then top > 2^-85, or infinite: exponents stay in [-120, 92])
            const float nf = __int_as_float((127 + 8 - __builtin_amdgcn_frexp_expf(top)) << 23), by = nf * pow2_inverse(f);
#pragma unroll
            for (int c = 0; c < CT; ++c) acc[c] *= by;
            f = nf;
        }
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) e[n] *= f;
}

// Where a tile of keys [k0, k0 + n) lies for queries at positions [pmin, pmax]: -1 / 1: all of it at least R to the left / right (one bias value), 0: near.
__device__ __forceinline__ int side_of(int k0, int n, int pmin, int pmax, int R) { return k0 + n - 1 - pmin <= -R ? -1 : (k0 - pmax >= R ? 1 : 0); }

// ... the scores of N16 result tiles (rows: keys k0 + 16 n + 4 (l / 16) + r; column: a query at pos) become log2 logits: raw * sl + bias,
// places past nk or (causal) past pos -inf.  lut points at distance 0.
template <int N16>
__device__ __forceinline__ void bias_mask(f32x4* s, float sl, const float* lut, int side, float b, bool masked, int k0, int nk, int pos, bool causal, int lane) {
    const int key = k0 + 4 * (lane >> 4);
    if (side) {
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = s[n][r] * sl + b;
    } else {
        const float* l = lut + (key - pos);
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = s[n][r] * sl + l[16 * n + r];
    }
    if (masked) {
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int kk = key + 16 * n + r;
                if (kk >= nk || (causal && kk > pos)) s[n][r] = -INFINITY;
            }
    }
}

template <int N16>
__device__ __forceinline__ float max_of(const f32x4* s) {
    float m = s[0][0];
#pragma unroll
    for (int n = 0; n < N16; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, s[n][r]);
    return m;
}

// ---------------------------------------------------------------------------------------------------------------------- host
[[maybe_unused]] static int check_common(const dua_rel_attention_args* a, const char* who, bool backward) {
    DUA_REQUIRE(a, "%s: null arguments", who);
    DUA_REQUIRE(dua_dtype_ok(a->dtype) && dua_dtype_ok(a->table_dtype) && (a->table_dtype == DUA_DTYPE_F32 || a->table_dtype == a->dtype),
                "%s: dtype must be fp32, bf16 or fp16 and the table's fp32 or the same", who);
    DUA_REQUIRE(a->B >= 0 && a->Tq >= 0 && a->Tk >= 0 && a->Tq < (1 << 29) && a->Tk < (1 << 29), "%s: lengths must be in [0, 2^29)", who);
    DUA_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0 && a->heads <= 65535, "%s: kv_heads must divide heads (at most 65535)", who);
    DUA_REQUIRE(a->ch >= 1 && a->ch <= 128 && a->ch * dua_dtype_size(a->dtype) % 16 == 0,
                "%s: head width must be a multiple of 8 (fp32: 4) up to 128", who);
    DUA_REQUIRE(a->radius >= 1 && a->radius <= RMAX && a->num_buckets >= 1, "%s: radius must be in [1, %d]", who, RMAX);
    for (long r : {a->q_row, a->k_row, a->v_row, a->out_row, a->dout_row, a->dq_row, a->dk_row, a->dv_row})
        DUA_REQUIRE(r >= 0 && r < (1L << 24), "%s: row strides must be in [0, 2^24) elements", who);
    DUA_REQUIRE(a->table && a->bucket_map, "%s: null table / bucket map", who);
    DUA_REQUIRE((a->B == 0 || a->Tq == 0 || a->q) && (a->B == 0 || a->Tk == 0 || (a->k && a->v)), "%s: null operand", who);
    // workgroups of a launch: at most one for 64 queries of a head, in the backward pass for 64 keys too (the factors one by one: no overflow)
    const long heads = (long)a->B * a->heads, blocks = (backward && a->Tk > a->Tq ? a->Tk : a->Tq) / 64 + 1;
    DUA_REQUIRE(heads < (1L << 23) && heads * blocks < (1L << 23), "%s: too many blocks for one launch", who);
    return DUA_OK;
}

[[maybe_unused]] static AttP pack(const dua_rel_attention_args* a) {
    AttP p{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.table = a->table; p.o = a->out; p.out = a->out; p.olo = a->out_lo; p.olo_in = a->out_lo; p.dout = a->dout;
    p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.dtable = a->dtable;
    p.qb = a->q_batch; p.qr = a->q_row; p.kb = a->k_batch; p.kr = a->k_row; p.vb = a->v_batch; p.vr = a->v_row; p.ob = a->out_batch; p.orow = a->out_row;
    p.db = a->dout_batch; p.dr = a->dout_row; p.dqb = a->dq_batch; p.dqr = a->dq_row; p.dkb = a->dk_batch; p.dkr = a->dk_row; p.dvb = a->dv_batch; p.dvr = a->dv_row;
    p.map = a->bucket_map; p.klen = a->klen; p.qstart = a->qstart; p.lse = a->lse;
    p.B = a->B; p.Tq = a->Tq; p.Tk = a->Tk; p.H = a->heads; p.Hk = a->kv_heads; p.ch = a->ch; p.R = a->radius; p.nb = a->num_buckets;
    p.causal = a->causal != 0; p.table_dtype = a->table_dtype; p.scale = a->scale;
    return p;
}

[[maybe_unused]] static unsigned grid_of(AttP& p, int heads_inner, int nblk) {
    p.nblk = nblk;
    const long units = (long)p.B * p.Hk, inner = (long)heads_inner * nblk;
    // eight XCDs: only where a last, partly filled round of kv heads does not leave them unevenly loaded
    p.swz = units % 8 == 0 || units >= 64;
    return (unsigned)((p.swz ? (units + 7) / 8 * 8 : units) * inner);
}

[[maybe_unused]] static int chp_of(int ch) { return ch <= 32 ? 32 : ch <= 64 ? 64 : ch <= 80 ? 80 : ch <= 96 ? 96 : 128; }
[[maybe_unused]] static int query_block(int dtype) { return (dtype == DUA_DTYPE_F32 ? 16 : 32) * NWAVE; }        // Shape::QB
[[maybe_unused]] static int key_block(int dtype, int ch) { return (dtype == DUA_DTYPE_F32 || chp_of(ch) > 64 ? 16 : 32) * NWAVE; }   // Shape::KB

// dk / dv where the blocks of keys alone do not fill the chip: a group's query heads are dealt to `heads` workgroups, and of single heads the tiles of
// queries to `tiles`; their sums (fp32) are added in order afterwards.  2 x 8 kv heads of 4 query heads, 940 tokens of 16 bf16, forward and backward: 344 us
// with one workgroup a block of keys (128 in all), 180 with four.  Shares of the queries, backward, 64 wide, 8 heads of 1024 tokens
// a sequence: fp32 (three workgroups a CU) 1 / 2 / 3 sequences (128 / 256 / 384 workgroups) 205 / 208 / 313 us without, 149 / 192 / 273 with 4 / 2 / 2
// shares; bf16 (two workgroups a CU) 64 / 128 workgroups 98 / 101 without, 78 / 88 with 8 / 4 shares; 192 / 256: 101 / 103 and 102 / 104 (256 of 4096
// tokens: 285 and 243) with 2.  Past 512 workgroups they lose: 192 in 3 shares 111, 320 / 384 / 448 in 2 142 / 157 / 167 us, 132 / 132 / 133 without.
struct KeySplits { int heads, tiles; };
[[maybe_unused]] static KeySplits key_splits(const dua_rel_attention_args* a) {
    const int rep = a->heads / a->kv_heads, nkb = (a->Tk + key_block(a->dtype, a->ch) - 1) / key_block(a->dtype, a->ch);
    const long wgs = (long)a->B * a->kv_heads * nkb;
    KeySplits s{1, 1};
    for (int d = 2; d <= rep && wgs * s.heads < 512; ++d)
        if (rep % d == 0) s.heads = d;
    const long now = wgs * s.heads, tiles = a->Tq / (a->dtype == DUA_DTYPE_F32 ? 64 : 128);        // two of Shape::KT
    if (s.heads == rep && now > 0 && now < 512) {
        const long t = a->dtype == DUA_DTYPE_F32 ? (512 + now - 1) / now : 512 / now;
        s.tiles = (int)(t < tiles ? t : (tiles > 1 ? tiles : 1));
    }
    return s;
}

// Workspace of the backward pass: D of every row, the diagonal sums of every head, and of every block of keys (and share of the queries) and head; dk
// and dv of the shares.
[[maybe_unused]] static size_t rel_attention_bwd_floats(const dua_rel_attention_args* a) {
    const size_t rows = (size_t)a->B * a->heads * a->Tq, nkb = (a->Tk + key_block(a->dtype, a->ch) - 1) / key_block(a->dtype, a->ch);
    return (rows + (1 + a->B * nkb * key_splits(a).tiles) * a->heads * (2 * a->radius + 1) + 3) / 4 * 4;
}

[[maybe_unused]] static size_t rel_attention_bwd_bytes(const dua_rel_attention_args* a) {
    const KeySplits k = key_splits(a);
    const int s = k.heads * k.tiles;
    return (rel_attention_bwd_floats(a) + (s > 1 ? 2 * (size_t)s * a->B * a->Tk * a->kv_heads * a->ch : 0)) * sizeof(float);
}

// Launch with `lds` bytes of dynamic LDS; more than 64 KB have to be asked for, once a kernel and device (the call takes microseconds)
template <auto Kernel, typename... A>
int launch(const char* what, dim3 grid, unsigned block, size_t lds, hipStream_t st, A... args) {
    if (lds > 64 * 1024) {
        static std::atomic<unsigned> asked{0};
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        const unsigned bit = 1u << (dev & 31);
        if (e == hipSuccess && !(asked.load() & bit)) {
            e = hipFuncSetAttribute((const void*)Kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
            if (e == hipSuccess) asked.fetch_or(bit);
        }
        if (e != hipSuccess) {
            dua_set_error("%s: %s", what, hipGetErrorString(e));
            return DUA_EHIP;
        }
    }
    hipLaunchKernelGGL(Kernel, grid, block, lds, st, args...);
    return dua_check_launch(what);
}

template <template <typename, int> class L>
int dispatch(int dtype, const AttP& p, bool few, hipStream_t st) {
#define GO(T)                                             \
    switch (chp_of(p.ch)) {                               \
        case 32: return L<T, 32>::run(p, few, st);        \
        case 64: return L<T, 64>::run(p, few, st);        \
        case 80: return L<T, 80>::run(p, few, st);        \
        case 96: return L<T, 96>::run(p, few, st);        \
        default: return L<T, 128>::run(p, few, st);       \
    }
    if (dtype == DUA_DTYPE_F32) { GO(float) } else if (dtype == DUA_DTYPE_BF16) { GO(bf16_t) } else { GO(f16_t) }
#undef GO
}

}  // namespace
