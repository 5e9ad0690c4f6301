// Attention with a learned relative position bias by buckets, fused, and its gradients:
//   s_ij = scale q_i . k_j + table[map[clip(j - p_i, -R, R) + R]][h]   for j < klen_b (causal: and j <= p_i),   p_i = qstart_b + i
//   P = softmax(s), o = P v, lse_i = log sum_j e^s_ij;   a row without keys: o = 0, lse = -inf, no gradient
//   dS = P (dO v^T - D), D_i = sum_c dO_ic o_ic;  dq = scale dS k;  dk = scale dS^T q;  dv = P^T dO;  dtable[n][h] = sum of dS where map = n
// The bias is never materialised: a head's 2R + 1 values lie in LDS (padded so that a tile near the diagonal indexes them without a clamp), and a
// tile farther than R from the diagonal sees one value.  All products run on 16x16 matrix instructions (K = 32 for sixteen-bit elements; fp32
// as eight K = 4 steps on the same fragments), softmax and sums in fp32.  Every product is arranged so that its result's columns are the axis the
// wave owns (queries in the forward and dq passes, keys in the dk / dv pass): scores come out with a query's keys in one lane's registers, and go
// straight back in as the next product's right operand - P and dS never pass through LDS.  Their key order inside a K = 32 step
// (16 (j / 4) + 4 (lane / 16) + j % 4) is matched by reading the other operand transposed from its row-major tile.
// dk / dv and dq are two passes (scores computed twice, 14 instead of 10 products' flops): no atomics, the same bits in every run.
#include "elem.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int RMAX = 1024;
constexpr int NWAVE = 4, NTHR = 64 * NWAVE;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Frag;
template <> struct Frag<float> { typedef f32x8 type; };
template <> struct Frag<bf16_t> { typedef bf16x8 type; };
template <> struct Frag<f16_t> { typedef f16x8 type; };

// D[16 x 16] += A[16 x 32] B[32 x 16]: lane l holds A[l % 16][8 (l / 16) + j], B[8 (l / 16) + j][l % 16], D[4 (l / 16) + r][l % 16]
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

struct AttP {
    const void *q, *k, *v, *table, *out, *dout;
    void *o, *dq, *dk, *dv, *dtable;
    long qb, qr, kb, kr, vb, vr, ob, orow, db, dr, dqb, dqr, dkb, dkr, dvb, dvr;      // batch and row strides, elements
    const int32_t *map, *klen, *qstart;
    float *lse, *dsum, *part;
    int B, Tq, Tk, H, Hk, ch, R, nb, causal, table_dtype, vec, splits, nblk, swz;
    float scale;
};

// Shapes of the tiles of a type and a padded head width.
template <typename T, int CHP> struct Shape {
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int KT = F32 ? 32 : 64;              // rows of a staged tile
    static constexpr int NQ = F32 ? 1 : (CHP > 64 ? 1 : 2);
    static constexpr int QB = 16 * NQ * NWAVE;            // columns (queries / keys) of a workgroup
    static constexpr int PITCH = CHP + (F32 ? 4 : 8);     // elements: 16 rows' 16-byte pieces fall on distinct banks
    static constexpr int PAD = KT + 16 * NQ;              // bias values beyond +-R that a tile near the diagonal can index
    static constexpr int KS = CHP / 32, CT = CHP / 16;
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

// Bias of head h in log2 units: lut[rel + R + pad], rel clipped to [-R, R]; a map entry outside [0, nb) adds nothing.
__device__ __forceinline__ void load_lut(const AttP& p, int h, int pad, float* lut, int tid, int nthr) {
    const int n = 2 * (p.R + pad) + 1;
    for (int i = tid; i < n; i += nthr) {
        const int m = p.map[min(max(i - pad, 0), 2 * p.R)];
        float v = 0.f;
        if (m >= 0 && m < p.nb) {
            const long at = (long)m * p.H + h;
            v = p.table_dtype == DUA_DTYPE_F32 ? ((const float*)p.table)[at] : (p.table_dtype == DUA_DTYPE_BF16 ? (float)((const bf16_t*)p.table)[at] : (float)((const f16_t*)p.table)[at]);
        }
        lut[i] = v * LOG2E;
    }
}

// VEC consecutive elements (16 bytes) of a row at column c, zero at and past ch
template <typename T>
__device__ __forceinline__ typename VecOf<T, Elem<T>::VEC>::type load16(const T* row, int c, int ch, bool vec) {
    constexpr int V = Elem<T>::VEC;
    typename VecOf<T, V>::type r;
    if (vec) {
        if (c < ch) return *(const typename VecOf<T, V>::type*)(row + c);
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = (T)0.f;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = c + j < ch ? row[c + j] : (T)0.f;
    }
    return r;
}

// 8 elements of a row as a fragment; a row that is not there reads as zeros
template <typename T>
__device__ __forceinline__ typename Frag<T>::type row_frag_global(const T* row, int c, int ch, bool vec, bool there) {
    typename Frag<T>::type f;
    constexpr int V = Elem<T>::VEC;
#pragma unroll
    for (int i = 0; i < 8; i += V) {
        if (there) {
            const auto x = load16<T>(row, c + i, ch, vec);
#pragma unroll
            for (int j = 0; j < V; ++j) f[i + j] = x[j];
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) f[i + j] = (T)0.f;
        }
    }
    return f;
}

// rows [0, n) of a tile of ROWS rows into LDS, the rest and the columns past ch as zeros
template <typename T, int CHP, int ROWS>
__device__ __forceinline__ void stage(T* tile, const T* src, long stride, int n, int ch, bool vec) {
    constexpr int V = Elem<T>::VEC, C = CHP / V, P = Shape<T, CHP>::PITCH;
#pragma unroll
    for (int i0 = 0; i0 < ROWS * C; i0 += NTHR) {
        const int i = i0 + (int)threadIdx.x, r = i / C, c = i % C * V;
        if (ROWS * C % NTHR != 0 && i >= ROWS * C) break;
        typename VecOf<T, V>::type x;
        if (r < n) {
            x = load16<T>(src + r * stride, c, ch, vec);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = (T)0.f;
        }
        *(typename VecOf<T, V>::type*)(tile + r * P + c) = x;
    }
}

// Fragment of a row-major tile: lane -> row row0 + l % 16, columns c .. c + 7
template <typename T>
__device__ __forceinline__ typename Frag<T>::type row_frag(const T* tile, int pitch, int row0, int c, int lane) {
    const T* a = tile + (row0 + (lane & 15)) * pitch + c + 8 * (lane >> 4);
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = *(const f32x4*)a, y = *(const f32x4*)(a + 4);
        return f32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    } else {
        return *(const typename Frag<T>::type*)a;
    }
}
// The same tile transposed: lane -> column c0 + l % 16, element j -> row row0 + 16 (j / 4) + 4 (l / 16) + j % 4.  Sixteen-bit elements by two
// transposing LDS reads (each 16-lane group reads a block of 4 rows x 16 columns, a lane gets its column's 4 rows).
template <typename T>
__device__ __forceinline__ typename Frag<T>::type col_frag(const T* tile, int pitch, int row0, int c0, int lane) {
    typename Frag<T>::type f;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = tile[(row0 + 16 * (j / 4) + 4 * (lane >> 4) + j % 4) * pitch + c0 + (lane & 15)];
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
// Two result tiles (16 + 16 rows) as the right operand of the next product
template <typename T>
__device__ __forceinline__ typename Frag<T>::type acc_frag(f32x4 a, f32x4 b) {
    typename Frag<T>::type f;
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = (T)a[j]; f[4 + j] = (T)b[j]; }
    return f;
}

// four consecutive channels of a row
template <typename T>
__device__ __forceinline__ void store4(T* row, int c, int ch, bool vec, f32x4 v) {
    if (vec) {
        if (c < ch) {
            typename VecOf<T, 4>::type x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = (T)v[j];
            *(typename VecOf<T, 4>::type*)(row + c) = x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < ch) row[c + j] = (T)v[j];
    }
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

// Scores of a tile in log2 units: S = raw * sl + bias, masked places -inf.  Columns are queries at position pos (this lane's), rows keys k0 + ...
template <int NT16>
__device__ __forceinline__ void bias_mask(f32x4 (&s)[NT16], float sl, const float* lut, int off, int far, float flo, float fhi, bool masked, int k0, int nk, int pos, bool causal, int lane) {
    const int key = k0 + 4 * (lane >> 4);
    if (far) {
        const float b = far < 0 ? flo : fhi;
#pragma unroll
        for (int n = 0; n < NT16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = s[n][r] * sl + b;
    } else {
        const float* l = lut + (key - pos + off);
#pragma unroll
        for (int n = 0; n < NT16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[n][r] = s[n][r] * sl + l[16 * n + r];
    }
    if (masked) {
#pragma unroll
        for (int n = 0; n < NT16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int kk = key + 16 * n + r;
                if (kk >= nk || (causal && kk > pos)) s[n][r] = -INFINITY;
            }
    }
}

// -------------------------------------------------------------------------------------------------------------------- forward
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, 2) void k_rel_attention(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int KT = S::KT, NQ = S::NQ, KS = S::KS, CT = S::CT, P = S::PITCH, N16 = KT / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const Kt = (T*)smem;
    T* const Vt = Kt + KT * P;
    float* const lut = (float*)(Vt + KT * P);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const Where w = place(p, p.H / p.Hk, blockIdx.x);
    if (w.b >= p.B) return;
    const int blk = p.causal ? p.nblk - 1 - w.blk : w.blk;                 // long rows first
    const int q0 = blk * S::QB, nk = keys_of(p, w.b), qs = start_of(p, w.b);
    const bool vec = p.vec;
    load_lut(p, w.h, S::PAD, lut, threadIdx.x, NTHR);
    const int qw = q0 + wave * 16 * NQ, pmin = qs + qw, pmax = pmin + 16 * NQ - 1;
    const T* qp = (const T*)p.q + w.b * p.qb + (long)w.h * p.ch;
    frag qf[NQ][KS];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = row_frag_global<T>(qp + q * p.qr, 32 * s + 8 * g, p.ch, vec, q < p.Tq);
    }
    f32x4 o[NQ][CT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int kend = p.causal ? max(0, min(nk, qs + min(q0 + S::QB, p.Tq))) : nk;
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    const float sl = p.scale * LOG2E;
    for (int k0 = 0; k0 < kend; k0 += KT) {
        __syncthreads();
        stage<T, CHP, KT>(Kt, kp + k0 * p.kr, p.kr, nk - k0, p.ch, vec);
        stage<T, CHP, KT>(Vt, vp + k0 * p.vr, p.vr, nk - k0, p.ch, vec);
        __syncthreads();
        const int far = k0 + KT - 1 - pmin <= -p.R ? -1 : (k0 - pmax >= p.R ? 1 : 0);
        const bool masked = k0 + KT > nk || (p.causal && k0 + KT - 1 > pmin);
        const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int pos = pmin + 16 * i + (lane & 15);
            f32x4 s[N16];
#pragma unroll
            for (int n = 0; n < N16; ++n) {
                s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) s[n] = mma(row_frag<T>(Kt, P, 16 * n, 32 * ks, lane), qf[i][ks], s[n]);
            }
            bias_mask<N16>(s, sl, lut, p.R + S::PAD, far, flo, fhi, masked, k0, nk, pos, p.causal, lane);
            float mx = s[0][0];
#pragma unroll
            for (int n = 0; n < N16; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[n][r]);
            const float mn = fmaxf(m[i], col_max(mx)), ms = mn == -INFINITY ? 0.f : mn;
            const float f = exp2_raw(m[i] - ms);
            m[i] = mn;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < N16; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[n][r] = exp2_raw(s[n][r] - ms);
                    sum += s[n][r];
                }
            l[i] = l[i] * f + sum;
#pragma unroll
            for (int c = 0; c < CT; ++c) o[i][c] *= f;
#pragma unroll
            for (int kb = 0; kb < N16 / 2; ++kb) {
                const frag pf = acc_frag<T>(s[2 * kb], s[2 * kb + 1]);
#pragma unroll
                for (int c = 0; c < CT; ++c) o[i][c] = mma(col_frag<T>(Vt, P, 32 * kb, 16 * c, lane), pf, o[i][c]);
            }
        }
    }
    T* op = (T*)p.o + w.b * p.ob + (long)w.h * p.ch;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        const float lt = col_sum(l[i]), inv = lt > 0.f || lt != lt ? 1.0f / lt : 0.f;
        if (q >= p.Tq) continue;
#pragma unroll
        for (int c = 0; c < CT; ++c) store4<T>(op + q * p.orow, 16 * c + 4 * g, p.ch, vec, o[i][c] * inv);
        if (p.lse && g == 0) p.lse[((long)w.b * p.H + w.h) * p.Tq + q] = lt == 0.f ? -INFINITY : (m[i] + log2f(lt)) * LN2;
    }
}

// ------------------------------------------------------------------------------------------------------------------ dq, dtable
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, 2) void k_rel_attention_dq(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int KT = S::KT, NQ = S::NQ, KS = S::KS, CT = S::CT, P = S::PITCH, N16 = KT / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const Kt = (T*)smem;
    T* const Vt = Kt + KT * P;
    float* const lut = (float*)(Vt + KT * P);
    const int nl = 2 * (p.R + S::PAD) + 1;
    float* const diag = lut + nl;                                          // [wave][nl]: sums of dS along the diagonals
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const Where w = place(p, p.H / p.Hk, blockIdx.x);
    if (w.b >= p.B) return;
    const int blk = p.causal ? p.nblk - 1 - w.blk : w.blk;
    const int q0 = blk * S::QB, nk = keys_of(p, w.b), qs = start_of(p, w.b);
    const bool vec = p.vec;
    load_lut(p, w.h, S::PAD, lut, threadIdx.x, NTHR);
    for (int i = threadIdx.x; i < NWAVE * nl; i += NTHR) diag[i] = 0.f;
    const int qw = q0 + wave * 16 * NQ, pmin = qs + qw, pmax = pmin + 16 * NQ - 1;
    const T* qp = (const T*)p.q + w.b * p.qb + (long)w.h * p.ch;
    const T* op = (const T*)p.out + w.b * p.ob + (long)w.h * p.ch;
    const T* dp = (const T*)p.dout + w.b * p.db + (long)w.h * p.ch;
    const long row0 = ((long)w.b * p.H + w.h) * p.Tq;
    frag qf[NQ][KS], df[NQ][KS];
    float ls[NQ], D[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        const bool there = q < p.Tq;
        float d = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[i][s] = row_frag_global<T>(qp + q * p.qr, 32 * s + 8 * g, p.ch, vec, there);
            df[i][s] = row_frag_global<T>(dp + q * p.dr, 32 * s + 8 * g, p.ch, vec, there);
            const frag of = row_frag_global<T>(op + q * p.orow, 32 * s + 8 * g, p.ch, vec, there);
#pragma unroll
            for (int j = 0; j < 8; ++j) d += (float)df[i][s][j] * (float)of[j];
        }
        D[i] = col_sum(d);
        ls[i] = there ? p.lse[row0 + q] * LOG2E : INFINITY;
        if (ls[i] == -INFINITY) ls[i] = INFINITY;                          // a row without keys: P = 0
        if (there && g == 0) p.dsum[row0 + q] = D[i];
    }
    f32x4 a[NQ][CT];
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c) a[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float far_lo = 0.f, far_hi = 0.f;
    const int kend = p.causal ? max(0, min(nk, qs + min(q0 + S::QB, p.Tq))) : nk;
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    const float sl = p.scale * LOG2E;
    for (int k0 = 0; k0 < kend; k0 += KT) {
        __syncthreads();
        stage<T, CHP, KT>(Kt, kp + k0 * p.kr, p.kr, nk - k0, p.ch, vec);
        stage<T, CHP, KT>(Vt, vp + k0 * p.vr, p.vr, nk - k0, p.ch, vec);
        __syncthreads();
        const int far = k0 + KT - 1 - pmin <= -p.R ? -1 : (k0 - pmax >= p.R ? 1 : 0);
        const bool masked = k0 + KT > nk || (p.causal && k0 + KT - 1 > pmin);
        const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int pos = pmin + 16 * i + (lane & 15);
            f32x4 s[N16], d[N16];
#pragma unroll
            for (int n = 0; n < N16; ++n) {
                s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
                d[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s[n] = mma(row_frag<T>(Kt, P, 16 * n, 32 * ks, lane), qf[i][ks], s[n]);
                    d[n] = mma(row_frag<T>(Vt, P, 16 * n, 32 * ks, lane), df[i][ks], d[n]);
                }
            }
            bias_mask<N16>(s, sl, lut, p.R + S::PAD, far, flo, fhi, masked, k0, nk, pos, p.causal, lane);
            float tot = 0.f;
#pragma unroll
            for (int n = 0; n < N16; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = s[n][r] == -INFINITY ? 0.f : exp2_raw(s[n][r] - ls[i]);
                    s[n][r] = e == 0.f ? 0.f : e * (d[n][r] - D[i]);       // (masked places may hold anything)
                    tot += s[n][r];
                }
            if (far < 0) far_lo += tot;
            else if (far > 0) far_hi += tot;
            else {
                // diagonal key - pos: the 16 lanes of a group hit 16 different places, the groups go one after the other
                float* dg = diag + wave * nl + (k0 + 4 * g - pos + p.R + S::PAD);
#pragma unroll
                for (int gg = 0; gg < 4; ++gg)
                    if (g == gg) {
#pragma unroll
                        for (int n = 0; n < N16; ++n)
#pragma unroll
                            for (int r = 0; r < 4; ++r) atomicAdd(dg + 16 * n + r, s[n][r]);
                    }
            }
#pragma unroll
            for (int kb = 0; kb < N16 / 2; ++kb) {
                const frag pf = acc_frag<T>(s[2 * kb] * p.scale, s[2 * kb + 1] * p.scale);
#pragma unroll
                for (int c = 0; c < CT; ++c) a[i][c] = mma(col_frag<T>(Kt, P, 32 * kb, 16 * c, lane), pf, a[i][c]);
            }
        }
    }
    T* gp = (T*)p.dq + w.b * p.dqb + (long)w.h * p.ch;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        if (q >= p.Tq) continue;
#pragma unroll
        for (int c = 0; c < CT; ++c) store4<T>(gp + q * p.dqr, 16 * c + 4 * g, p.ch, vec, a[i][c]);
    }
    // this workgroup's sums along the 2R + 1 clipped diagonals
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {
        diag[wave * nl] += far_lo;
        diag[wave * nl + nl - 1] += far_hi;
    }
    __syncthreads();
    float* out = p.part + (((long)w.b * p.nblk + blk) * p.H + w.h) * (2 * p.R + 1);
    for (int i = threadIdx.x; i <= 2 * p.R; i += NTHR) {
        const int lo = i == 0 ? 0 : i + S::PAD, hi = i == 2 * p.R ? nl - 1 : i + S::PAD;
        float t = 0.f;
        for (int j = lo; j <= hi; ++j)
#pragma unroll
            for (int x = 0; x < NWAVE; ++x) t += diag[x * nl + j];
        out[i] = t;
    }
}

// dtable[n][h]: the workgroups' diagonal sums of head h in their order, then the diagonals of each bucket.
template <typename TT>
__global__ __launch_bounds__(1024) void k_rel_attention_dtable(AttP p, int nparts) {
    __shared__ float sum[2 * RMAX + 1];
    const int h = blockIdx.x, nd = 2 * p.R + 1;
    for (int i = threadIdx.x; i < nd; i += 1024) {
        float t = 0.f;
        for (int j = 0; j < nparts; ++j) t += p.part[((long)j * p.H + h) * nd + i];
        sum[i] = t;
    }
    __syncthreads();
    for (int n = threadIdx.x; n < p.nb; n += 1024) {
        float t = 0.f;
        for (int i = 0; i < nd; ++i) t += p.map[i] == n ? sum[i] : 0.f;
        ((TT*)p.dtable)[(long)n * p.H + h] = (TT)t;
    }
}

// -------------------------------------------------------------------------------------------------------------------- dk, dv
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, 2) void k_rel_attention_dkv(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int QT = S::KT, NK = S::NQ, KS = S::KS, CT = S::CT, P = S::PITCH, N16 = QT / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const Qt = (T*)smem;
    T* const Dt = Qt + QT * P;
    float* const row_ls = (float*)(Dt + QT * P);
    float* const row_d = row_ls + QT;
    float* const lut = row_d + QT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const Where w = place(p, 1, blockIdx.x);
    if (w.b >= p.B) return;
    const int k0 = w.blk * S::QB, nk = keys_of(p, w.b), qs = start_of(p, w.b);
    const bool vec = p.vec;
    const int kw = k0 + wave * 16 * NK;
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    frag kf[NK][KS], vf[NK][KS];
    f32x4 ak[NK][CT], av[NK][CT];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int kk = kw + 16 * i + (lane & 15);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[i][s] = row_frag_global<T>(kp + kk * p.kr, 32 * s + 8 * g, p.ch, vec, kk < nk);
            vf[i][s] = row_frag_global<T>(vp + kk * p.vr, 32 * s + 8 * g, p.ch, vec, kk < nk);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) { ak[i][c] = f32x4{0.f, 0.f, 0.f, 0.f}; av[i][c] = f32x4{0.f, 0.f, 0.f, 0.f}; }
    }
    const float sl = p.scale * LOG2E;
    const int rep = p.H / p.Hk;
    // queries that see this block's first key: position >= k0
    const int qbeg = p.causal ? max(0, k0 - qs) / QT * QT : 0;
    if (k0 < nk)
        for (int hh = 0; hh < rep; ++hh) {
            const int h = w.hk * rep + hh;
            const T* qp = (const T*)p.q + w.b * p.qb + (long)h * p.ch;
            const T* dp = (const T*)p.dout + w.b * p.db + (long)h * p.ch;
            const long row0 = ((long)w.b * p.H + h) * p.Tq;
            __syncthreads();
            load_lut(p, h, S::PAD, lut, threadIdx.x, NTHR);
            for (int q0 = qbeg; q0 < p.Tq; q0 += QT) {
                __syncthreads();
                stage<T, CHP, QT>(Qt, qp + q0 * p.qr, p.qr, p.Tq - q0, p.ch, vec);
                stage<T, CHP, QT>(Dt, dp + q0 * p.dr, p.dr, p.Tq - q0, p.ch, vec);
                for (int i = threadIdx.x; i < QT; i += NTHR) {
                    float x = q0 + i < p.Tq ? p.lse[row0 + q0 + i] * LOG2E : INFINITY;
                    row_ls[i] = x == -INFINITY ? INFINITY : x;
                    row_d[i] = q0 + i < p.Tq ? p.dsum[row0 + q0 + i] : 0.f;
                }
                __syncthreads();
                const int pmin = qs + q0, pmax = pmin + QT - 1;
                const int far = kw + 16 * NK - 1 - pmin <= -p.R ? -1 : (kw - pmax >= p.R ? 1 : 0);
                const bool masked = kw + 16 * NK > nk || (p.causal && kw + 16 * NK - 1 > pmin);
                const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)];
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    const int key = kw + 16 * i + (lane & 15);
                    f32x4 s[N16], d[N16];
#pragma unroll
                    for (int n = 0; n < N16; ++n) {
                        s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
                        d[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            s[n] = mma(row_frag<T>(Qt, P, 16 * n, 32 * ks, lane), kf[i][ks], s[n]);
                            d[n] = mma(row_frag<T>(Dt, P, 16 * n, 32 * ks, lane), vf[i][ks], d[n]);
                        }
                    }
                    const float* lp = lut + (far ? 0 : key - pmin - 4 * g + p.R + S::PAD);
#pragma unroll
                    for (int n = 0; n < N16; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int qi = 16 * n + 4 * g + r;
                            const float b = far ? (far < 0 ? flo : fhi) : lp[-16 * n - r];
                            float e = exp2_raw(s[n][r] * sl + b - row_ls[qi]);
                            if (masked && (key >= nk || (p.causal && key > pmin + qi))) e = 0.f;
                            s[n][r] = e;
                            d[n][r] = e == 0.f ? 0.f : e * (d[n][r] - row_d[qi]) * p.scale;
                        }
#pragma unroll
                    for (int qb = 0; qb < N16 / 2; ++qb) {
                        const frag pf = acc_frag<T>(s[2 * qb], s[2 * qb + 1]), sf = acc_frag<T>(d[2 * qb], d[2 * qb + 1]);
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            av[i][c] = mma(col_frag<T>(Dt, P, 32 * qb, 16 * c, lane), pf, av[i][c]);
                            ak[i][c] = mma(col_frag<T>(Qt, P, 32 * qb, 16 * c, lane), sf, ak[i][c]);
                        }
                    }
                }
            }
        }
    T* gk = (T*)p.dk + w.b * p.dkb + (long)w.hk * p.ch;
    T* gv = (T*)p.dv + w.b * p.dvb + (long)w.hk * p.ch;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int kk = kw + 16 * i + (lane & 15);
        if (kk >= p.Tk) continue;                                          // keys behind klen: zeros
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            store4<T>(gk + kk * p.dkr, 16 * c + 4 * g, p.ch, vec, ak[i][c]);
            store4<T>(gv + kk * p.dvr, 16 * c + 4 * g, p.ch, vec, av[i][c]);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------- host
int check_common(const dua_rel_attention_args* a, const char* who) {
    DUA_REQUIRE(a, "%s: null arguments", who);
    DUA_REQUIRE(dua_dtype_ok(a->dtype) && dua_dtype_ok(a->table_dtype) && (a->table_dtype == DUA_DTYPE_F32 || a->table_dtype == a->dtype),
                "%s: dtype must be fp32, bf16 or fp16 and the table's fp32 or the same", who);
    DUA_REQUIRE(a->B >= 0 && a->Tq >= 0 && a->Tk >= 0 && a->Tq < (1 << 29) && a->Tk < (1 << 29), "%s: lengths must be in [0, 2^29)", who);
    DUA_REQUIRE(a->heads >= 1 && a->kv_heads >= 1 && a->heads % a->kv_heads == 0, "%s: kv_heads must divide heads", who);
    DUA_REQUIRE(a->ch >= 1 && a->ch <= 128, "%s: head width must be in [1, 128]", who);
    DUA_REQUIRE(a->radius >= 1 && a->radius <= RMAX && a->num_buckets >= 1, "%s: radius must be in [1, %d]", who, RMAX);
    DUA_REQUIRE(a->table && a->bucket_map, "%s: null table / bucket map", who);
    DUA_REQUIRE((a->B == 0 || a->Tq == 0 || a->q) && (a->B == 0 || a->Tk == 0 || (a->k && a->v)), "%s: null operand", who);
    DUA_REQUIRE((long)a->B * a->heads * ((a->Tq > a->Tk ? a->Tq : a->Tk) / 64 + 1) < (1L << 23), "%s: too many blocks for one launch", who);
    return DUA_OK;
}

// 16-byte accesses everywhere: widths, strides and addresses in whole 16 bytes
struct Align {
    size_t bits = 0;
    void ptr(const void* q) { bits |= (uintptr_t)q; }
    void str(long s, size_t es) { bits |= (size_t)s * es; }
    bool ok() const { return (bits & 15) == 0; }
};

AttP pack(const dua_rel_attention_args* a, bool bwd) {
    AttP p{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.table = a->table; p.o = a->out; p.out = a->out; p.dout = a->dout;
    p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.dtable = a->dtable;
    p.qb = a->q_batch; p.qr = a->q_row; p.kb = a->k_batch; p.kr = a->k_row; p.vb = a->v_batch; p.vr = a->v_row; p.ob = a->out_batch; p.orow = a->out_row;
    p.db = a->dout_batch; p.dr = a->dout_row; p.dqb = a->dq_batch; p.dqr = a->dq_row; p.dkb = a->dk_batch; p.dkr = a->dk_row; p.dvb = a->dv_batch; p.dvr = a->dv_row;
    p.map = a->bucket_map; p.klen = a->klen; p.qstart = a->qstart; p.lse = a->lse;
    p.B = a->B; p.Tq = a->Tq; p.Tk = a->Tk; p.H = a->heads; p.Hk = a->kv_heads; p.ch = a->ch; p.R = a->radius; p.nb = a->num_buckets;
    p.causal = a->causal != 0; p.table_dtype = a->table_dtype; p.scale = a->scale;
    const size_t es = dua_dtype_size(a->dtype);
    Align al;
    al.bits |= (size_t)a->ch * es;
    al.ptr(a->q); al.ptr(a->k); al.ptr(a->v); al.ptr(a->out);
    for (long s : {p.qb, p.qr, p.kb, p.kr, p.vb, p.vr, p.ob, p.orow}) al.str(s, es);
    if (bwd) {
        al.ptr(a->dout); al.ptr(a->dq); al.ptr(a->dk); al.ptr(a->dv);
        for (long s : {p.db, p.dr, p.dqb, p.dqr, p.dkb, p.dkr, p.dvb, p.dvr}) al.str(s, es);
    }
    p.vec = al.ok();
    return p;
}

unsigned grid_of(AttP& p, int heads_inner, int nblk) {
    p.nblk = nblk;
    const long units = (long)p.B * p.Hk, inner = (long)heads_inner * nblk;
    // eight XCDs: only where a last, partly filled round of kv heads does not leave them unevenly loaded
    p.swz = units % 8 == 0 || units >= 64;
    return (unsigned)((p.swz ? (units + 7) / 8 * 8 : units) * inner);
}

int chp_of(int ch) { return ch <= 32 ? 32 : ch <= 64 ? 64 : ch <= 96 ? 96 : 128; }

// Launch with `lds` bytes of dynamic LDS (more than 64 KB, wide radii with wide fp32 heads, have to be asked for)
template <typename... A>
int launch(void (*kernel)(A...), const char* what, unsigned grid, unsigned block, size_t lds, hipStream_t st, A... args) {
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            dua_set_error("%s: %s", what, hipGetErrorString(e));
            return DUA_EHIP;
        }
    }
    hipLaunchKernelGGL(kernel, grid, block, lds, st, args...);
    return dua_check_launch(what);
}

template <typename T, int CHP> struct Fwd {
    static int run(AttP p, hipStream_t st) {
        typedef Shape<T, CHP> S;
        const unsigned grid = grid_of(p, p.H / p.Hk, (p.Tq + S::QB - 1) / S::QB);
        const size_t lds = 2 * S::KT * S::PITCH * sizeof(T) + (2 * (p.R + S::PAD) + 1) * sizeof(float);
        return launch(k_rel_attention<T, CHP>, "dua_rel_attention", grid, NTHR, lds, st, p);
    }
};
template <typename T, int CHP> struct Bwd {
    static int run(AttP p, hipStream_t st) {
        typedef Shape<T, CHP> S;
        const int nqb = (p.Tq + S::QB - 1) / S::QB, nl = 2 * (p.R + S::PAD) + 1;
        const size_t tiles = 2 * S::KT * S::PITCH * sizeof(T);
        if (p.B > 0 && nqb > 0) {
            const unsigned grid = grid_of(p, p.H / p.Hk, nqb);
            if (int rc = launch(k_rel_attention_dq<T, CHP>, "dua_rel_attention_bwd", grid, NTHR, tiles + (1 + NWAVE) * nl * sizeof(float), st, p)) return rc;
        }
        if (p.B > 0 && p.Tk > 0) {
            const unsigned grid = grid_of(p, 1, (p.Tk + S::QB - 1) / S::QB);
            if (int rc = launch(k_rel_attention_dkv<T, CHP>, "dua_rel_attention_bwd", grid, NTHR, tiles + (2 * S::KT + nl) * sizeof(float), st, p)) return rc;
        }
        const int nparts = p.B * nqb;
        if (p.table_dtype == DUA_DTYPE_F32) return launch(k_rel_attention_dtable<float>, "dua_rel_attention_bwd", p.H, 1024, 0, st, p, nparts);
        if (p.table_dtype == DUA_DTYPE_BF16) return launch(k_rel_attention_dtable<bf16_t>, "dua_rel_attention_bwd", p.H, 1024, 0, st, p, nparts);
        return launch(k_rel_attention_dtable<f16_t>, "dua_rel_attention_bwd", p.H, 1024, 0, st, p, nparts);
    }
};

template <template <typename, int> class L>
int dispatch(int dtype, const AttP& p, hipStream_t st) {
#define GO(T)                                             \
    switch (chp_of(p.ch)) {                               \
        case 32: return L<T, 32>::run(p, st);             \
        case 64: return L<T, 64>::run(p, st);             \
        case 96: return L<T, 96>::run(p, st);             \
        default: return L<T, 128>::run(p, st);            \
    }
    if (dtype == DUA_DTYPE_F32) { GO(float) } else if (dtype == DUA_DTYPE_BF16) { GO(bf16_t) } else { GO(f16_t) }
#undef GO
}

// queries of a workgroup, smallest over the types and widths: bounds the number of partial tables
int query_blocks(const dua_rel_attention_args* a) {
    const int qb = a->dtype == DUA_DTYPE_F32 || chp_of(a->ch) > 64 ? 16 * NWAVE : 32 * NWAVE;
    return (a->Tq + qb - 1) / qb;
}

}  // namespace

extern "C" size_t dua_rel_attention_workspace_bytes(const dua_rel_attention_args* a, int backward) {
    if (!a || check_common(a, "dua_rel_attention_workspace_bytes")) return 0;
    if (!backward) return 0;
    return ((size_t)a->B * a->heads * a->Tq + (size_t)a->B * query_blocks(a) * a->heads * (2 * a->radius + 1)) * sizeof(float);
}

extern "C" int dua_rel_attention(const dua_rel_attention_args* a, void* stream) {
    if (int rc = check_common(a, "dua_rel_attention")) return rc;
    if (a->B == 0 || a->Tq == 0) return DUA_OK;
    DUA_REQUIRE(a->out, "dua_rel_attention: null output");
    return dispatch<Fwd>(a->dtype, pack(a, false), as_stream(stream));
}

extern "C" int dua_rel_attention_bwd(const dua_rel_attention_args* a, void* stream) {
    if (int rc = check_common(a, "dua_rel_attention_bwd")) return rc;
    DUA_REQUIRE(a->dtable, "dua_rel_attention_bwd: null dtable");
    DUA_REQUIRE(a->B == 0 || a->Tq == 0 || (a->out && a->lse && a->dout && a->dq), "dua_rel_attention_bwd: null operand");
    DUA_REQUIRE(a->B == 0 || a->Tk == 0 || (a->dk && a->dv), "dua_rel_attention_bwd: null output");
    const size_t need = dua_rel_attention_workspace_bytes(a, 1);
    DUA_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), "dua_rel_attention_bwd: workspace smaller than dua_rel_attention_workspace_bytes");
    AttP p = pack(a, true);
    p.dsum = (float*)a->workspace;
    p.part = p.dsum + (size_t)a->B * a->heads * a->Tq;
    return dispatch<Bwd>(a->dtype, p, as_stream(stream));
}
