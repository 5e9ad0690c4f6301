// Gradients of attention with a bucketed relative bias (rel_attention.h): dq with the table's diagonal sums, dk and dv, the table.
#include "rel_attention.h"

namespace {

// ------------------------------------------------------------------------------------------------------------------ diagonals
// Sums along the diagonals of a 16 x 16 block x (row 4 g + r, column c of lane 16 g + c): lane (g, c) of `a` collects diagonal row - column =
// 4 g - c, of `b` (c >= 13) diagonal 4 g + 16 - c.  A lane's four rows are shifted along its 16 columns, zeros coming in.
__device__ __forceinline__ void diagonals(f32x4 x, float& a, float& b) {
    a = x[0] + dpp_move<0x101>(x[1]) + dpp_move<0x102>(x[2]) + dpp_move<0x103>(x[3]);      // row_shl: from the column 1, 2, 3 to the right
    b = dpp_move<0x11F>(x[1]) + dpp_move<0x11E>(x[2]) + dpp_move<0x11D>(x[3]);              // row_shr by 15, 14, 13: what left the row there
}

// The four waves' sums along the diagonals (diag [wave][nl], distance 0 at R + pad) clipped to 2R + 1 distances, into this workgroup's row of the
// partial sums, times `unit`; then zeros again.
__device__ __forceinline__ void flush_diagonals(float* diag, int nl, int R, int pad, float far_lo, float far_hi, float unit, float* out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    far_lo = wave_sum(far_lo);
    far_hi = wave_sum(far_hi);
    if (lane == 0) {
        diag[wave * nl] += far_lo;
        diag[wave * nl + nl - 1] += far_hi;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nl; i += NTHR) diag[i] = (diag[i] + diag[nl + i]) + (diag[2 * nl + i] + diag[3 * nl + i]);
    __syncthreads();
    for (int i = 1 + threadIdx.x; i < 2 * R; i += NTHR) out[i] = diag[i + pad] * unit;
    if (wave < 2) {                                            // the two ends: all that lies beyond
        float t = 0.f;
        for (int i = lane; i <= pad; i += 64) t += diag[(wave ? nl - 1 - pad : 0) + i];
        t = wave_sum(t);
        if (lane == 0) out[wave ? 2 * R : 0] = t * unit;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NWAVE * nl; i += NTHR) diag[i] = 0.f;
}
static_assert(NWAVE == 4, "flush_diagonals adds four waves");

// ------------------------------------------------------------------------------------------------------------------------ dq
// dq: 6 ch matrix operations a pair; a wave holds 32 queries' q, dO and dq, the keys and values pass through LDS, and every fragment read from there
// feeds two products.  Bound by three units that take turns more than they overlap: at 64 bf16 the vector unit is busy 55 % of the CUs' time, LDS 32, the
// matrix unit 25, and a wave waits 40 % of its time for data.  Three waves a SIMD at head widths up to 64 (20 bytes of spill, fp16 40): 4 x 16 heads of 64,
// 4096 tokens bf16 1282 us a backward pass, 1356 with two.  8 x 16 heads, 1024 tokens of 64 bf16 in a padded batch: 77 us.  fp32: matrix unit 58 %.
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, CHP > 64 ? 2 : 3) void k_rel_attention_dq(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int KT = S::KT, NQ = S::NQ, KS = S::KS, CT = S::CT, P = S::PITCH, NP = S::NP;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const tiles = (T*)smem;                                             // [2][K, V]
    float* const lut = (float*)(smem + 4 * S::TILE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const Where w = place(p, p.H / p.Hk, blockIdx.x);
    if (w.b >= p.B) return;
    const int blk = p.causal ? p.nblk - 1 - w.blk : w.blk;
    const int q0 = blk * S::QB, nk = keys_of(p, w.b), qs = start_of(p, w.b);
    const int kend = p.causal ? max(0, min(nk, qs + min(q0 + S::QB, p.Tq))) : nk;
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    Carrier<T, CHP, KT> ck(p.kr, p.ch, tid), cv(p.vr, p.ch, tid);
    if (kend > 0) {
        ck.fetch(kp, p.kr, kend, p.ch, tid);
        cv.fetch(vp, p.vr, kend, p.ch, tid);
    }
    load_lut(p, w.h, S::PAD, lut);
    const int qw = q0 + wave * 16 * NQ, pmin = qs + qw, pmax = pmin + 16 * NQ - 1;
    const T* qp = (const T*)p.q + w.b * p.qb + (long)w.h * p.ch;
    const T* op = (const T*)p.out + w.b * p.ob + (long)w.h * p.ch;
    const T* dp = (const T*)p.dout + w.b * p.db + (long)w.h * p.ch;
    const long row0 = ((long)w.b * p.H + w.h) * p.Tq;
    frag qf[NQ][KS], df[NQ][KS];
    float ls[NQ], D[NQ], rest[NQ], f[NQ];
    f32x4 a[NQ][CT];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        const bool there = q < p.Tq;
        const int qr = min(q, p.Tq - 1);
        float d = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = S::KSTEP * s + Frag<T>::N * g;
            qf[i][s] = row_frag_global<T>(qp + qr * p.qr, c, p.ch, there);
            df[i][s] = row_frag_global<T>(dp + qr * p.dr, c, p.ch, there);
            const frag of = row_frag_global<T>(op + qr * p.orow, c, p.ch, there);
            frag lo = zero16<T>();                                          // the output's rounding: D's error would be the gradients' largest
            if (sizeof(T) == 2 && p.olo_in) lo = row_frag_global<T>((const T*)p.olo_in + (row0 + qr) * p.ch, c, p.ch, there);
#pragma unroll
            for (int j = 0; j < Frag<T>::N; ++j) d += (float)df[i][s][j] * ((float)of[j] + (float)lo[j]);
        }
        D[i] = col_sum(d);
        ls[i] = there ? p.lse[row0 + q] * LOG2E : INFINITY;
        if (ls[i] == -INFINITY) ls[i] = INFINITY;                          // a row without keys: P = 0
        rest[i] = 0.f;
        f[i] = F_START;
#pragma unroll
        for (int c = 0; c < CT; ++c) a[i][c] = ZERO4;
    }
    const float sl = p.scale * LOG2E;
    __syncthreads();
    const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)], *lut0 = lut + p.R + S::PAD;
    for (int k0 = 0, t = 0; k0 < kend; k0 += KT, ++t) {
        T* const Kt = tiles + (t & 1) * 2 * KT * P;
        T* const Vt = Kt + KT * P;
        ck.put(Kt, p.ch, tid);
        cv.put(Vt, p.ch, tid);
        __syncthreads();
        if (k0 + KT < kend) {
            ck.fetch(kp + (long)(k0 + KT) * p.kr, p.kr, kend - k0 - KT, p.ch, tid);
            cv.fetch(vp + (long)(k0 + KT) * p.vr, p.vr, kend - k0 - KT, p.ch, tid);
        }
        if (qw >= p.Tq) continue;
        // steps of 16 NP keys: scores, dP, dS, and dS straight into dq - few registers live
        for (int n0 = 0; n0 < KT / 16; n0 += NP) {
            const int ks0 = k0 + 16 * n0;
            if (ks0 >= kend || (p.causal && ks0 > pmax)) break;
            f32x4 s[NQ][NP], d[NQ][NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) {
#pragma unroll
                for (int i = 0; i < NQ; ++i) { s[i][n] = ZERO4; d[i][n] = ZERO4; }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const frag x = row_frag<T>(Kt, P, 16 * (n0 + n), S::KSTEP * ks, lane), y = row_frag<T>(Vt, P, 16 * (n0 + n), S::KSTEP * ks, lane);
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        s[i][n] = mma(x, qf[i][ks], s[i][n]);
                        d[i][n] = mma(y, df[i][ks], d[i][n]);
                    }
                }
            }
            const int side = side_of(ks0, 16 * NP, pmin, pmax, p.R);
            const bool masked = ks0 + 16 * NP > nk || (p.causal && ks0 + 16 * NP - 1 > pmin);
            frag pf[NQ];
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                bias_mask<NP>(s[i], sl, lut0, side, side < 0 ? flo : fhi, masked, ks0, nk, pmin + 16 * i + (lane & 15), p.causal, lane);
                f32x4 e[NP];
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = exp2_raw(s[i][n][r] - ls[i]);
                        s[i][n][r] = x;
                        e[n][r] = x * (d[i][n][r] - D[i]);
                    }
                if (masked) {                                               // (masked places may hold anything)
#pragma unroll
                    for (int n = 0; n < NP; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) e[n][r] = s[i][n][r] == 0.f ? 0.f : e[n][r];
                }
#pragma unroll
                for (int n = 0; n < NP; ++n) rest[i] += (e[n][0] + e[n][1]) + (e[n][2] + e[n][3]);
                if constexpr (S::NARROW) in_range<NP, CT>(e, f[i], a[i]);
                pf[i] = acc_frag<T>(e);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const frag x = col_frag<T>(Kt, P, 16 * n0, 16 * c, lane);
#pragma unroll
                for (int i = 0; i < NQ; ++i) a[i][c] = mma(x, pf[i], a[i][c]);
            }
        }
    }
    T* gp = (T*)p.dq + w.b * p.dqb + (long)w.h * p.ch;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        // sum_j dS_ij is 0 for the exact D: what is left is D's error (the output came from P rounded for its product, and was rounded itself).
        // dk and the table take the corrected value - the table's sums cancel to little, it would be their largest error.
        const float dt = D[i] + col_sum(rest[i]);
        if (q >= p.Tq) continue;
        if (g == 0) p.dsum[row0 + q] = dt;
#pragma unroll
        for (int c = 0; c < CT; ++c) store4<T>(gp + q * p.dqr, 16 * c + 4 * g, p.ch, S::NARROW ? a[i][c] * p.scale * pow2_inverse(f[i]) : a[i][c] * p.scale);
    }
}

// The workgroups' diagonal sums of head h added in their order, 64 distances a workgroup and a run of parts for each of its 16 waves ...
__global__ __launch_bounds__(1024) void k_rel_attention_diag(AttP p, int nparts) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, nd = 2 * p.R + 1, i = blockIdx.x * 64 + lane;
    const int per = (nparts + 15) / 16, j0 = wave * per, j1 = min(j0 + per, nparts);
    float t = 0.f;
    if (i < nd) {
#pragma unroll 8
        for (int j = j0; j < j1; ++j) t += p.part[((long)j * p.H + h) * nd + i];
    }
    sm[wave][lane] = t;
    __syncthreads();
    if (wave || i >= nd) return;
    for (int x = 1; x < 16; ++x) t += sm[x][lane];
    p.diag[h * nd + i] = t;
}
// ... and dtable[n][h]: the distances of bucket n, a wave a bucket.
template <typename TT>
__device__ __forceinline__ void sum_buckets(const AttP& p, int h, const float* diag) {
    const int lane = threadIdx.x & 63, nd = 2 * p.R + 1;
    for (int n = threadIdx.x >> 6; n < p.nb; n += 16) {
        float t = 0.f;
        for (int i = lane; i < nd; i += 64) t += p.map[i] == n ? diag[i] : 0.f;
        t = wave_sum(t);
        if (lane == 0) ((TT*)p.dtable)[(long)n * p.H + h] = (TT)t;
    }
}
template <typename TT>
__global__ __launch_bounds__(1024) void k_rel_attention_dtable(AttP p) { sum_buckets<TT>(p, blockIdx.x, p.diag + blockIdx.x * (2 * p.R + 1)); }

// Both at once where there are few parts, a workgroup a head: runs of parts side by side (together at most 1024 sums, or one run of 2R + 1), a thread
// a distance; the runs added in order.  A launch less: 1.5 us on the GPU, 5 us of host time; backward of 32 parts of 257 distances 78.3 us against
// 79.8 with two kernels, of 64 parts 136.3 against 135.5.
constexpr int FEW_PARTS = 32;
template <typename TT>
__global__ __launch_bounds__(1024) void k_rel_attention_dtable_few(AttP p, int nparts) {
    __shared__ float sm[2 * RMAX + 1];
    const int h = blockIdx.x, nd = 2 * p.R + 1, runs = max(1, 1024 / nd), per = (nparts + runs - 1) / runs;
    for (int at = threadIdx.x; at < runs * nd; at += 1024) {
        const int run = at / nd, i = at % nd, j0 = run * per, j1 = min(j0 + per, nparts);
        float t = 0.f;
#pragma unroll 8
        for (int j = j0; j < j1; ++j) t += p.part[((long)j * p.H + h) * nd + i];
        sm[at] = t;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nd; i += 1024)
        for (int run = 1; run < runs; ++run) sm[i] += sm[run * nd + i];
    __syncthreads();
    sum_buckets<TT>(p, h, sm);
}
template <typename TT>
int table_gradient(const AttP& p, int nparts, hipStream_t st) {
    if (nparts <= FEW_PARTS) return launch<k_rel_attention_dtable_few<TT>>("dua_rel_attention_bwd", dim3(p.H), 1024, 0, st, p, nparts);
    if (int rc = launch<k_rel_attention_diag>("dua_rel_attention_bwd", dim3((2 * p.R + 64) / 64, p.H), 1024, 0, st, p, nparts)) return rc;
    return launch<k_rel_attention_dtable<TT>>("dua_rel_attention_bwd", dim3(p.H), 1024, 0, st, p);
}

// -------------------------------------------------------------------------------------------------------------------- dk, dv
// dk, dv and the diagonal sums: 8 ch matrix operations a pair; a wave holds 32 keys' k, v, dk and dv (wide heads and fp32: 16), the queries and dO pass
// through LDS, read as rows for the scores and as columns for the sums.  LDS, busy 51 % of the CUs' time (vector unit 31, matrix unit 17), is the fullest unit
// and a wave waits 40 % of its time: 16 keys a wave on three waves a SIMD read twice as much and take 286 us a backward pass, on four 309, where 32 keys on two
// take 243 (8 x 16 heads, 1024 tokens of 64 bf16; 152 us are this kernel in a padded batch).  The sums along the diagonals cost there 210 -> 246 us at
// radius 128, 369 at radius 512: where a tile is nearer than the radius every dS is shifted to its diagonal.  fp32: matrix unit 47 %, LDS 38; at 65 to
// 80 wide three waves a SIMD spill 17 registers (72 bytes a lane: addresses and the like, written once, read again by every tile).
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, sizeof(T) == 4 && CHP <= 80 ? 3 : 2) void k_rel_attention_dkv(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int QT = S::KT, NK = S::NK, KS = S::KS, CT = S::CT, P = S::PITCH, NP = S::NP;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const tiles = (T*)smem;                                             // [2][Q, dO]
    float* const rows = (float*)(smem + 4 * S::TILE);                       // [2][lse, D][QT]
    float* const lut = rows + 4 * QT;
    const int nl = 2 * (p.R + S::PAD) + 1;
    float* const diag = lut + nl;                                          // [wave][nl]: a head's sums of dS along the diagonals
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const Where w = place(p, 1, blockIdx.x);
    const int split = blockIdx.y, qsplit = split % p.qsplits;
    if (w.b >= p.B) return;
    const int k0 = w.blk * S::KB, qs = start_of(p, w.b);
    const int nk = p.causal ? max(0, min(keys_of(p, w.b), qs + p.Tq)) : keys_of(p, w.b);   // (what lies behind it is not read: no query sees it)
    const int kw = k0 + wave * 16 * NK;
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    frag kf[NK][KS], vf[NK][KS];
    f32x4 ak[NK][CT], av[NK][CT];
    float f[NK];
    constexpr float UNIT = S::NARROW ? 0x1p-14f : 1.f;                       // 2^-P_SHIFT: P, and dS with it, are 2^P_SHIFT times themselves here
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int kk = kw + 16 * i + (lane & 15);
        f[i] = F_START;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int c = S::KSTEP * s + Frag<T>::N * g;
            const int kr = min(kk, max(nk - 1, 0));
            kf[i][s] = row_frag_global<T>(kp + kr * p.kr, c, p.ch, kk < nk);
            vf[i][s] = row_frag_global<T>(vp + kr * p.vr, c, p.ch, kk < nk);
        }
#pragma unroll
        for (int c = 0; c < CT; ++c) { ak[i][c] = ZERO4; av[i][c] = ZERO4; }
    }
    const float sl = p.scale * LOG2E;
    const int rep = p.H / p.Hk / (p.splits / p.qsplits), h0 = w.hk * (p.H / p.Hk) + split / p.qsplits * rep;   // this workgroup's query heads
    // tiles of queries that see this block's first key (position >= k0), head after head of the group; of a single head (qsplits > 1) a share of them
    const int qmin = p.causal ? max(0, k0 - qs) / QT : 0, all_tiles = max(0, (p.Tq + QT - 1) / QT - qmin);
    const int qbeg = qmin + (int)((long)all_tiles * qsplit / p.qsplits), per = qmin + (int)((long)all_tiles * (qsplit + 1) / p.qsplits) - qbeg;
    const int total = k0 < nk ? per * rep : 0;
    Carrier<T, CHP, QT> cq(p.qr, p.ch, tid), cd(p.dr, p.ch, tid);
    float row_next = 0.f;
    auto fetch = [&](int t) {
        const int h = h0 + t / per, q0 = (qbeg + t % per) * QT;
        cq.fetch((const T*)p.q + w.b * p.qb + (long)h * p.ch + (long)q0 * p.qr, p.qr, p.Tq - q0, p.ch, tid);
        cd.fetch((const T*)p.dout + w.b * p.db + (long)h * p.ch + (long)q0 * p.dr, p.dr, p.Tq - q0, p.ch, tid);
        if (tid < 2 * QT) {
            const int q = q0 + tid % QT;
            const float* src = tid < QT ? p.lse : p.dsum;
            row_next = q < p.Tq ? src[((long)w.b * p.H + h) * p.Tq + q] : (tid < QT ? -INFINITY : 0.f);
        }
    };
    for (int i = tid; i < NWAVE * nl; i += NTHR) diag[i] = 0.f;
    float far_lo = 0.f, far_hi = 0.f;
    float* const part = p.part + ((((long)w.b * p.nblk + w.blk) * p.qsplits + qsplit) * p.H + h0) * (2 * p.R + 1);
    if (total > 0) fetch(0);
    for (int t = 0; t < total; ++t) {
        if (t % per == 0) {
            __syncthreads();                                                // (the last head's bias is read until here)
            if (t > 0) flush_diagonals(diag, nl, p.R, S::PAD, far_lo, far_hi, UNIT, part + (t / per - 1) * (2 * p.R + 1));
            far_lo = far_hi = 0.f;
            load_lut(p, h0 + t / per, S::PAD, lut);
        }
        T* const Qt = tiles + (t & 1) * 2 * QT * P;
        T* const Dt = Qt + QT * P;
        float* const row_ls = rows + (t & 1) * 2 * QT, *const row_d = row_ls + QT;
        cq.put(Qt, p.ch, tid);
        cd.put(Dt, p.ch, tid);
        if (tid < QT) row_ls[tid] = row_next == -INFINITY ? INFINITY : row_next * LOG2E - S::P_SHIFT;   // no keys, no query: P = 0
        else if (tid < 2 * QT) row_ls[tid] = row_next;
        __syncthreads();
        if (t + 1 < total) fetch(t + 1);
        const int q0 = (qbeg + t % per) * QT;
        if (kw >= nk) continue;
        const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)], *lut0 = lut + p.R + S::PAD;
        for (int n0 = 0; n0 < QT / 16; n0 += NP) {
            const int qq = q0 + 16 * n0, pmin = qs + qq, pmax = pmin + 16 * NP - 1;
            if (qq >= p.Tq) break;
            if (p.causal && kw > pmax) continue;
            f32x4 s[NK][NP], d[NK][NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) {
#pragma unroll
                for (int i = 0; i < NK; ++i) { s[i][n] = ZERO4; d[i][n] = ZERO4; }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const frag x = row_frag<T>(Qt, P, 16 * (n0 + n), S::KSTEP * ks, lane), y = row_frag<T>(Dt, P, 16 * (n0 + n), S::KSTEP * ks, lane);
#pragma unroll
                    for (int i = 0; i < NK; ++i) {
                        s[i][n] = mma(x, kf[i][ks], s[i][n]);
                        d[i][n] = mma(y, vf[i][ks], d[i][n]);
                    }
                }
            }
            const int side = side_of(kw, 16 * NK, pmin, pmax, p.R);
            const bool masked = kw + 16 * NK > nk || (p.causal && kw + 16 * NK - 1 > pmin);
            const float b = side < 0 ? flo : fhi;
            frag pf[NK], sf[NK];
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                const int key = kw + 16 * i + (lane & 15);
                if (side) {
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const f32x4 L = b - *(const f32x4*)(row_ls + 16 * (n0 + n) + 4 * g);
                        s[i][n] = s[i][n] * sl + L;
                    }
                } else {
                    const float* lp = lut0 + (key - pmin - 4 * g);
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const f32x4 L = *(const f32x4*)(row_ls + 16 * (n0 + n) + 4 * g);
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][n][r] = s[i][n][r] * sl + (lp[-16 * n - r] - L[r]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    const f32x4 Dr = *(const f32x4*)(row_d + 16 * (n0 + n) + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[i][n][r] = exp2_raw(s[i][n][r]);
                        d[i][n][r] = s[i][n][r] * (d[i][n][r] - Dr[r]);
                    }
                }
                if (masked) {                                               // (masked places may hold anything)
#pragma unroll
                    for (int n = 0; n < NP; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const bool out = key >= nk || (p.causal && key > pmin + 16 * n + 4 * g + r);
                            s[i][n][r] = out ? 0.f : s[i][n][r];
                            d[i][n][r] = out || s[i][n][r] == 0.f ? 0.f : d[i][n][r];
                        }
                }
                pf[i] = acc_frag<T>(s[i]);
            }
            if (side) {
                float tot = 0.f;
#pragma unroll
                for (int i = 0; i < NK; ++i)
#pragma unroll
                    for (int n = 0; n < NP; ++n) tot += (d[i][n][0] + d[i][n][1]) + (d[i][n][2] + d[i][n][3]);
                if (side < 0) far_lo += tot;
                else far_hi += tot;
            } else {
                // blocks with the same i - n share their diagonals; block dd's `b` diagonals are block dd - 1's `a` diagonals
                float keep = 0.f;
                float* dg = diag + wave * nl + (kw + (lane & 15) - pmin - 4 * g + p.R + S::PAD);
#pragma unroll
                for (int dd = NK - 1; dd >= -NP; --dd) {
                    float x = keep;
                    if (dd > -NP) {
                        f32x4 z = ZERO4;
#pragma unroll
                        for (int n = 0; n < NP; ++n)
                            if (dd + n >= 0 && dd + n < NK) z += d[dd + n][n];
                        float a, bb;
                        diagonals(z, a, bb);
                        x += a;
                        keep = bb;
                    }
                    // a group's 16 lanes hit 16 places, the groups go one after the other: the order of a wave's sums is fixed
#pragma unroll
                    for (int gg = 0; gg < 4; ++gg)
                        if (g == gg) atomicAdd(dg + 16 * dd, x);
                }
            }
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                if constexpr (S::NARROW) in_range<NP, CT>(d[i], f[i], ak[i]);
                sf[i] = acc_frag<T>(d[i]);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const frag x = col_frag<T>(Dt, P, 16 * n0, 16 * c, lane), y = col_frag<T>(Qt, P, 16 * n0, 16 * c, lane);
#pragma unroll
                for (int i = 0; i < NK; ++i) {
                    av[i][c] = mma(x, pf[i], av[i][c]);
                    ak[i][c] = mma(y, sf[i], ak[i][c]);
                }
            }
        }
    }
    __syncthreads();
    if (total > 0) {
        flush_diagonals(diag, nl, p.R, S::PAD, far_lo, far_hi, UNIT, part + (rep - 1) * (2 * p.R + 1));
    } else {
        for (int i = tid; i < rep * (2 * p.R + 1); i += NTHR) part[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            ak[i][c] *= p.scale;
            if constexpr (S::NARROW) {
                ak[i][c] = ak[i][c] * UNIT * pow2_inverse(f[i]);
                av[i][c] *= UNIT;
            }
        }
    if (p.splits > 1) {
        // [split][dk, dv][B][Tk][Hk ch]
        const long row = (long)p.Hk * p.ch, all = (long)p.B * p.Tk * row;
        float* const fk = p.kv_part + 2 * split * all + (long)w.b * p.Tk * row + w.hk * p.ch;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            const int kk = kw + 16 * i + (lane & 15);
            if (kk >= p.Tk) continue;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                store4<float>(fk + kk * row, 16 * c + 4 * g, p.ch, ak[i][c]);
                store4<float>(fk + all + kk * row, 16 * c + 4 * g, p.ch, av[i][c]);
            }
        }
        return;
    }
    T* gk = (T*)p.dk + w.b * p.dkb + (long)w.hk * p.ch;
    T* gv = (T*)p.dv + w.b * p.dvb + (long)w.hk * p.ch;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
        const int kk = kw + 16 * i + (lane & 15);
        if (kk >= p.Tk) continue;                                          // keys behind klen: zeros
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            store4<T>(gk + kk * p.dkr, 16 * c + 4 * g, p.ch, ak[i][c]);
            store4<T>(gv + kk * p.dvr, 16 * c + 4 * g, p.ch, av[i][c]);
        }
    }
}

// dk and dv of split blocks: the splits' sums in their order, four elements a thread
template <typename T>
__global__ __launch_bounds__(NTHR) void k_rel_attention_kv_join(AttP p) {
    const int row = p.Hk * p.ch, quads = row / 4;
    const long all = (long)p.B * p.Tk * row, n = 2 * all / 4, stride = (long)gridDim.x * NTHR;
    for (long i = (long)blockIdx.x * NTHR + threadIdx.x; i < n; i += stride) {
        f32x4 a = ZERO4;
        for (int s = 0; s < p.splits; ++s) a += *(const f32x4*)(p.kv_part + 2 * s * all + 4 * i);
        const bool v = 4 * i >= all;
        const long at = v ? i - all / 4 : i, r = at / quads, b = r / p.Tk;
        T* dst = v ? (T*)p.dv + b * p.dvb + (r % p.Tk) * p.dvr : (T*)p.dk + b * p.dkb + (r % p.Tk) * p.dkr;
        store4<T>(dst, 4 * (int)(at % quads), row, a);
    }
}

template <typename T, int CHP> struct Bwd {
    static int run(AttP p, bool, hipStream_t st) {
        typedef Shape<T, CHP> S;
        const int nqb = (p.Tq + S::QB - 1) / S::QB, nl = 2 * (p.R + S::PAD) + 1;
        if (p.B > 0 && nqb > 0) {
            const unsigned grid = grid_of(p, p.H / p.Hk, nqb);
            if (int rc = launch<k_rel_attention_dq<T, CHP>>("dua_rel_attention_bwd", dim3(grid), NTHR, 4 * S::TILE + nl * sizeof(float), st, p)) return rc;
        }
        if (p.B > 0 && p.Tk > 0) {
            const unsigned grid = grid_of(p, 1, (p.Tk + S::KB - 1) / S::KB);
            if (int rc = launch<k_rel_attention_dkv<T, CHP>>("dua_rel_attention_bwd", dim3(grid, p.splits), NTHR, 4 * S::TILE + (4 * S::KT + (1 + NWAVE) * nl) * sizeof(float), st, p)) return rc;
            if (p.splits > 1) {
                const long quads = (long)p.B * p.Tk * p.Hk * p.ch / 2;
                if (int rc = launch<k_rel_attention_kv_join<T>>("dua_rel_attention_bwd", dim3(stream_grid(quads, NTHR)), NTHR, 0, st, p)) return rc;
            }
        }
        const int nparts = p.B * ((p.Tk + S::KB - 1) / S::KB) * p.qsplits;
        if (p.table_dtype == DUA_DTYPE_F32) return table_gradient<float>(p, nparts, st);
        if (p.table_dtype == DUA_DTYPE_BF16) return table_gradient<bf16_t>(p, nparts, st);
        return table_gradient<f16_t>(p, nparts, st);
    }
};

}  // namespace

extern "C" int dua_rel_attention_bwd(const dua_rel_attention_args* a, void* stream) {
    if (int rc = check_common(a, "dua_rel_attention_bwd", true)) return rc;
    DUA_REQUIRE(a->dtable, "dua_rel_attention_bwd: null dtable");
    DUA_REQUIRE(a->B == 0 || a->Tq == 0 || (a->out && a->lse && a->dout && a->dq), "dua_rel_attention_bwd: null operand");
    DUA_REQUIRE(a->B == 0 || a->Tk == 0 || (a->dk && a->dv), "dua_rel_attention_bwd: null output");
    const size_t need = rel_attention_bwd_bytes(a);
    DUA_REQUIRE(need == 0 || (a->workspace && ((uintptr_t)a->workspace & 15) == 0 && a->workspace_bytes >= need),
                "dua_rel_attention_bwd: workspace smaller than dua_rel_attention_workspace_bytes, or not 16-byte aligned");
    AttP p = pack(a);
    p.dsum = (float*)a->workspace;
    const KeySplits ks = key_splits(a);
    p.splits = ks.heads * ks.tiles;
    p.qsplits = ks.tiles;
    p.kv_part = p.dsum + rel_attention_bwd_floats(a);
    p.diag = p.dsum + (size_t)a->B * a->heads * a->Tq;
    p.part = p.diag + (size_t)a->heads * (2 * a->radius + 1);
    return dispatch<Bwd>(a->dtype, p, false, as_stream(stream));
}
