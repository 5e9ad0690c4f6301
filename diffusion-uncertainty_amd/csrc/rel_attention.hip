// Forward kernels of attention with a bucketed relative bias (rel_attention.h): tiles of queries, few queries (decoding), and the join of split keys.
#include "rel_attention.h"

namespace {

// -------------------------------------------------------------------------------------------------------------------- forward
// A row of the result: written, or (keys split over workgroups) left as unnormalised sums with its maximum and sum for the join.
// o: columns' channels 16 c + 4 (l / 16) + r of one query; m in log2 units, l its whole sum.
template <typename T, int CT>
__device__ __forceinline__ void finish_query(const AttP& p, int b, int h, int q, int split, const f32x4* o, float m, float l, int g) {
    const long row = ((long)b * p.H + h) * p.Tq + q;
    if (p.splits > 1) {
        const long at = (long)split * p.B * p.H * p.Tq + row;
        float* po = p.part + at * p.ch;
#pragma unroll
        for (int c = 0; c < CT; ++c)
            if (16 * c + 4 * g < p.ch) *(f32x4*)(po + 16 * c + 4 * g) = o[c];
        if (g == 0) *(float2*)(p.part_ml + 2 * at) = make_float2(m, l);
        return;
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const long at = b * p.ob + q * p.orow + (long)h * p.ch;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const f32x4 v = o[c] * inv;
        store4<T>((T*)p.o + at, 16 * c + 4 * g, p.ch, v);
        if (sizeof(T) == 2 && p.olo) store4<T>((T*)p.olo + row * p.ch, 16 * c + 4 * g, p.ch, rest4<T>(v));
    }
    if (p.lse && g == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
}

// Online softmax with a lazy maximum: the sums are moved to a new maximum only when a score exceeds the old one by more than 2^8 - fp32 sums and
// the rounded P (relative) lose nothing, and after a row's first tile it hardly ever happens.
// Sixteen bit: no unit is full - two waves a SIMD take turns on products, softmax and the products that wait for it.  Busy of the CUs' time: vector unit 44 %
// (128 wide) to 57 % (64), LDS 45 % (18 of them bank conflicts) and 32 %, matrix unit 35 % and 22 %; a wave waits a third of its time for data, a quarter to
// issue.  fp32: matrix unit 54 %, half of a wave's time waiting for it; 72 channels run as 80, 258 queries as 320, 1280 workgroups in two rounds of
// 768 places.  4 x 16 heads of 64, 4096 tokens bf16: 370 us, 740 TFLOP/s (a large matrix product: 1120); 4 x 16 heads of 128 on 4, 4001 tokens
// causal: 362 us, 725 (402 in an unbroken run of such calls); 16 x 16 heads of 72, 258 tokens fp32: 80 us, 61 (154).
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, 2) void k_rel_attention(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int KT = S::KT, NQ = S::NQ, KS = S::KS, CT = S::CT, P = S::PITCH, N16 = KT / 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    T* const tiles = (T*)smem;                                             // [2][K, V]
    float* const lut = (float*)(smem + 4 * S::TILE);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int split = blockIdx.y;
    const Where w = place(p, p.H / p.Hk, blockIdx.x);
    if (w.b >= p.B) return;
    const int blk = p.causal ? p.nblk - 1 - w.blk : w.blk;                 // long rows first
    const int q0 = blk * S::QB, nk = keys_of(p, w.b), qs = start_of(p, w.b);
    const int kend = p.causal ? max(0, min(nk, qs + min(q0 + S::QB, p.Tq))) : nk;   // (what lies behind it is not read)
    const int nt = (kend + KT - 1) / KT, t0 = (int)((long)nt * split / p.splits), t1 = (int)((long)nt * (split + 1) / p.splits);
    const T* kp = (const T*)p.k + w.b * p.kb + (long)w.hk * p.ch;
    const T* vp = (const T*)p.v + w.b * p.vb + (long)w.hk * p.ch;
    Carrier<T, CHP, KT> ck(p.kr, p.ch, tid), cv(p.vr, p.ch, tid);
    if (t0 < t1) {
        ck.fetch(kp + (long)t0 * KT * p.kr, p.kr, kend - t0 * KT, p.ch, tid);
        cv.fetch(vp + (long)t0 * KT * p.vr, p.vr, kend - t0 * KT, p.ch, tid);
    }
    const int qw = q0 + wave * 16 * NQ, pmin = qs + qw, pmax = pmin + 16 * NQ - 1;
    const T* qp = (const T*)p.q + w.b * p.qb + (long)w.h * p.ch;
    frag qf[NQ][KS];
    f32x4 o[NQ][CT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = row_frag_global<T>(qp + min(q, p.Tq - 1) * p.qr, S::KSTEP * s + Frag<T>::N * g, p.ch, q < p.Tq);
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[i][c] = ZERO4;
    }
    load_lut(p, w.h, S::PAD, lut);
    __syncthreads();
    const float flo = lut[0], fhi = lut[2 * (p.R + S::PAD)], *lut0 = lut + p.R + S::PAD;
    const float sl = p.scale * LOG2E;
    for (int t = t0; t < t1; ++t) {
        T* const Kt = tiles + (t & 1) * 2 * KT * P;
        T* const Vt = Kt + KT * P;
        ck.put(Kt, p.ch, tid);
        cv.put(Vt, p.ch, tid);
        __syncthreads();                                                    // (the other pair of tiles is read until here)
        const int k0 = t * KT;
        if (t + 1 < t1) {
            ck.fetch(kp + (long)(k0 + KT) * p.kr, p.kr, kend - k0 - KT, p.ch, tid);
            cv.fetch(vp + (long)(k0 + KT) * p.vr, p.vr, kend - k0 - KT, p.ch, tid);
        }
        if (qw >= p.Tq || (p.causal && k0 > pmax)) continue;               // (a wave without queries, or past its last key)
        f32x4 s[NQ][N16];
#pragma unroll
        for (int n = 0; n < N16; ++n) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) s[i][n] = ZERO4;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const frag a = row_frag<T>(Kt, P, 16 * n, S::KSTEP * ks, lane);
#pragma unroll
                for (int i = 0; i < NQ; ++i) s[i][n] = mma(a, qf[i][ks], s[i][n]);
            }
        }
        const int side = side_of(k0, KT, pmin, pmax, p.R);
        const bool masked = k0 + KT > nk || (p.causal && k0 + KT - 1 > pmin);
        // far from the diagonal and whole: one multiply-add turns a raw score into the exponent (its maximum is the raw maximum's)
        const bool plain = side && !masked && sl > 0.f;
        const float b = side < 0 ? flo : fhi, mul = plain ? sl : 1.f, add = plain ? b : 0.f;
        if (!plain) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) bias_mask<N16>(s[i], sl, lut0, side, b, masked, k0, nk, pmin + 16 * i + (lane & 15), p.causal, lane);
        }
        float mx[NQ], c0[NQ];
        bool rise = false;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            mx[i] = max_of<N16>(s[i]) * mul + add;
            rise = rise || mx[i] > m[i] + 8.f;
        }
        if (__any(rise)) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const float mn = fmaxf(m[i], col_max(mx[i])), f = exp2_raw(m[i] - (mn == -INFINITY ? 0.f : mn));
                m[i] = mn;
                l[i] *= f;
#pragma unroll
                for (int c = 0; c < CT; ++c) o[i][c] *= f;
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) c0[i] = add - (m[i] == -INFINITY ? 0.f : m[i]);
        // the exponentials of one step beside the products of the one before
#pragma unroll
        for (int kb = 0; kb < N16; kb += S::NP) {
            frag pf[NQ];
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
#pragma unroll
                for (int n = 0; n < S::NP; ++n) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[i][kb + n][r] = exp2_raw(s[i][kb + n][r] * mul + c0[i]);
                    l[i] += (s[i][kb + n][0] + s[i][kb + n][1]) + (s[i][kb + n][2] + s[i][kb + n][3]);
                }
                pf[i] = acc_frag<T>(&s[i][kb]);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const frag a = col_frag<T>(Vt, P, 16 * kb, 16 * c, lane);
#pragma unroll
                for (int i = 0; i < NQ; ++i) o[i][c] = mma(a, pf[i], o[i][c]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int q = qw + 16 * i + (lane & 15);
        const float lt = col_sum(l[i]);
        if (q < p.Tq) finish_query<T, CT>(p, w.b, w.h, q, split, o[i], m[i], lt, g);
    }
}

// Few queries (a kv head's query heads times Tq at most 16 - decoding): they are the 16 columns of one tile, so the group's heads share one
// read of the keys and values.  Bound by that read: the waves split the keys, key fragments go from memory straight to the matrix unit, values
// through the wave's own LDS tile to be read transposed; workgroups split the keys further and k_rel_attention_join adds up.
// The matrix unit waits for memory here, so P goes into its product with v twice, rounded and what the rounding left: the output is off by its own rounding
// alone (bf16 1.66e-3 of its size against 2.3e-3, fp16 2.1e-4 against 2.9e-4; 48.1 -> 48.4 and 26.5 -> 27.0 us in the first two examples).
// 32 sequences of 4096 keys, 4 kv heads of 128 bf16: 48 us, 5.6 TB/s; 2 of 30001 fp16: 27 + 4 us, 3.9 TB/s; 8 of 1000, 16 heads of 64: 15 + 4 us, where
// the launches and the dependent loads of three tiles count.
template <typename T, int CHP>
__global__ __launch_bounds__(NTHR, CHP > 64 ? 2 : 4) void k_rel_attention_few(AttP p) {
    typedef Shape<T, CHP> S;
    typedef typename Frag<T>::type frag;
    constexpr int KT = S::F32 ? 16 : 32, KS = S::KS, CT = S::CT, P = S::PITCH, N16 = KT / 16, OP = CHP + 4;
    constexpr size_t TILE = KT * P * sizeof(T), OUT = 16 * OP * sizeof(float);
    __shared__ __attribute__((aligned(16))) unsigned char smem[NWAVE * (TILE > OUT ? TILE : OUT)];
    __shared__ float ml[NWAVE][16][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, col = lane & 15;
    const int rep = p.H / p.Hk, split = blockIdx.x % p.splits, unit = blockIdx.x / p.splits, b = unit / p.Hk, hk = unit % p.Hk;
    const int nk = keys_of(p, b), qs = start_of(p, b);
    const bool there = col < rep * p.Tq;
    const int h = hk * rep + (there ? col / p.Tq : 0), q = there ? col % p.Tq : 0, pos = qs + q;
    const int kend = p.causal ? max(0, min(nk, qs + p.Tq)) : nk;
    const int nt = (kend + KT - 1) / KT, t0 = (int)((long)nt * split / p.splits), t1 = (int)((long)nt * (split + 1) / p.splits);
    const T* kp = (const T*)p.k + b * p.kb + (long)hk * p.ch;
    const T* vp = (const T*)p.v + b * p.vb + (long)hk * p.ch;
    const T* qp = (const T*)p.q + b * p.qb + q * p.qr + (long)h * p.ch;
    T* const Vt = (T*)(smem + wave * TILE);
    Carrier<T, CHP, KT, 64> cv(p.vr, p.ch, lane);
    frag kf[N16][KS];
    auto fetch_k = [&](int t) {
#pragma unroll
        for (int n = 0; n < N16; ++n) {
            const int key = min(t * KT + 16 * n + col, kend - 1);
#pragma unroll
            for (int s = 0; s < KS; ++s) kf[n][s] = load16<T>(kp + key * p.kr, S::KSTEP * s + Frag<T>::N * g, p.ch);
        }
    };
    if (t0 + wave < t1) {
        fetch_k(t0 + wave);
        cv.fetch(vp + (long)(t0 + wave) * KT * p.vr, p.vr, kend - (t0 + wave) * KT, p.ch, lane);
    }
    frag qf[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = row_frag_global<T>(qp, S::KSTEP * s + Frag<T>::N * g, p.ch, there);
    const float flo = bias_at(p, h, 0), fhi = bias_at(p, h, 2 * p.R), sl = p.scale * LOG2E;
    f32x4 o[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c] = ZERO4;
    float m = -INFINITY, l = 0.f;
    // the next tile's keys are requested as soon as the products have taken the present ones, its values once those lie in LDS
    for (int t = t0 + wave; t < t1; t += NWAVE) {
        const int k0 = t * KT;
        f32x4 s[N16];
        const bool whole = k0 + KT <= kend && p.ch == S::KW;
#pragma unroll
        for (int n = 0; n < N16; ++n) {
            s[n] = ZERO4;
            if (!whole) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kf[n][ks] = keep16<T>(kf[n][ks], S::KSTEP * ks + Frag<T>::N * g, p.ch, k0 + 16 * n + col < kend);
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[n] = mma(kf[n][ks], qf[ks], s[n]);
        }
        if (t + NWAVE < t1) fetch_k(t + NWAVE);
        __builtin_amdgcn_wave_barrier();                                    // (the tile is this wave's own; LDS keeps a wave's order)
        cv.put(Vt, p.ch, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (t + NWAVE < t1) cv.fetch(vp + (long)(k0 + NWAVE * KT) * p.vr, p.vr, kend - k0 - NWAVE * KT, p.ch, lane);
        const int side = side_of(k0, KT, qs, qs + p.Tq - 1, p.R);
        if (side) {
            const float bias = side < 0 ? flo : fhi;
#pragma unroll
            for (int n = 0; n < N16; ++n) s[n] = s[n] * sl + bias;
        } else {
#pragma unroll
            for (int n = 0; n < N16; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[n][r] = s[n][r] * sl + bias_at(p, h, min(max(k0 + 16 * n + 4 * g + r - pos, -p.R), p.R) + p.R);
        }
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int kk = k0 + 16 * n + 4 * g + r;
                if (kk >= nk || (p.causal && kk > pos)) s[n][r] = -INFINITY;
            }
        const float mx = max_of<N16>(s);
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, col_max(mx)), f = exp2_raw(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= f;
#pragma unroll
            for (int c = 0; c < CT; ++c) o[c] *= f;
        }
        const float c0 = m == -INFINITY ? 0.f : -m;
#pragma unroll
        for (int n = 0; n < N16; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = exp2_raw(s[n][r] + c0);
                l += s[n][r];
            }
#pragma unroll
        for (int kb = 0; kb < N16; kb += S::NP) {
            const frag pf = acc_frag<T>(&s[kb]);
            frag pl;                                                        // P as two numbers of the tensors' type
            if constexpr (!S::F32) {
                const f32x4 lo[2] = {rest4<T>(s[kb]), rest4<T>(s[kb + 1])};
                pl = acc_frag<T>(lo);
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const frag x = col_frag<T>(Vt, P, 16 * kb, 16 * c, lane);
                o[c] = mma(x, pf, o[c]);
                if constexpr (!S::F32) o[c] = mma(x, pl, o[c]);
            }
        }
    }
    l = col_sum(l);
    __syncthreads();
    float* const mine = (float*)(smem + wave * OUT) + col * OP;
#pragma unroll
    for (int c = 0; c < CT; ++c) *(f32x4*)(mine + 16 * c + 4 * g) = o[c];
    if (g == 0) { ml[wave][col][0] = m; ml[wave][col][1] = l; }
    __syncthreads();
    if (wave != 0 || !there) return;
    // the first wave adds the waves up and finishes its columns
    float M = -INFINITY, L = 0.f, f[NWAVE];
#pragma unroll
    for (int x = 0; x < NWAVE; ++x) M = fmaxf(M, ml[x][col][0]);
#pragma unroll
    for (int x = 0; x < NWAVE; ++x) {
        f[x] = exp2_raw(ml[x][col][0] - (M == -INFINITY ? 0.f : M));
        L += f[x] * ml[x][col][1];
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        o[c] = ZERO4;
#pragma unroll
        for (int x = 0; x < NWAVE; ++x) o[c] += f[x] * *(const f32x4*)((float*)(smem + x * OUT) + col * OP + 16 * c + 4 * g);
    }
    finish_query<T, CT>(p, b, h, q, split, o, M, L, g);
}

// One workgroup a row (b, h, q): the splits' weights (a thread each), then their sums times the weights, 32 threads across the channels and 8
// runs of splits side by side, added in order.
constexpr int SMAX = 128;
template <typename T>
__global__ __launch_bounds__(NTHR) void k_rel_attention_join(AttP p) {
    __shared__ float wt[SMAX], red[2 * NWAVE];
    __shared__ f32x4 sum[8][32];
    const long rows = (long)p.B * p.H * p.Tq, row = blockIdx.x;
    const int tid = threadIdx.x, c = 4 * (tid & 31), run = tid >> 5, per = (p.splits + 7) / 8, s0 = run * per, s1 = min(s0 + per, p.splits);
    float m = -INFINITY, l = 0.f;
    if (tid < p.splits) {
        const float2 x = *(const float2*)(p.part_ml + 2 * (tid * rows + row));
        m = x.x;
        l = x.y;
    }
    float M = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float w = exp2_raw(m - (M == -INFINITY ? 0.f : M)), part = wave_sum(w * l);
    if (tid < p.splits) wt[tid] = w;
    if ((tid & 63) == 0) red[NWAVE + (tid >> 6)] = part;
    __syncthreads();
    const float L = (red[NWAVE] + red[NWAVE + 1]) + (red[NWAVE + 2] + red[NWAVE + 3]);
    f32x4 a = ZERO4;
    if (c < p.ch) {
        const float* src = p.part + row * p.ch + c;
#pragma unroll 4
        for (int s = s0; s < s1; ++s) a += wt[s] * *(const f32x4*)(src + s * rows * p.ch);
    }
    sum[run][tid & 31] = a;
    __syncthreads();
    if (run || c >= p.ch) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) a += sum[i][tid];
    a *= L > 0.f || L != L ? 1.0f / L : 0.f;
    const int q = (int)(row % p.Tq), h = (int)(row / p.Tq % p.H), b = (int)(row / p.Tq / p.H);
    store4<T>((T*)p.o + b * p.ob + q * p.orow + (long)h * p.ch, c, p.ch, a);
    if (sizeof(T) == 2 && p.olo) store4<T>((T*)p.olo + row * p.ch, c, p.ch, rest4<T>(a));
    if (p.lse && c == 0) p.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * LN2;
}

// How the forward pass splits the keys: a few queries a kv head go to k_rel_attention_few; too few workgroups for the 256 CUs share a row's
// keys - about 512 workgroups of at least 128 keys (few queries) or 256 (tiles of queries).  Few queries, 2 x 30001 keys of 4 heads of 128: 30 us with
// 512, 35 with 1024 workgroups; 4 x 2000 keys of 16 heads of 72 in fp32: 23 and 28 us.  Tiles of queries, bf16, whole and split: 8 workgroups of 2000 keys
// 44 and 20 us, 64 of 4096 (64 wide) 80 and 38, of 1024 27 and 26.  More workgroups than 64 fill enough of the chip that the sums' way through memory costs
// more than the rest of it gives, but for long rows: 128 of 1024 keys 28 and 40 us, 192 28 and 51, 216 of 2048 47 and 61; 128 of 4096 79 and 51, 160 (128 wide)
// 116 and 88, 192 of 8192 152 and 132 - in as many whole shares as 512 workgroups hold (160 in four instead of three: 100).  fp32, slower a key and three workgroups
// a CU: 128 of 1024 58 and 42, 240 of 2048 111 and 103, 240 of 4096 211 and 173.
struct Plan { bool few; int splits; };
Plan plan(const dua_rel_attention_args* a) {
    const long rep = a->heads / a->kv_heads, units = (long)a->B * a->kv_heads;
    Plan pl{rep * a->Tq <= 16, 1};
    const long wgs = pl.few ? units : units * rep * ((a->Tq + query_block(a->dtype) - 1) / query_block(a->dtype));
    const long up = (512 + wgs - 1) / wgs, most = a->Tk / (pl.few ? 128 : 256);
    long s = up;
    if (!pl.few) {
        if (wgs >= 256) s = 1;
        else if (a->dtype != DUA_DTYPE_F32 && wgs > 64) s = a->Tk >= 4096 ? 512 / wgs : 1;
    }
    if (s > most) s = most;
    s = s < 1 ? 1 : (s > SMAX ? SMAX : s);
    pl.splits = (int)s;
    return pl;
}

// Unnormalised sums of the splits
size_t split_floats(const dua_rel_attention_args* a, int splits) { return (size_t)splits * a->B * a->heads * a->Tq * a->ch; }

template <typename T, int CHP> struct Fwd {
    static int run(AttP p, bool few, hipStream_t st) {
        typedef Shape<T, CHP> S;
        const long rows = (long)p.B * p.H * p.Tq;
        if (few) {
            if (int rc = launch<k_rel_attention_few<T, CHP>>("dua_rel_attention", dim3((unsigned)(p.B * p.Hk * p.splits)), NTHR, 0, st, p)) return rc;
        } else {
            const unsigned grid = grid_of(p, p.H / p.Hk, (p.Tq + S::QB - 1) / S::QB);
            const size_t lds = 4 * S::TILE + (2 * (p.R + S::PAD) + 1) * sizeof(float);
            if (int rc = launch<k_rel_attention<T, CHP>>("dua_rel_attention", dim3(grid, p.splits), NTHR, lds, st, p)) return rc;
        }
        return p.splits > 1 ? launch<k_rel_attention_join<T>>("dua_rel_attention", dim3((unsigned)rows), NTHR, 0, st, p) : DUA_OK;
    }
};
}  // namespace

extern "C" size_t dua_rel_attention_workspace_bytes(const dua_rel_attention_args* a, int backward) {
    if (!a || check_common(a, "dua_rel_attention_workspace_bytes", backward != 0)) return 0;
    const size_t rows = (size_t)a->B * a->heads * a->Tq;
    if (backward) return rel_attention_bwd_bytes(a);
    if (rows == 0) return 0;
    const int s = plan(a).splits;
    return s > 1 ? (split_floats(a, s) + 2 * s * rows) * sizeof(float) : 0;
}

extern "C" int dua_rel_attention(const dua_rel_attention_args* a, void* stream) {
    if (int rc = check_common(a, "dua_rel_attention", false)) return rc;
    if (a->B == 0 || a->Tq == 0) return DUA_OK;
    DUA_REQUIRE(a->out, "dua_rel_attention: null output");
    const Plan pl = plan(a);
    DUA_REQUIRE(pl.splits == 1 || (a->workspace && ((uintptr_t)a->workspace & 15) == 0 && a->workspace_bytes >= dua_rel_attention_workspace_bytes(a, 0)),
                "dua_rel_attention: workspace smaller than dua_rel_attention_workspace_bytes, or not 16-byte aligned");
    AttP p = pack(a);
    p.splits = pl.splits;
    p.part = (float*)a->workspace;
    p.part_ml = p.part + split_floats(a, pl.splits);
    return dispatch<Fwd>(a->dtype, p, pl.few, as_stream(stream));
}
