// The norms around a transformer block fused with its gate and residual scale, and their gradients:
//   u = post(y)        post: none, RMS norm or LayerNorm of the block's output, times post_w (+ post_b)
//   r = a * x + g * u  the residual stream after the block (a: residual scale; g: gate of a channel, of a sample's channels, or none)
//   z = pre(r)         the next block's input: none, RMS norm or LayerNorm of the UNROUNDED r, times pre_w (+ pre_b)
// One pass: x and y are read once, r and z written once (4 elements of traffic; backward 6: x, y, dr, dz -> dx, dy).  Both norms of a row
// need the whole row, so the lanes of one unit hold it in registers, 16 bytes a lane, and walk several rows;
// the parameters of its columns stay in registers over the rows (read per row they would be L2 traffic of the size of the tensors' own).
// All sums and statistics are fp32; variances are sums of squared differences from the mean (no E[x^2] - mean^2 cancellation).
#include <atomic>
#include "elem.h"

namespace {

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
constexpr int MAX_WAVES = 16;
constexpr int MAX_D = MAX_WAVES * 64 * 8;

// Rows go to UNITS of threads: 16 or 32 lanes or a whole wavefront (narrow rows; 4 wavefronts a workgroup), or a workgroup of up to 16 wavefronts.
// A unit's rows lie side by side with the other units' (consecutive addresses at any time: rows dealt in runs met the same memory channels,
// 83 against 58 us on 16512 rows of 1152 floats) but within one gate row where there are enough of them.
struct NormP {
    const void *x, *y, *post_w, *post_b, *gate, *pre_w, *pre_b;
    void *r, *z;
    float* stats;
    long rows, per_gate, gates;           // per_gate: rows that share a gate row
    int D, post, pre;
    float res_scale, eps, inv_d;
    long units, per_sample;               // units in all; of one gate row (0: a unit takes whole gate rows)
    // backward
    const void *dr, *dz;
    void *dx, *dy;
    float *part, *gate_part;              // [blocks][5][D]: gate (if it has one row), post_w, post_b, pre_w, pre_b;  [units][D]: gate of several rows
    void* dgate;
    int one_gate;
};

// A unit's walk: rows c, c + per_sample, ... of its gate row, or gate rows unit, unit + units, ... whole.
struct Walk {
    long row, end, gate, step;
    __device__ Walk(const NormP& p, long unit) {
        if (p.per_sample > 0) {
            const unsigned u = (unsigned)unit, ps = (unsigned)p.per_sample;   // (units are launched threads: below 2^32)
            gate = u / ps;
            step = ps;
            row = gate * p.per_gate + u % ps;
        } else {
            gate = unit;
            step = 1;
            row = gate * p.per_gate;
        }
        end = unit < p.units ? min((gate + 1) * p.per_gate, p.rows) : row;
    }
    __device__ bool live() const { return row < end; }
    __device__ void next(const NormP& p) {
        row += step;
        if (row >= end && p.per_sample == 0 && gate + p.units < p.gates) {
            gate += p.units;
            row = gate * p.per_gate;
            end = row + p.per_gate;
        }
    }
};

// Sums over a unit.  LANES = 0: the workgroup's waves meet in LDS; `buf` holds two sets so that one barrier per sum is enough (the set written two
// sums ago is no longer read once everybody passed the barrier in between).
template <int LANES> struct UnitSum {
    float* buf;
    int nw, wave, lane, set;
    __device__ UnitSum(float* b) : buf(b), nw(blockDim.x >> 6), wave(threadIdx.x >> 6), lane(threadIdx.x & 63), set(0) {}
    __device__ __forceinline__ float in_wave(float v) {
        if constexpr (LANES == 16 || LANES == 32) {
            v += dpp_move<0x128>(v);                            // rotations by 8, 4, 2, 1 of the 16 lanes of a row: everyone gets the sum
            v += dpp_move<0x124>(v);
            v += dpp_move<0x122>(v);
            v += dpp_move<0x121>(v);
            if (LANES == 32) v += __shfl_xor(v, 16, 64);
            return v;
        } else {
            return wave_sum(v);
        }
    }
    __device__ __forceinline__ void two(float& a, float& b) {
        a = in_wave(a);
        b = in_wave(b);
        if (LANES) return;
        float* s = buf + set * 2 * MAX_WAVES;
        set ^= 1;
        if (lane == 0) { s[wave] = a; s[MAX_WAVES + wave] = b; }
        __syncthreads();
        a = row_sum16(lane < nw ? s[lane] : 0.f);
        b = row_sum16(lane < nw ? s[MAX_WAVES + lane] : 0.f);
    }
    __device__ __forceinline__ float one(float a) {
        a = in_wave(a);
        if (LANES) return a;
        float* s = buf + set * 2 * MAX_WAVES;
        set ^= 1;
        if (lane == 0) s[wave] = a;
        __syncthreads();
        return row_sum16(lane < nw ? s[lane] : 0.f);
    }
    // Mean and sum of squared differences from it over the row in one barrier: every wave about its own mean, then the waves' means about the
    // whole one (nothing is subtracted that is large against the spread).  s, q: of this wave; n: elements of wave `lane`.
    __device__ __forceinline__ void moments(float s, float q, float n, float inv_d, float& mean, float& m2) {
        float* x = buf + set * 2 * MAX_WAVES;
        set ^= 1;
        if (lane == 0) { x[wave] = s; x[MAX_WAVES + wave] = q; }
        __syncthreads();
        const bool in = lane < nw;
        const float sl = in ? x[lane] : 0.f, ql = in ? x[MAX_WAVES + lane] : 0.f;
        mean = row_sum16(sl) * inv_d;
        const float d = in && n > 0.f ? sl / n - mean : 0.f;
        m2 = row_sum16(ql + n * d * d);
    }
};

// Elements of one access: 16 bytes, or all that a thread holds
template <typename T, int PL> constexpr int chunk_of() { return PL < Elem<T>::VEC ? PL : Elem<T>::VEC; }

// Where a thread stands in its unit, and the columns it holds: chunks of V elements, threads side by side, PL elements in all.  A chunk that
// would stick out of the row lies at its end instead (the elements it shares with the chunk before do not count: valid), and so does one past
// the row: every load is a whole, unconditional one.  (Loads behind a lane's own condition, zeros otherwise, cost half the bandwidth: the zeros wait for
// the loads into the same registers.  16512 rows of 1152 floats: 82 us, 1024: 45 us.)
template <int V, int PL, int LANES> struct Cols {
    static constexpr int THREADS = LANES;
    __device__ static __forceinline__ int width() { return LANES ? LANES : (int)blockDim.x; }
    __device__ static __forceinline__ int pos() { return LANES ? (int)threadIdx.x % (LANES ? LANES : 1) : (int)threadIdx.x; }
    __device__ static __forceinline__ long unit() { return LANES ? (long)blockIdx.x * (256 / (LANES ? LANES : 256)) + (int)threadIdx.x / (LANES ? LANES : 1) : (long)blockIdx.x; }
    __device__ static __forceinline__ int start(int e) { return ((e / V) * width() + pos()) * V; }
    __device__ static __forceinline__ int of(int e, int D) { return min(start(e), max(D - V, 0)) + e % V; }
    __device__ static __forceinline__ bool valid(int e, int D) { return of(e, D) >= start(e) && of(e, D) < D; }
    // elements of the row that wave w of the workgroup holds
    __device__ static __forceinline__ int held_by(int w, int D) {
        int n = 0;
#pragma unroll
        for (int e = 0; e < PL; e += V) n += min(max(D - ((e / V) * width() + w * 64) * V, 0), 64 * V);
        return n;
    }
};

// This thread's part of a row as it lies in memory (rows may begin anywhere); elements that are not valid hold others of the row
template <typename T, typename C, int PL> struct Part {
    static constexpr int V = chunk_of<T, PL>(), N = PL / V;
    typename VecOf<T, V>::type x[N];
    __device__ __forceinline__ void load(const T* p, int D) {
        if (D >= V) {
#pragma unroll
            for (int u = 0; u < N; ++u) x[u] = *(const typename MemVec<T, V>::type*)(p + C::of(u * V, D));
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int j = 0; j < V; ++j) x[u][j] = p[min(j, D - 1)];
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return (float)x[e / V][e % V]; }
};
// (V: consecutive elements of a thread - those of the tensors' type, whatever T is)
template <typename T, int V, typename C, int PL>
__device__ __forceinline__ void store_row(T* p, int D, const float* f) {
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        if (C::start(e) + V <= D) {
            st_elems<T, V>(p + C::start(e), f + e);
        } else if (C::start(e) < D) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (C::valid(e + j, D)) p[C::of(e + j, D)] = (T)f[e + j];
        }
    }
}
// Parameters of this thread's columns; `dflt` where there are none.
template <typename T, typename PT, typename C, int PL>
__device__ __forceinline__ void load_param(const void* p, int D, float dflt, float* f) {
    constexpr int V = chunk_of<T, PL>();
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        if (!p) {
#pragma unroll
            for (int j = 0; j < V; ++j) f[e + j] = dflt;
        } else if (D >= V) {
            ld_elems<PT, V>((const PT*)p + C::of(e, D), f + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) f[e + j] = (float)((const PT*)p)[min(j, D - 1)];
        }
    }
}
// ... kept over the unit's rows in registers, or (rows of more than 4096 elements in the backward pass, whose state fills the registers) in LDS slots
// of the thread's own
template <int PL, bool LDS> struct Kept {
    float f[LDS ? 1 : PL];
    float* slot;
    __device__ __forceinline__ void set(float* lds, int which, const float* v) {
        if constexpr (LDS) {
            slot = lds + which * PL * (int)blockDim.x + 4 * threadIdx.x;
#pragma unroll
            for (int e = 0; e < PL; e += 4) *(float4*)(slot + e * (int)blockDim.x) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
#pragma unroll
            for (int e = 0; e < PL; ++e) f[e] = v[e];
        }
    }
    __device__ __forceinline__ void get(float* v) const {
        if constexpr (LDS) {
#pragma unroll
            for (int e = 0; e < PL; e += 4) {
                const float4 q = *(const float4*)(slot + e * (int)blockDim.x);
                v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < PL; ++e) v[e] = f[e];
        }
    }
};

template <typename C, int V, int PL, int LANES>
__device__ __forceinline__ void row_stats(const float* f, int D, int kind, float inv_d, float eps, UnitSum<LANES>& us, float& mean, float& rstd) {
    float q = 0.f, m2;
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PL; ++e) s += C::valid(e, D) ? f[e] : 0.f;
        s = us.in_wave(s);
        mean = LANES ? s * inv_d : s / fmaxf((float)C::held_by(us.wave, D), 1.f);
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float d = f[e] - mean;
            q += C::valid(e, D) ? d * d : 0.f;
        }
        q = us.in_wave(q);
        if (LANES) m2 = q;
        else us.moments(s, q, us.lane < us.nw ? (float)C::held_by(us.lane, D) : 0.f, inv_d, mean, m2);
    } else {
#pragma unroll
        for (int e = 0; e < PL; ++e) q += C::valid(e, D) ? f[e] * f[e] : 0.f;
        mean = 0.f;
        m2 = us.one(q);
    }
    rstd = 1.0f / sqrtf(m2 * inv_d + eps);
}

// LANES: a unit's lanes (16, 32, 64), 0: the workgroup of at most WAVES wavefronts.  PL: elements of a row a thread.  The loads of the next row are in
// flight while one is reduced (of the next two: no faster, 5 - 20 % slower where the registers then hold fewer waves).  Bound by memory: called over and
// over on the same rows, partly from the 256 MB cache, 5.2 - 6.3 TB/s at widths that fill their waves (8192 rows of 4096 bf16 47 us, 16384 of 1024 fp32
// 43 us; a copy of 512 MB: 5.3), in a training step 56 us (4.8 TB/s) for the first; the vector unit is busy two thirds of the time.  Rows whose last wave is
// mostly empty wait for their barriers (16512 rows of 1152 fp32, 4.5 of 5 waves: 74 us, 4.1 TB/s, in a training step 88; bf16, 2.25 of 3:
// 34 - 49 us, 3.1 - 4.4).
template <typename T, typename PT, int LANES, int WAVES, int PL>
__global__ __launch_bounds__(64 * WAVES) void k_sandwich_norm(NormP p) {
    constexpr int V = chunk_of<T, PL>();
    typedef Cols<V, PL, LANES> C;
    __shared__ float buf[4 * MAX_WAVES];
    UnitSum<LANES> us(buf);
    const int D = p.D;
    Walk w(p, C::unit()), ahead = w;                             // the row at hand, the row to request next
    Part<T, C, PL> nx, ny;
    auto fetch = [&] {
        if (ahead.live()) {
            nx.load((const T*)p.x + ahead.row * D, D);
            ny.load((const T*)p.y + ahead.row * D, D);
            ahead.next(p);
        }
    };
    fetch();
    float pw[PL], pb[PL], qw[PL], qb[PL], g[PL];
    load_param<T, PT, C, PL>(p.gate && w.live() ? (const PT*)p.gate + w.gate * D : nullptr, D, 1.f, g);
    load_param<T, PT, C, PL>(p.post_w, D, 1.f, pw);
    load_param<T, PT, C, PL>(p.post_b, D, 0.f, pb);
    load_param<T, PT, C, PL>(p.pre_w, D, 1.f, qw);
    load_param<T, PT, C, PL>(p.pre_b, D, 0.f, qb);
    while (w.live()) {
        const long row = w.row, gate = w.gate;
        float x[PL], y[PL], u[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) { x[e] = p.res_scale * nx[e]; y[e] = ny[e]; u[e] = g[e]; }
        fetch();
        w.next(p);
        if (p.gate && w.live() && w.gate != gate) load_param<T, PT, C, PL>((const PT*)p.gate + w.gate * D, D, 1.f, g);
        float my = 0.f, ry = 1.f, mr = 0.f, rr = 1.f;
        if (p.post != NORM_NONE) row_stats<C, V, PL, LANES>(y, D, p.post, p.inv_d, p.eps, us, my, ry);
        float r[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            u[e] *= p.post != NORM_NONE ? (y[e] - my) * ry * pw[e] + pb[e] : y[e];
            r[e] = x[e] + u[e];
        }
        store_row<T, V, C, PL>((T*)p.r + row * D, D, r);
        if (p.pre != NORM_NONE) {
            row_stats<C, V, PL, LANES>(r, D, p.pre, p.inv_d, p.eps, us, mr, rr);
            float z[PL];
#pragma unroll
            for (int e = 0; e < PL; ++e) z[e] = (r[e] - mr) * rr * qw[e] + qb[e];
            store_row<T, V, C, PL>((T*)p.z + row * D, D, z);
        }
        if (p.stats && C::pos() == 0) *(float4*)(p.stats + 4 * row) = make_float4(my, ry, mr, rr);
    }
}

// Gradients.  With h the normalised row and e = d * w, the input gradient of a norm is rstd * (e - mean(e) [LayerNorm] - h * mean(e h)).
//   t = dr + pre'(dz);  dx = a t;  du = g t;  dgate = sum t u;  dy = post'(du);  dpost_w = sum du hy;  dpost_b = sum du;  dpre_w = sum dz hr.
// r is not read: it is x, y and the saved statistics again, in fp32 (reading it would replace x and bring its rounding into hr).
// A unit sums its rows' columns in registers, a workgroup its units in their order, k_sandwich_cols the workgroups in theirs: the same
// sums in every run.  Bound by memory and by the registers of five column sums: 8192 rows of 4096 bf16 82 us, 4.9 TB/s; 16512 of 1152 fp32 114 us, 4.0;
// rows of more than 4096 elements spill (4096 rows of 8192 fp32 294 us, 2.7; bf16 rows of 8192 3.3).
template <typename T, typename PT, int LANES, int WAVES, int PL, bool LDS>
__global__ __launch_bounds__(64 * WAVES) void k_sandwich_norm_bwd(NormP p) {
    constexpr int V = chunk_of<T, PL>();
    typedef Cols<V, PL, LANES> C;
    __shared__ float buf[4 * MAX_WAVES];
    extern __shared__ __attribute__((aligned(16))) float dyn[];
    UnitSum<LANES> us(buf);
    const int D = p.D;
    Walk w(p, C::unit()), ahead = w;
    Part<T, C, PL> nx, ny, ndr, ndz;
    float4 nst;
    auto fetch = [&] {
        if (ahead.live()) {
            const long row = ahead.row;
            ny.load((const T*)p.y + row * D, D);
            ndr.load((const T*)p.dr + row * D, D);
            nx.load((const T*)p.x + row * D, D);
            if (p.pre != NORM_NONE) ndz.load((const T*)p.dz + row * D, D);
            nst = *(const float4*)(p.stats + 4 * row);
            ahead.next(p);
        }
    };
    Kept<PL, LDS> kg, kpw, kpb, kqw;
    auto fetch_gate = [&] {
        float v[PL];
        load_param<T, PT, C, PL>(p.gate ? (const PT*)p.gate + w.gate * D : nullptr, D, 1.f, v);
        kg.set(dyn, 0, v);
    };
    if (w.live()) fetch_gate();
    fetch();
    {
        float v[PL];
        load_param<T, PT, C, PL>(p.post_w, D, 1.f, v);
        kpw.set(dyn, 1, v);
        load_param<T, PT, C, PL>(p.post_b, D, 0.f, v);
        kpb.set(dyn, 2, v);
        load_param<T, PT, C, PL>(p.pre_w, D, 1.f, v);
        kqw.set(dyn, 3, v);
    }
    float ag[PL], apw[PL], apb[PL], aqw[PL], aqb[PL];
#pragma unroll
    for (int e = 0; e < PL; ++e) ag[e] = apw[e] = apb[e] = aqw[e] = aqb[e] = 0.f;
    while (w.live()) {
        const long row = w.row, gate = w.gate;
        const float4 st = nst;
        float g[PL], u[PL], hy[PL], t[PL], hr[PL], dz[PL], v[PL];
        kg.get(g);
        kpw.get(v);
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float y = ny[e];
            hy[e] = (y - st.x) * st.y;
            u[e] = p.post != NORM_NONE ? hy[e] * v[e] : y;
        }
        if (p.post_b) {
            kpb.get(v);
#pragma unroll
            for (int e = 0; e < PL; ++e) u[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            t[e] = ndr[e];
            hr[e] = (p.res_scale * nx[e] + g[e] * u[e] - st.z) * st.w;
            dz[e] = p.pre != NORM_NONE && C::valid(e, D) ? ndz[e] : 0.f;
        }
        fetch();
        w.next(p);
        const bool last = !w.live() || w.gate != gate;          // of its gate row (for a unit of whole gate rows: its sums are complete)
        if (w.live() && w.gate != gate) fetch_gate();
        if (p.pre != NORM_NONE) {
            float s1 = 0.f, s2 = 0.f;
            kqw.get(v);
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const float q = dz[e] * v[e];
                s1 += q;
                s2 += C::valid(e, D) ? q * hr[e] : 0.f;
                aqw[e] += dz[e] * hr[e];
                aqb[e] += dz[e];
                v[e] = q;
            }
            if (p.pre == NORM_LAYER) {
                us.two(s1, s2);
                s1 *= p.inv_d;
            } else {
                s2 = us.one(s2);
                s1 = 0.f;
            }
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) t[e] += st.w * (v[e] - s1 - hr[e] * s2);
        }
        float o[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) o[e] = p.res_scale * t[e];
        store_row<T, V, C, PL>((T*)p.dx + row * D, D, o);
        float s1 = 0.f, s2 = 0.f;
        kpw.get(v);
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const bool in = C::valid(e, D);
            t[e] = in ? t[e] : 0.f;
            ag[e] += t[e] * u[e];
            o[e] = t[e] * g[e];                                // du
            apw[e] += o[e] * hy[e];
            apb[e] += o[e];
            o[e] *= p.post != NORM_NONE ? v[e] : 1.f;
            s1 += o[e];
            s2 += in ? o[e] * hy[e] : 0.f;
        }
        if (p.post != NORM_NONE) {
            if (p.post == NORM_LAYER) {
                us.two(s1, s2);
                s1 *= p.inv_d;
            } else {
                s2 = us.one(s2);
                s1 = 0.f;
            }
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = st.y * (o[e] - s1 - hy[e] * s2);
        }
        store_row<T, V, C, PL>((T*)p.dy + row * D, D, o);
        if (p.gate && last && p.per_sample == 0) {
            store_row<PT, V, C, PL>((PT*)p.dgate + gate * D, D, ag);
#pragma unroll
            for (int e = 0; e < PL; ++e) ag[e] = 0.f;
        }
    }
    if (p.gate && p.per_sample > 0 && !p.one_gate && C::unit() < p.units) store_row<float, V, C, PL>(p.gate_part + C::unit() * D, D, ag);
    const bool want[5] = {p.gate && p.one_gate, p.post_w != nullptr, p.post_b != nullptr, p.pre_w != nullptr, p.pre_b != nullptr};
    float* const acc[5] = {ag, apw, apb, aqw, aqb};
    float* out = p.part + (long)blockIdx.x * 5 * D;
    if constexpr (LANES == 0) {
#pragma unroll
        for (int i = 0; i < 5; ++i)
            if (want[i]) store_row<float, V, C, PL>(out + i * D, D, acc[i]);
    } else {
        // the workgroup's units, one after the other
        for (int i = threadIdx.x; i < 5 * D; i += 256) dyn[i] = 0.f;
        const int mine = (int)threadIdx.x / LANES;
        for (int x = 0; x < 256 / LANES; ++x) {
            __syncthreads();
            if (x != mine) continue;
#pragma unroll
            for (int i = 0; i < 5; ++i)
                if (want[i]) {
#pragma unroll
                    for (int e = 0; e < PL; ++e) {
                        if (C::valid(e, D)) dyn[i * D + C::of(e, D)] += acc[i][e];
                    }
                }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 5 * D; i += 256) out[i] = dyn[i];
    }
}

// Column sums of the workgroups' partial sums, in their order; all parameters in one launch (blockIdx.y walks the gate's rows, then the
// parameters).  64 columns a workgroup, its 16 waves a run of partial sums each.
struct ColsP {
    const float *part, *gate_part;
    int D;
    void* dst[5];
    long blocks, gate_per;
    int gate_rows, which[5];                                  // gate_rows: of a gate with several rows; which[i]: the parameter of blockIdx.y = gate_rows + i
};
template <typename PT>
__global__ __launch_bounds__(1024) void k_sandwich_cols(ColsP p) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const bool gate = (int)blockIdx.y < p.gate_rows;
    const int w = gate ? 0 : p.which[blockIdx.y - p.gate_rows];
    const long s = gate ? blockIdx.y : 0, per = gate ? p.gate_per : p.blocks, step = (gate ? 1 : 5) * (long)p.D;
    const long q = (per + 15) / 16, i0 = wave * q, i1 = min(i0 + q, per);
    float a = 0.f;
    if (c < p.D) {
        const float* src = (gate ? p.gate_part + s * per * p.D : p.part + (long)w * p.D) + c;
#pragma unroll 8
        for (long i = i0; i < i1; ++i) a += src[i * step];
    }
    sm[wave][lane] = a;
    __syncthreads();
    if (wave == 0 && c < p.D) {
        for (int i = 1; i < 16; ++i) a += sm[i][lane];
        ((PT*)p.dst[w])[s * p.D + c] = (PT)a;
    }
}

int check_common(const dua_sandwich_norm_args* a, const char* who) {
    DUA_REQUIRE(a, "%s: null arguments", who);
    DUA_REQUIRE(dua_dtype_ok(a->dtype) && dua_dtype_ok(a->param_dtype) && (a->param_dtype == DUA_DTYPE_F32 || a->param_dtype == a->dtype),
                "%s: dtype must be fp32, bf16 or fp16 and the parameters' fp32 or the same", who);
    DUA_REQUIRE(a->rows >= 0 && a->D >= 1 && a->D <= MAX_D, "%s: D must be in [1, %d]", who, MAX_D);
    DUA_REQUIRE(a->post >= 0 && a->post <= 2 && a->pre >= 0 && a->pre <= 2, "%s: norm kinds are 0 (none), 1 (RMS), 2 (LayerNorm)", who);
    DUA_REQUIRE((a->post || (!a->post_w && !a->post_b)) && (a->pre || (!a->pre_w && !a->pre_b)), "%s: parameters given for a norm that is off", who);
    DUA_REQUIRE(!a->gate || (a->gate_rows >= 1 && a->rows % a->gate_rows == 0), "%s: the gate's rows must divide the rows", who);
    DUA_REQUIRE(a->rows == 0 || (a->x && a->y), "%s: null operand", who);
    DUA_REQUIRE(a->eps >= 0.f, "%s: eps must not be negative", who);
    return DUA_OK;
}

NormP pack(const dua_sandwich_norm_args* a) {
    NormP p{};
    p.x = a->x; p.y = a->y; p.post_w = a->post_w; p.post_b = a->post_b; p.gate = a->gate; p.pre_w = a->pre_w; p.pre_b = a->pre_b;
    p.r = a->r; p.z = a->z; p.stats = a->stats; p.rows = a->rows; p.D = a->D; p.post = a->post; p.pre = a->pre;
    p.gates = a->gate ? a->gate_rows : 1;
    p.per_gate = a->rows / p.gates;
    p.res_scale = a->res_scale; p.eps = a->eps; p.inv_d = 1.0f / (float)a->D;
    p.dr = a->dr; p.dz = a->dz; p.dx = a->dx; p.dy = a->dy; p.dgate = a->dgate;
    p.one_gate = a->gate_rows == 1;
    return p;
}

bool aligned16(const void* q) { return ((uintptr_t)q & 15) == 0; }

// The unit of a row: 16 bytes a lane up to D = 4096 (sixteen-bit elements: 8, fp32: 4), beyond it 16 waves with 8 elements a lane.  Backward, sixteen-bit
// rows take 4 elements a lane too: with 8 the registers leave two waves a SIMD, and a unit of few waves leaves some of those empty (65536 rows
// of 128 bf16 43 -> 32 us, 16512 of 1152 75 -> 57, 8192 of 2560 67 -> 57) - but units of 7 and 8 waves fill them (8192 rows of 3584: 76 us
// against 81, of 4096: 82 against 84).
struct Unit { int pl, lanes, waves, per_block; };
Unit unit_of(const dua_sandwich_norm_args* a, bool backward) {
    const bool eight = a->D > 4096 || (a->dtype != DUA_DTYPE_F32 && (!backward || (a->D + 511) / 512 >= 7));
    const int pl = eight ? 8 : 4, threads = (a->D + pl - 1) / pl;
    if (threads <= 16) return {pl, 16, 4, 16};
    if (threads <= 32) return {pl, 32, 4, 8};
    if (threads <= 64) return {pl, 64, 4, 4};
    return {pl, 0, (threads + 63) / 64, 1};
}
// How the rows are dealt: the same number of workgroups to every CU (half a round more cost a third: 3 against 2 workgroups of 8 waves on 8192 rows of
// 4096 bf16, 55 against 47 us), `waves` wavefronts a CU; each unit takes at least `least` rows where there are that many.
struct Deal { long units, per_sample, blocks; };
Deal deal(const dua_sandwich_norm_args* a, const Unit& u, int waves, long least) {
    Deal d{0, 1, 0};
    if (a->rows == 0) return d;
    const long most = 256L * (waves / u.waves > 1 ? waves / u.waves : 1) * u.per_block, g = a->gate ? a->gate_rows : 1, t = a->rows / g;
    long each = (a->rows + most - 1) / most;
    if (each < least) each = least;
    if (t >= each) {
        d.per_sample = most / g > 1 && most / g <= t ? most / g : (t + each - 1) / each;
        if (t / d.per_sample < least) d.per_sample = (t + least - 1) / least;
        d.units = g * d.per_sample;
    } else {
        d.per_sample = 0;
        d.units = (g + each / t - 1) / (each / t);
    }
    d.blocks = (d.units + u.per_block - 1) / u.per_block;
    return d;
}
// Wavefronts that the kernels' registers let a CU hold.  Forward (fp32 rows keep half the elements a lane): 16512 rows of 1152 floats 74 us with 20 or 24
// waves, 83 with 16; 8192 rows of 4096 bf16 47 us with 16 to 24.  Backward (the partial sums, 5 rows of floats a workgroup, want few): 16512 rows
// of 1152 floats 117 us with 12, 135 with 16; bf16 57 us with 16, 64 with 12; 8192 rows of 4096 bf16 82 us with 12, 87 with 16.
Deal deal_fwd(const dua_sandwich_norm_args* a) { return deal(a, unit_of(a, false), a->dtype == DUA_DTYPE_F32 ? 20 : 16, 1); }
Deal deal_bwd(const dua_sandwich_norm_args* a) {
    const Unit u = unit_of(a, true);
    return deal(a, u, a->dtype == DUA_DTYPE_F32 || u.pl == 8 ? 12 : 16, 4);
}
size_t gate_floats(const dua_sandwich_norm_args* a, const Deal& d) { return a->gate && a->gate_rows > 1 && d.per_sample > 0 ? (size_t)d.units * a->D : 0; }

template <template <typename, typename, int, int, int> class L, bool BWD>
void dispatch(const dua_sandwich_norm_args* a, const NormP& p, unsigned grid, hipStream_t st) {
    const Unit u = unit_of(a, BWD);
    const bool pf = a->param_dtype == DUA_DTYPE_F32;
    const unsigned block = 64 * u.waves;
#define GO(T, PT)                                                                                        \
    {                                                                                                    \
        constexpr int PL = BWD ? 4 : Elem<T>::VEC;                                                       \
        if (a->D > 4096) L<T, PT, 0, 16, 8>::run(p, grid, block, st);                                    \
        else if (u.lanes == 16) L<T, PT, 16, 4, PL>::run(p, grid, block, st);                            \
        else if (u.lanes == 32) L<T, PT, 32, 4, PL>::run(p, grid, block, st);                            \
        else if (u.lanes == 64) L<T, PT, 64, 4, PL>::run(p, grid, block, st);                            \
        else if (u.pl == 8) L<T, PT, 0, 8, Elem<T>::VEC>::run(p, grid, block, st);                       \
        else if constexpr (PL == 4) {                                                                    \
            if (u.waves > 8) L<T, PT, 0, 16, 4>::run(p, grid, block, st);                                \
            else L<T, PT, 0, 8, 4>::run(p, grid, block, st);                                             \
        }                                                                                                \
    }
    if (a->dtype == DUA_DTYPE_F32) GO(float, float)
    else if (a->dtype == DUA_DTYPE_BF16) { if (pf) GO(bf16_t, float) else GO(bf16_t, bf16_t) }
    else { if (pf) GO(f16_t, float) else GO(f16_t, f16_t) }
#undef GO
}
template <typename T, typename PT, int LANES, int W, int PL> struct LFwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) { hipLaunchKernelGGL((k_sandwich_norm<T, PT, LANES, W, PL>), grid, block, 0, st, p); }
};
template <typename T, typename PT, int LANES, int W, int PL> struct LBwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) {
        constexpr bool LDS = LANES == 0 && PL == 8 && W == 16;                 // the four parameters of a thread's columns in LDS: at most 128 KB
        const size_t lds = LDS ? 4 * PL * (size_t)block * sizeof(float) : (LANES ? 5 * (size_t)p.D * sizeof(float) : 0);
        auto* kernel = &k_sandwich_norm_bwd<T, PT, LANES, W, PL, LDS>;
        if (lds > 64 * 1024) {                                                 // asked for once a device; refused, the launch reports it
            static std::atomic<unsigned> asked{0};
            int dev = 0;
            (void)hipGetDevice(&dev);
            const unsigned bit = 1u << (dev & 31);
            if (!(asked.load() & bit) && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024) == hipSuccess) asked.fetch_or(bit);
        }
        hipLaunchKernelGGL(kernel, grid, block, lds, st, p);
    }
};

}  // namespace

extern "C" int dua_sandwich_norm(const dua_sandwich_norm_args* a, void* stream) {
    if (int rc = check_common(a, "dua_sandwich_norm")) return rc;
    if (a->rows == 0) return DUA_OK;
    DUA_REQUIRE(a->r && (a->pre == NORM_NONE || a->z), "dua_sandwich_norm: null output");
    DUA_REQUIRE(!a->stats || aligned16(a->stats), "dua_sandwich_norm: stats must be 16-byte aligned");
    NormP p = pack(a);
    const Deal d = deal_fwd(a);
    p.units = d.units;
    p.per_sample = d.per_sample;
    dispatch<LFwd, false>(a, p, (unsigned)d.blocks, as_stream(stream));
    return dua_check_launch("dua_sandwich_norm");
}

extern "C" size_t dua_sandwich_norm_bwd_workspace_bytes(const dua_sandwich_norm_args* a) {
    if (!a || check_common(a, "dua_sandwich_norm_bwd_workspace_bytes")) return 0;
    const Deal d = deal_bwd(a);
    return ((size_t)d.blocks * 5 * a->D + gate_floats(a, d)) * sizeof(float);
}

extern "C" int dua_sandwich_norm_bwd(const dua_sandwich_norm_args* a, void* stream) {
    if (int rc = check_common(a, "dua_sandwich_norm_bwd")) return rc;
    DUA_REQUIRE((!a->gate || a->dgate) && (!a->post_w || a->dpost_w) && (!a->post_b || a->dpost_b) && (!a->pre_w || a->dpre_w) &&
                (!a->pre_b || a->dpre_b), "dua_sandwich_norm_bwd: a parameter without its gradient's buffer");
    DUA_REQUIRE(a->rows == 0 || (a->dr && a->dx && a->dy && a->stats && (a->pre == NORM_NONE || a->dz)), "dua_sandwich_norm_bwd: null operand");
    DUA_REQUIRE(a->rows == 0 || aligned16(a->stats), "dua_sandwich_norm_bwd: stats must be 16-byte aligned");
    const Deal d = deal_bwd(a);
    DUA_REQUIRE(a->rows == 0 || (a->workspace && a->workspace_bytes >= dua_sandwich_norm_bwd_workspace_bytes(a)),
                "dua_sandwich_norm_bwd: workspace smaller than dua_sandwich_norm_bwd_workspace_bytes");
    // (k_sandwich_cols' grid; with rows there are at most as many gate rows with sums of their own as units on the chip)
    DUA_REQUIRE(!a->gate || a->gate_rows <= 65000 || d.per_sample == 0, "dua_sandwich_norm_bwd: an empty call's gate has at most 65000 rows");
    NormP p = pack(a);
    p.units = d.units;
    p.per_sample = d.per_sample;
    p.part = (float*)a->workspace;
    p.gate_part = p.part + (size_t)d.blocks * 5 * a->D;
    hipStream_t st = as_stream(stream);
    if (a->rows > 0) dispatch<LBwd, true>(a, p, (unsigned)d.blocks, st);
    ColsP q{};
    q.part = p.part; q.gate_part = p.gate_part; q.D = a->D; q.blocks = d.blocks;
    q.dst[0] = a->dgate; q.dst[1] = a->dpost_w; q.dst[2] = a->dpost_b; q.dst[3] = a->dpre_w; q.dst[4] = a->dpre_b;
    if (a->gate && a->gate_rows > 1 && (a->rows == 0 || d.per_sample > 0)) { q.gate_rows = (int)a->gate_rows; q.gate_per = a->rows ? d.per_sample : 0; }
    const bool given[5] = {a->gate && a->gate_rows == 1 && (a->rows == 0 || d.per_sample > 0), a->post_w != nullptr, a->post_b != nullptr,
                           a->pre_w != nullptr, a->pre_b != nullptr};
    int n = 0;
    for (int i = 0; i < 5; ++i)
        if (given[i]) q.which[n++] = i;
    if (q.gate_rows + n > 0) {
        const dim3 grid((a->D + 63) / 64, q.gate_rows + n);
        if (a->param_dtype == DUA_DTYPE_F32) hipLaunchKernelGGL(k_sandwich_cols<float>, grid, 1024, 0, st, q);
        else if (a->param_dtype == DUA_DTYPE_BF16) hipLaunchKernelGGL(k_sandwich_cols<bf16_t>, grid, 1024, 0, st, q);
        else hipLaunchKernelGGL(k_sandwich_cols<f16_t>, grid, 1024, 0, st, q);
    }
    return dua_check_launch("dua_sandwich_norm_bwd");
}
