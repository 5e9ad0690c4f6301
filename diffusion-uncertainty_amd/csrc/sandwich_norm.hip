// The norms around a transformer block fused with its gate and residual scale, and their gradients:
//   u = post(y)        post: none, RMS norm or LayerNorm of the block's output, times post_w (+ post_b)
//   r = a * x + g * u  the residual stream after the block (a: residual scale; g: gate of a channel, of a sample's channels, or none)
//   z = pre(r)         the next block's input: none, RMS norm or LayerNorm of the UNROUNDED r, times pre_w (+ pre_b)
// One pass: x and y are read once, r and z written once (4 elements of traffic; backward 6: x, y, dr, dz -> dx, dy).  Both norms of a row
// need the whole row, so one workgroup holds it in registers, 16 bytes a lane, and walks rows with a stride;
// the parameters of its columns stay in registers over the rows (read per row they would be L2 traffic of the size of the tensors' own).
// All sums and statistics are fp32; variances are sums of squared differences from the mean (no E[x^2] - mean^2 cancellation).
#include "elem.h"

namespace {

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
constexpr int MAX_WAVES = 16;
constexpr int MAX_D = MAX_WAVES * 64 * 8;

struct NormP {
    const void *x, *y, *post_w, *post_b, *gate, *pre_w, *pre_b;
    void *r, *z;
    float* stats;
    long rows, rows_per_gate;
    int D, post, pre;
    float res_scale, eps, inv_d;
    // backward
    const void *dr, *dz;
    void *dx, *dy;
    float* part;                          // [chunks][5][D]: gate, post_w, post_b, pre_w, pre_b column sums of a chunk of rows
    void* dgate;
    long chunk_rows, chunks_per_sample;   // chunks_per_sample == 0: a chunk holds whole samples and writes their gate gradients itself
};

// Sum over the workgroup's waves of up to two values; `buf` holds two sets so that one barrier per sum is enough (the set written two
// sums ago is no longer read once everybody passed the barrier in between).
struct BlockSum {
    float* buf;
    int nw, wave, lane, set;
    __device__ BlockSum(float* b, int n) : buf(b), nw(n), wave(threadIdx.x >> 6), lane(threadIdx.x & 63), set(0) {}
    __device__ __forceinline__ void two(float& a, float& b) {
        a = wave_sum(a);
        b = wave_sum(b);
        if (nw == 1) return;
        float* s = buf + set * 2 * MAX_WAVES;
        set ^= 1;
        if (lane == 0) { s[wave] = a; s[MAX_WAVES + wave] = b; }
        __syncthreads();
        const bool in = lane < nw;
        a = row_sum16(in ? s[lane] : 0.f);
        b = row_sum16(in ? s[MAX_WAVES + lane] : 0.f);
    }
    // Mean and sum of squared differences from it over the row in one barrier: every wave about its own mean, then the waves' means about the
    // whole one (nothing is subtracted that is large against the spread).  n: elements of wave `lane`, q, s: of this wave.
    __device__ __forceinline__ void moments(float s, float mw, float q, float n, float inv_d, float& mean, float& m2) {
        if (nw == 1) {
            mean = mw;
            m2 = q;
            return;
        }
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
    __device__ __forceinline__ float one(float a) {
        a = wave_sum(a);
        if (nw == 1) return a;
        float* s = buf + set * 2 * MAX_WAVES;
        set ^= 1;
        if (lane == 0) s[wave] = a;
        __syncthreads();
        return row_sum16(lane < nw ? s[lane] : 0.f);
    }
};

// Column of element e of this lane: 16-byte chunks of V elements, lanes side by side.
template <int V> __device__ __forceinline__ int col_of(int e) { return (e / V) * (int)blockDim.x * V + (int)threadIdx.x * V + e % V; }

// This lane's part of a row as it lies in memory (rows may begin anywhere), zeros past D
template <typename T, int PL> struct Part {
    static constexpr int V = Elem<T>::VEC, N = PL / V;
    typename VecOf<T, V>::type x[N];
    __device__ __forceinline__ void load(const T* p, int D) {
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = col_of<V>(u * V);
            if (c + V <= D) {
                x[u] = *(const typename MemVec<T, V>::type*)(p + c);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) x[u][j] = c + j < D ? p[c + j] : (T)0.f;
            }
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return (float)x[e / V][e % V]; }
};
template <typename T, int PL>
__device__ __forceinline__ void store_row(T* p, int D, const float* f) {
    constexpr int V = Elem<T>::VEC;
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        const int c = col_of<V>(e);
        if (c + V <= D) {
            st_elems<T, V>(p + c, f + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < D) p[c + j] = (T)f[e + j];
        }
    }
}
template <int V, int PL>
__device__ __forceinline__ void store_row_f32(float* p, int D, const float* f) {
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        const int c = col_of<V>(e);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < D) p[c + j] = f[e + j];
    }
}
// Parameters of this lane's columns; `dflt` where there are none.
template <typename T, typename PT, int PL>
__device__ __forceinline__ void load_param(const void* p, int D, float dflt, float* f) {
    constexpr int V = Elem<T>::VEC;
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        const int c = col_of<V>(e);
        if (p && c + V <= D) {
            ld_elems<PT, V>((const PT*)p + c, f + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) f[e + j] = p && c + j < D ? (float)((const PT*)p)[c + j] : dflt;
        }
    }
}

// Elements of the row that wave w holds
template <int V, int PL> __device__ __forceinline__ int held_by(int w, int D) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < PL; e += V) n += min(max(D - (e / V) * (int)blockDim.x * V - w * 64 * V, 0), 64 * V);
    return n;
}

template <int V, int PL>
__device__ __forceinline__ void row_stats(const float* f, int D, int kind, float inv_d, float eps, BlockSum& bs, float& mean, float& rstd) {
    float q = 0.f, m2;
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PL; ++e) s += f[e];            // (elements past D are zero)
        s = wave_sum(s);
        const int mine = held_by<V, PL>(bs.wave, D);
        const float mw = s / fmaxf((float)mine, 1.f);
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float d = f[e] - mw;
            q += col_of<V>(e) < D ? d * d : 0.f;
        }
        bs.moments(s, mw, wave_sum(q), bs.lane < bs.nw ? (float)held_by<V, PL>(bs.lane, D) : 0.f, inv_d, mean, m2);
    } else {
#pragma unroll
        for (int e = 0; e < PL; ++e) q += f[e] * f[e];
        mean = 0.f;
        m2 = bs.one(q);
    }
    rstd = 1.0f / sqrtf(m2 * inv_d + eps);
}

// PL elements of a row a lane, at most WAVES wavefronts a row: 16 bytes a lane (PL = 8, fp32 4) up to D = 4096, beyond it 16 waves of 8 elements.  The next row's loads are in flight while the present
// one is reduced.
template <typename T, typename PT, int WAVES, int PL>
__global__ __launch_bounds__(64 * WAVES) void k_sandwich_norm(NormP p) {
    constexpr int V = Elem<T>::VEC;
    __shared__ float buf[4 * MAX_WAVES];
    BlockSum bs(buf, blockDim.x >> 6);
    const int D = p.D;
    long row = blockIdx.x;
    Part<T, PL> nx, ny;
    nx.load((const T*)p.x + row * D, D);
    ny.load((const T*)p.y + row * D, D);
    float pw[PL], pb[PL], g[PL], qw[PL], qb[PL];
    load_param<T, PT, PL>(p.post_w, D, 1.f, pw);
    load_param<T, PT, PL>(p.post_b, D, 0.f, pb);
    load_param<T, PT, PL>(p.pre_w, D, 1.f, qw);
    load_param<T, PT, PL>(p.pre_b, D, 0.f, qb);
    long gate_at = -1;
#pragma unroll
    for (int e = 0; e < PL; ++e) g[e] = 1.f;
    while (row < p.rows) {
        float x[PL], y[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) { x[e] = nx[e]; y[e] = ny[e]; }
        if (p.gate) {
            const long gi = row / p.rows_per_gate;
            if (gi != gate_at) load_param<T, PT, PL>((const PT*)p.gate + gi * D, D, 0.f, g);
            gate_at = gi;
        }
        const long next = row + gridDim.x;
        if (next < p.rows) {
            nx.load((const T*)p.x + next * D, D);
            ny.load((const T*)p.y + next * D, D);
        }
        float my = 0.f, ry = 1.f, mr = 0.f, rr = 1.f;
        if (p.post != NORM_NONE) row_stats<V, PL>(y, D, p.post, p.inv_d, p.eps, bs, my, ry);
        float r[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float u = p.post != NORM_NONE ? (y[e] - my) * ry * pw[e] + pb[e] : y[e];
            r[e] = col_of<V>(e) < D ? p.res_scale * x[e] + g[e] * u : 0.f;
        }
        store_row<T, PL>((T*)p.r + row * D, D, r);
        if (p.pre != NORM_NONE) {
            row_stats<V, PL>(r, D, p.pre, p.inv_d, p.eps, bs, mr, rr);
            float z[PL];
#pragma unroll
            for (int e = 0; e < PL; ++e) z[e] = (r[e] - mr) * rr * qw[e] + qb[e];
            store_row<T, PL>((T*)p.z + row * D, D, z);
        }
        if (p.stats && threadIdx.x == 0) *(float4*)(p.stats + 4 * row) = make_float4(my, ry, mr, rr);
        row = next;
    }
}

// Gradients.  With h the normalised row and e = d * w, the input gradient of a norm is rstd * (e - mean(e) [LayerNorm] - h * mean(e h)).
//   t = dr + pre'(dz);  dx = a t;  du = g t;  dgate = sum t u;  dy = post'(du);  dpost_w = sum du hy;  dpost_b = sum du;  dpre_w = sum dz hr.
// r is not read: it is x, y and the saved statistics again, in fp32 (reading it would replace x and bring its rounding into hr).
// A workgroup owns a chunk of consecutive rows and sums its columns in registers; k_sandwich_cols adds the chunks in their order, so
// the sums are the same in every run.
template <typename T, typename PT, int WAVES, int PL>
__global__ __launch_bounds__(64 * WAVES) void k_sandwich_norm_bwd(NormP p) {
    constexpr int V = Elem<T>::VEC;
    __shared__ float buf[4 * MAX_WAVES];
    BlockSum bs(buf, blockDim.x >> 6);
    const int D = p.D;
    long r0, r1;
    const long ch = blockIdx.x;
    if (p.chunks_per_sample > 0) {
        const long s = ch / p.chunks_per_sample, c = ch % p.chunks_per_sample;
        r0 = s * p.rows_per_gate + c * p.chunk_rows;
        r1 = min(s * p.rows_per_gate + min((c + 1) * p.chunk_rows, p.rows_per_gate), p.rows);
    } else {
        r0 = ch * p.chunk_rows;
        r1 = min(r0 + p.chunk_rows, p.rows);
    }
    Part<T, PL> nx, ny, ndr, ndz;
    auto fetch = [&](long row) {
        ny.load((const T*)p.y + row * D, D);
        ndr.load((const T*)p.dr + row * D, D);
        nx.load((const T*)p.x + row * D, D);
        if (p.pre != NORM_NONE) ndz.load((const T*)p.dz + row * D, D);
    };
    if (r0 < r1) fetch(r0);
    float pw[PL], pb[PL], g[PL], qw[PL];
    load_param<T, PT, PL>(p.post_w, D, 1.f, pw);
    load_param<T, PT, PL>(p.post_b, D, 0.f, pb);
    load_param<T, PT, PL>(p.pre_w, D, 1.f, qw);
    float ag[PL], apw[PL], apb[PL], aqw[PL], aqb[PL];
#pragma unroll
    for (int e = 0; e < PL; ++e) { g[e] = 1.f; ag[e] = apw[e] = apb[e] = aqw[e] = aqb[e] = 0.f; }
    long gate_at = -1;
    for (long row = r0; row < r1; ++row) {
        const float4 st = *(const float4*)(p.stats + 4 * row);
        if (p.gate) {
            const long gi = row / p.rows_per_gate;
            if (gi != gate_at) {
                load_param<T, PT, PL>((const PT*)p.gate + gi * D, D, 0.f, g);
                if (p.chunks_per_sample == 0) {
#pragma unroll
                    for (int e = 0; e < PL; ++e) ag[e] = 0.f;
                }
                gate_at = gi;
            }
        }
        float u[PL], hy[PL], t[PL], hr[PL], dz[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float y = ny[e];
            hy[e] = (y - st.x) * st.y;
            u[e] = p.post != NORM_NONE ? hy[e] * pw[e] + pb[e] : y;
            t[e] = ndr[e];
            hr[e] = (p.res_scale * nx[e] + g[e] * u[e] - st.z) * st.w;
            dz[e] = p.pre != NORM_NONE ? ndz[e] : 0.f;
        }
        if (row + 1 < r1) fetch(row + 1);
        if (p.pre != NORM_NONE) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const float q = dz[e] * qw[e];               // (dz is zero past D)
                s1 += q;
                s2 += q * hr[e];
                aqw[e] += dz[e] * hr[e];
                aqb[e] += dz[e];
            }
            if (p.pre == NORM_LAYER) {
                bs.two(s1, s2);
                s1 *= p.inv_d;
            } else {
                s2 = bs.one(s2);
                s1 = 0.f;
            }
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) t[e] += st.w * (dz[e] * qw[e] - s1 - hr[e] * s2);
        }
        float o[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) o[e] = p.res_scale * t[e];
        store_row<T, PL>((T*)p.dx + row * D, D, o);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const bool in = col_of<V>(e) < D;
            t[e] = in ? t[e] : 0.f;
            ag[e] += t[e] * u[e];
            o[e] = t[e] * g[e];                              // du
            apw[e] += o[e] * hy[e];
            apb[e] += o[e];
            o[e] *= pw[e];
            s1 += o[e];
            s2 += in ? o[e] * hy[e] : 0.f;
        }
        if (p.post != NORM_NONE) {
            if (p.post == NORM_LAYER) {
                bs.two(s1, s2);
                s1 *= p.inv_d;
            } else {
                s2 = bs.one(s2);
                s1 = 0.f;
            }
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = st.y * (o[e] - s1 - hy[e] * s2);
        }
        store_row<T, PL>((T*)p.dy + row * D, D, o);
        if (p.gate && p.chunks_per_sample == 0 && (row + 1) % p.rows_per_gate == 0) {
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const int c = col_of<V>(e);
                if (c < D) ((PT*)p.dgate)[gate_at * D + c] = (PT)ag[e];
            }
        }
    }
    float* out = p.part + ch * 5 * D;
    if (p.gate && p.chunks_per_sample > 0) store_row_f32<V, PL>(out, D, ag);
    if (p.post_w) store_row_f32<V, PL>(out + D, D, apw);
    if (p.post_b) store_row_f32<V, PL>(out + 2 * D, D, apb);
    if (p.pre_w) store_row_f32<V, PL>(out + 3 * D, D, aqw);
    if (p.pre_b) store_row_f32<V, PL>(out + 4 * D, D, aqb);
}

// Column sums of the chunks' partial sums, in chunk order: dst[s][c] = sum over sample s's chunks of part[chunk][which][c].  All parameters in
// one launch (blockIdx.y walks the parameters and, for the gate, the samples); 64 columns a workgroup, its 16 waves a run of chunks each.
struct ColsP {
    const float* part;
    int D;
    void* dst[5];
    long chunks, gate_per;
    int gate_rows, nwhich, which[5];                          // which[i]: the parameters of blockIdx.y = gate_rows + i
};
template <typename PT>
__global__ __launch_bounds__(1024) void k_sandwich_cols(ColsP p) {
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const bool gate = (int)blockIdx.y < p.gate_rows;
    const int w = gate ? 0 : p.which[blockIdx.y - p.gate_rows];
    const long s = gate ? blockIdx.y : 0, per = gate ? p.gate_per : p.chunks, q = (per + 15) / 16, i0 = wave * q, i1 = min(i0 + q, per);
    float a = 0.f;
    if (c < p.D) {
        const float* src = p.part + (s * per * 5 + w) * p.D + c;
#pragma unroll 8
        for (long i = i0; i < i1; ++i) a += src[i * 5 * p.D];
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
    p.rows_per_gate = a->gate ? a->rows / a->gate_rows : a->rows;
    p.res_scale = a->res_scale; p.eps = a->eps; p.inv_d = 1.0f / (float)a->D;
    p.dr = a->dr; p.dz = a->dz; p.dx = a->dx; p.dy = a->dy; p.dgate = a->dgate;
    return p;
}

bool aligned16(const void* q) { return ((uintptr_t)q & 15) == 0; }

// wavefronts of a row: 16 bytes a lane up to D = 4096, fp32 beyond it 32
unsigned waves_of(const dua_sandwich_norm_args* a) {
    const int per = 64 * (a->dtype == DUA_DTYPE_F32 && a->D <= 4096 ? 4 : 8);
    return (unsigned)((a->D + per - 1) / per);
}

// Chunks of rows of the backward pass: about 12 waves a CU, at least 512 workgroups - the partial sums (5 rows of D floats a chunk) stay small
// against the tensors.
struct Chunks { long rows, per_sample, count; };
Chunks plan(const dua_sandwich_norm_args* a) {
    Chunks c{1, 1, 0};
    if (a->rows == 0) return c;
    const long most = 256L * 12 / waves_of(a) > 512 ? 256L * 12 / waves_of(a) : 512, target = (a->rows + most - 1) / most, g = a->gate ? a->gate_rows : 1, t = a->rows / g;
    if (t >= target) {
        c.per_sample = (t + target - 1) / target;
        c.rows = (t + c.per_sample - 1) / c.per_sample;
        c.per_sample = (t + c.rows - 1) / c.rows;
        c.count = g * c.per_sample;
    } else {
        c.per_sample = 0;
        c.rows = target / t * t;
        c.count = (a->rows + c.rows - 1) / c.rows;
    }
    return c;
}

template <template <typename, typename, int, int> class L>
void dispatch(const dua_sandwich_norm_args* a, const NormP& p, unsigned grid, unsigned waves, hipStream_t st) {
    const bool pf = a->param_dtype == DUA_DTYPE_F32;
#define GO(T, PT)                                                              \
    {                                                                          \
        if (a->D > 4096) L<T, PT, 16, 8>::run(p, grid, 64 * waves, st);        \
        else L<T, PT, sizeof(T) == 4 ? 16 : 8, Elem<T>::VEC>::run(p, grid, 64 * waves, st); \
    }
    if (a->dtype == DUA_DTYPE_F32) GO(float, float)
    else if (a->dtype == DUA_DTYPE_BF16) { if (pf) GO(bf16_t, float) else GO(bf16_t, bf16_t) }
    else { if (pf) GO(f16_t, float) else GO(f16_t, f16_t) }
#undef GO
}
template <typename T, typename PT, int W, int PL> struct LFwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) { hipLaunchKernelGGL((k_sandwich_norm<T, PT, W, PL>), grid, block, 0, st, p); }
};
template <typename T, typename PT, int W, int PL> struct LBwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) { hipLaunchKernelGGL((k_sandwich_norm_bwd<T, PT, W, PL>), grid, block, 0, st, p); }
};

}  // namespace

extern "C" int dua_sandwich_norm(const dua_sandwich_norm_args* a, void* stream) {
    if (int rc = check_common(a, "dua_sandwich_norm")) return rc;
    if (a->rows == 0) return DUA_OK;
    DUA_REQUIRE(a->r && (a->pre == NORM_NONE || a->z), "dua_sandwich_norm: null output");
    DUA_REQUIRE(!a->stats || aligned16(a->stats), "dua_sandwich_norm: stats must be 16-byte aligned");
    const NormP p = pack(a);
    const unsigned nw = waves_of(a);
    // at most 16 waves a CU, the rows dealt evenly: a workgroup's parameters cost as much as several of its rows
    const long cap = 256L * 16 / nw, each = (a->rows + cap - 1) / cap;
    dispatch<LFwd>(a, p, (unsigned)((a->rows + each - 1) / each), nw, as_stream(stream));
    return dua_check_launch("dua_sandwich_norm");
}

extern "C" size_t dua_sandwich_norm_bwd_workspace_bytes(const dua_sandwich_norm_args* a) {
    if (!a || check_common(a, "dua_sandwich_norm_bwd_workspace_bytes")) return 0;
    return (size_t)plan(a).count * 5 * a->D * sizeof(float);
}

extern "C" int dua_sandwich_norm_bwd(const dua_sandwich_norm_args* a, void* stream) {
    if (int rc = check_common(a, "dua_sandwich_norm_bwd")) return rc;
    DUA_REQUIRE((!a->gate || a->dgate) && (!a->post_w || a->dpost_w) && (!a->post_b || a->dpost_b) && (!a->pre_w || a->dpre_w) &&
                (!a->pre_b || a->dpre_b), "dua_sandwich_norm_bwd: a parameter without its gradient's buffer");
    DUA_REQUIRE(a->rows == 0 || (a->dr && a->dx && a->dy && a->stats && (a->pre == NORM_NONE || a->dz)), "dua_sandwich_norm_bwd: null operand");
    DUA_REQUIRE(a->rows == 0 || aligned16(a->stats), "dua_sandwich_norm_bwd: stats must be 16-byte aligned");
    const Chunks c = plan(a);
    DUA_REQUIRE(a->rows == 0 || (a->workspace && a->workspace_bytes >= (size_t)c.count * 5 * a->D * sizeof(float)),
                "dua_sandwich_norm_bwd: workspace smaller than dua_sandwich_norm_bwd_workspace_bytes");
    DUA_REQUIRE(!a->gate || a->gate_rows <= 65000 || c.per_sample == 0, "dua_sandwich_norm_bwd: more than 65000 gate rows of many rows each");
    NormP p = pack(a);
    p.part = (float*)a->workspace; p.chunk_rows = c.rows; p.chunks_per_sample = c.per_sample;
    hipStream_t st = as_stream(stream);
    if (a->rows > 0) dispatch<LBwd>(a, p, (unsigned)c.count, waves_of(a), st);
    ColsP q{};
    q.part = p.part; q.D = a->D; q.chunks = c.count;
    q.dst[0] = a->dgate; q.dst[1] = a->dpost_w; q.dst[2] = a->dpost_b; q.dst[3] = a->dpre_w; q.dst[4] = a->dpre_b;
    if (a->gate && (a->rows == 0 || c.per_sample > 0)) { q.gate_rows = (int)a->gate_rows; q.gate_per = a->rows ? c.per_sample : 0; }
    const void* given[5] = {nullptr, a->post_w, a->post_b, a->pre_w, a->pre_b};
    for (int i = 1; i < 5; ++i)
        if (given[i]) q.which[q.nwhich++] = i;
    if (q.gate_rows + q.nwhich > 0) {
        const dim3 grid((a->D + 63) / 64, q.gate_rows + q.nwhich);
        if (a->param_dtype == DUA_DTYPE_F32) hipLaunchKernelGGL(k_sandwich_cols<float>, grid, 1024, 0, st, q);
        else if (a->param_dtype == DUA_DTYPE_BF16) hipLaunchKernelGGL(k_sandwich_cols<bf16_t>, grid, 1024, 0, st, q);
        else hipLaunchKernelGGL(k_sandwich_cols<f16_t>, grid, 1024, 0, st, q);
    }
    return dua_check_launch("dua_sandwich_norm_bwd");
}
