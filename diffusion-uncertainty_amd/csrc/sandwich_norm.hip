// The norms around a transformer block fused with its gate and residual scale, and their gradients:
//   u = post(y)        post: none, RMS norm or LayerNorm of the block's output, times post_w (+ post_b)
//   r = a * x + g * u  the residual stream after the block (a: residual scale; g: gate of a channel, of a sample's channels, or none)
//   z = pre(r)         the next block's input: none, RMS norm or LayerNorm of the UNROUNDED r, times pre_w (+ pre_b)
// One pass: x and y are read once, r and z written once (4 elements of traffic; backward 6: x, y, dr, dz -> dx, dy).  Both norms of a row
// need the whole row, so one workgroup of D / 512 wavefronts holds it in registers, 8 elements a lane, and walks rows with a stride;
// the parameters of its columns stay in registers over the rows (read per row they would be L2 traffic of the size of the tensors' own).
// All sums and statistics are fp32; variances are sums of squared differences from the mean (no E[x^2] - mean^2 cancellation).
#include "elem.h"

namespace {

enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
constexpr int PL = 8;                    // elements of a row per lane
constexpr int MAX_WAVES = 16;            // 16 waves * 64 lanes * 8 elements: D <= 8192

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
        a = b = 0.f;
        for (int i = 0; i < nw; ++i) { a += s[i]; b += s[MAX_WAVES + i]; }
    }
    __device__ __forceinline__ float one(float a) {
        float b = 0.f;
        two(a, b);
        return a;
    }
};

// Column of element e of this lane: chunks of V consecutive elements, lanes side by side.
template <int V> __device__ __forceinline__ int col_of(int e) { return (e / V) * (int)blockDim.x * V + (int)threadIdx.x * V + e % V; }

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int D, float* f) {
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        const int c = col_of<V>(e);
        if (c < D) {
            ld_elems<T, V>(p + c, f + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) f[e + j] = 0.f;
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int D, const float* f) {
#pragma unroll
    for (int e = 0; e < PL; e += V) {
        const int c = col_of<V>(e);
        if (c < D) st_elems<T, V>(p + c, f + e);
    }
}
// Parameters of this lane's columns (their own type and alignment: element loads, once a workgroup); `dflt` where there are none.
template <typename PT, int V>
__device__ __forceinline__ void load_param(const void* p, int D, float dflt, float* f) {
#pragma unroll
    for (int e = 0; e < PL; ++e) {
        const int c = col_of<V>(e);
        f[e] = p && c < D ? (float)((const PT*)p)[c] : dflt;
    }
}

template <int V>
__device__ __forceinline__ void row_stats(const float* f, int D, int kind, float inv_d, float eps, BlockSum& bs, float& mean, float& rstd) {
    mean = 0.f;
    if (kind == NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PL; ++e) s += f[e];            // (elements past D are zero)
        mean = bs.one(s) * inv_d;
    }
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < PL; ++e) {
        const float d = f[e] - mean;
        q += col_of<V>(e) < D ? d * d : 0.f;
    }
    rstd = 1.0f / sqrtf(bs.one(q) * inv_d + eps);
}

template <typename T, typename PT, int V>
__global__ __launch_bounds__(64 * MAX_WAVES) void k_sandwich_norm(NormP p) {
    __shared__ float buf[4 * MAX_WAVES];
    BlockSum bs(buf, blockDim.x >> 6);
    const int D = p.D;
    float pw[PL], pb[PL], g[PL], qw[PL], qb[PL];
    load_param<PT, V>(p.post_w, D, 1.f, pw);
    load_param<PT, V>(p.post_b, D, 0.f, pb);
    load_param<PT, V>(p.pre_w, D, 1.f, qw);
    load_param<PT, V>(p.pre_b, D, 0.f, qb);
    long gate_at = -1;
#pragma unroll
    for (int e = 0; e < PL; ++e) g[e] = 1.f;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        float x[PL], y[PL];
        load_row<T, V>((const T*)p.x + row * D, D, x);
        load_row<T, V>((const T*)p.y + row * D, D, y);
        if (p.gate) {
            const long gi = row / p.rows_per_gate;
            if (gi != gate_at) load_param<PT, V>((const PT*)p.gate + gi * D, D, 0.f, g);
            gate_at = gi;
        }
        float my = 0.f, ry = 1.f, mr = 0.f, rr = 1.f;
        if (p.post != NORM_NONE) row_stats<V>(y, D, p.post, p.inv_d, p.eps, bs, my, ry);
        float r[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            const float u = p.post != NORM_NONE ? (y[e] - my) * ry * pw[e] + pb[e] : y[e];
            r[e] = col_of<V>(e) < D ? p.res_scale * x[e] + g[e] * u : 0.f;
        }
        store_row<T, V>((T*)p.r + row * D, D, r);
        if (p.pre != NORM_NONE) {
            row_stats<V>(r, D, p.pre, p.inv_d, p.eps, bs, mr, rr);
            float z[PL];
#pragma unroll
            for (int e = 0; e < PL; ++e) z[e] = (r[e] - mr) * rr * qw[e] + qb[e];
            store_row<T, V>((T*)p.z + row * D, D, z);
        }
        if (p.stats && threadIdx.x == 0) *(float4*)(p.stats + 4 * row) = make_float4(my, ry, mr, rr);
    }
}

// Gradients.  With h the normalised row and e = d * w, the input gradient of a norm is rstd * (e - mean(e) [LayerNorm] - h * mean(e h)).
//   t = dr + pre'(dz);  dx = a t;  du = g t;  dgate = sum t u;  dy = post'(du);  dpost_w = sum du hy;  dpost_b = sum du;  dpre_w = sum dz hr.
// r is not read: it is x, y and the saved statistics again, in fp32 (reading it would replace x and bring its rounding into hr).
// A workgroup owns a chunk of consecutive rows and sums its columns in registers; k_sandwich_cols adds the chunks in their order, so
// the sums are the same in every run.
template <typename T, typename PT, int V>
__global__ __launch_bounds__(64 * MAX_WAVES) void k_sandwich_norm_bwd(NormP p) {
    __shared__ float buf[4 * MAX_WAVES];
    BlockSum bs(buf, blockDim.x >> 6);
    const int D = p.D;
    float pw[PL], pb[PL], g[PL], qw[PL];
    load_param<PT, V>(p.post_w, D, 1.f, pw);
    load_param<PT, V>(p.post_b, D, 0.f, pb);
    load_param<PT, V>(p.pre_w, D, 1.f, qw);
    float ag[PL], apw[PL], apb[PL], aqw[PL], aqb[PL];
#pragma unroll
    for (int e = 0; e < PL; ++e) { g[e] = 1.f; ag[e] = apw[e] = apb[e] = aqw[e] = aqb[e] = 0.f; }
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
    long gate_at = -1;
    for (long row = r0; row < r1; ++row) {
        float x[PL], y[PL], dr[PL], dz[PL];
        load_row<T, V>((const T*)p.x + row * D, D, x);
        load_row<T, V>((const T*)p.y + row * D, D, y);
        load_row<T, V>((const T*)p.dr + row * D, D, dr);
        if (p.pre != NORM_NONE) load_row<T, V>((const T*)p.dz + row * D, D, dz);
        const float4 st = *(const float4*)(p.stats + 4 * row);
        if (p.gate) {
            const long gi = row / p.rows_per_gate;
            if (gi != gate_at) {
                load_param<PT, V>((const PT*)p.gate + gi * D, D, 0.f, g);
                if (p.chunks_per_sample == 0) {
#pragma unroll
                    for (int e = 0; e < PL; ++e) ag[e] = 0.f;
                }
                gate_at = gi;
            }
        }
        float u[PL], hy[PL], t[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) {
            hy[e] = (y[e] - st.x) * st.y;
            u[e] = p.post != NORM_NONE ? hy[e] * pw[e] + pb[e] : y[e];
            t[e] = dr[e];
        }
        if (p.pre != NORM_NONE) {
            float hr[PL], s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                hr[e] = (p.res_scale * x[e] + g[e] * u[e] - st.z) * st.w;
                const float q = dz[e] * qw[e];               // (dz is zero past D)
                s1 += q;
                s2 += q * hr[e];
                aqw[e] += dz[e] * hr[e];
                aqb[e] += dz[e];
            }
            bs.two(s1, s2);
            s1 = p.pre == NORM_LAYER ? s1 * p.inv_d : 0.f;
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) t[e] += st.w * (dz[e] * qw[e] - s1 - hr[e] * s2);
        }
        float o[PL];
#pragma unroll
        for (int e = 0; e < PL; ++e) o[e] = p.res_scale * t[e];
        store_row<T, V>((T*)p.dx + row * D, D, o);
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
            bs.two(s1, s2);
            s1 = p.post == NORM_LAYER ? s1 * p.inv_d : 0.f;
            s2 *= p.inv_d;
#pragma unroll
            for (int e = 0; e < PL; ++e) o[e] = st.y * (o[e] - s1 - hy[e] * s2);
        }
        store_row<T, V>((T*)p.dy + row * D, D, o);
        if (p.gate && p.chunks_per_sample == 0 && (row + 1) % p.rows_per_gate == 0) {
#pragma unroll
            for (int e = 0; e < PL; ++e) {
                const int c = col_of<V>(e);
                if (c < D) ((PT*)p.dgate)[gate_at * D + c] = (PT)ag[e];
            }
        }
    }
    float* out = p.part + ch * 5 * D;
#pragma unroll
    for (int e = 0; e < PL; ++e) {
        const int c = col_of<V>(e);
        if (c >= D) continue;
        if (p.gate && p.chunks_per_sample > 0) out[c] = ag[e];
        if (p.post_w) out[D + c] = apw[e];
        if (p.post_b) out[2 * D + c] = apb[e];
        if (p.pre_w) out[3 * D + c] = aqw[e];
        if (p.pre_b) out[4 * D + c] = aqb[e];
    }
}

// dst[s][c] = sum over the `per` chunks of sample s of part[chunk][which][c], in chunk order: 64 columns a workgroup, its 4 waves a
// quarter of the chunks each.
template <typename PT>
__global__ __launch_bounds__(256) void k_sandwich_cols(const float* part, int which, int D, long per, PT* dst) {
    __shared__ float sm[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    const long s = blockIdx.y, q = (per + 3) / 4, i0 = wave * q, i1 = min(i0 + q, per);
    float a = 0.f;
    if (c < D)
        for (long i = i0; i < i1; ++i) a += part[((s * per + i) * 5 + which) * D + c];
    sm[wave][lane] = a;
    __syncthreads();
    if (wave == 0 && c < D) dst[s * D + c] = (PT)((sm[0][lane] + sm[1][lane]) + (sm[2][lane] + sm[3][lane]));
}

int check_common(const dua_sandwich_norm_args* a, const char* who) {
    DUA_REQUIRE(a, "%s: null arguments", who);
    DUA_REQUIRE(dua_dtype_ok(a->dtype) && dua_dtype_ok(a->param_dtype) && (a->param_dtype == DUA_DTYPE_F32 || a->param_dtype == a->dtype),
                "%s: dtype must be fp32, bf16 or fp16 and the parameters' fp32 or the same", who);
    DUA_REQUIRE(a->rows >= 0 && a->D >= 1 && a->D <= 512 * MAX_WAVES, "%s: D must be in [1, %d]", who, 512 * MAX_WAVES);
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

// Chunks of rows of the backward pass: 512 workgroups fill the chip twice and keep the partial sums (5 rows of D floats a chunk) small
// against the tensors.
struct Chunks { long rows, per_sample, count; };
Chunks plan(const dua_sandwich_norm_args* a) {
    Chunks c{1, 1, 0};
    if (a->rows == 0) return c;
    const long target = (a->rows + 511) / 512, g = a->gate ? a->gate_rows : 1, t = a->rows / g;
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

template <template <typename, typename, int> class L>
int dispatch(const dua_sandwich_norm_args* a, const NormP& p, bool vec, unsigned grid, unsigned block, hipStream_t st) {
    const bool pf = a->param_dtype == DUA_DTYPE_F32;
#define GO(T, PT)                                                              \
    {                                                                          \
        if (vec) L<T, PT, Elem<T>::VEC>::run(p, grid, block, st);              \
        else L<T, PT, 1>::run(p, grid, block, st);                             \
    }
    if (a->dtype == DUA_DTYPE_F32) GO(float, float)
    else if (a->dtype == DUA_DTYPE_BF16) { if (pf) GO(bf16_t, float) else GO(bf16_t, bf16_t) }
    else { if (pf) GO(f16_t, float) else GO(f16_t, f16_t) }
#undef GO
    return DUA_OK;
}
template <typename T, typename PT, int V> struct LFwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) { hipLaunchKernelGGL((k_sandwich_norm<T, PT, V>), grid, block, 0, st, p); }
};
template <typename T, typename PT, int V> struct LBwd {
    static void run(const NormP& p, unsigned grid, unsigned block, hipStream_t st) { hipLaunchKernelGGL((k_sandwich_norm_bwd<T, PT, V>), grid, block, 0, st, p); }
};

unsigned waves_of(int D) { return (unsigned)((D + 64 * PL - 1) / (64 * PL)); }

}  // namespace

extern "C" int dua_sandwich_norm(const dua_sandwich_norm_args* a, void* stream) {
    if (int rc = check_common(a, "dua_sandwich_norm")) return rc;
    if (a->rows == 0) return DUA_OK;
    DUA_REQUIRE(a->r && (a->pre == NORM_NONE || a->z), "dua_sandwich_norm: null output");
    DUA_REQUIRE(!a->stats || aligned16(a->stats), "dua_sandwich_norm: stats must be 16-byte aligned");
    const NormP p = pack(a);
    const bool vec = (size_t)a->D * dua_dtype_size(a->dtype) % 16 == 0 && aligned16(a->x) && aligned16(a->y) && aligned16(a->r) &&
                     (a->pre == NORM_NONE || aligned16(a->z));
    const unsigned nw = waves_of(a->D);
    const long cap = 256L * 32 / nw;
    dispatch<LFwd>(a, p, vec, (unsigned)(a->rows < cap ? a->rows : cap), 64 * nw, as_stream(stream));
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
    DUA_REQUIRE(!a->gate || a->gate_rows <= 65535 || c.per_sample == 0, "dua_sandwich_norm_bwd: more than 65535 gate rows of many rows each");
    NormP p = pack(a);
    p.part = (float*)a->workspace; p.chunk_rows = c.rows; p.chunks_per_sample = c.per_sample;
    hipStream_t st = as_stream(stream);
    if (a->rows > 0) {
        const bool vec = (size_t)a->D * dua_dtype_size(a->dtype) % 16 == 0 && aligned16(a->x) && aligned16(a->y) && aligned16(a->dr) &&
                         (a->pre == NORM_NONE || aligned16(a->dz)) && aligned16(a->dx) && aligned16(a->dy);
        dispatch<LBwd>(a, p, vec, (unsigned)c.count, 64 * waves_of(a->D), st);
    }
    auto cols = [&](int which, void* dst, long per, unsigned samples) {
        if (!dst) return;
        const dim3 grid((a->D + 63) / 64, samples);
        if (a->param_dtype == DUA_DTYPE_F32) hipLaunchKernelGGL(k_sandwich_cols<float>, grid, 256, 0, st, p.part, which, a->D, per, (float*)dst);
        else if (a->param_dtype == DUA_DTYPE_BF16) hipLaunchKernelGGL(k_sandwich_cols<bf16_t>, grid, 256, 0, st, p.part, which, a->D, per, (bf16_t*)dst);
        else hipLaunchKernelGGL(k_sandwich_cols<f16_t>, grid, 256, 0, st, p.part, which, a->D, per, (f16_t*)dst);
    };
    if (a->gate && (a->rows == 0 || c.per_sample > 0)) cols(0, a->dgate, a->rows ? c.per_sample : 0, (unsigned)a->gate_rows);
    cols(1, a->post_w ? a->dpost_w : nullptr, c.count, 1);
    cols(2, a->post_b ? a->dpost_b : nullptr, c.count, 1);
    cols(3, a->pre_w ? a->dpre_w : nullptr, c.count, 1);
    cols(4, a->pre_b ? a->dpre_b : nullptr, c.count, 1);
    return dua_check_launch("dua_sandwich_norm_bwd");
}
