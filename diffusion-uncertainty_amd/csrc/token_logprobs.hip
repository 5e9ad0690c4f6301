// Log probabilities of given tokens with the entropy of each row's distribution and its k best alternatives, and their gradient.
//   l = t x;  lse = log sum e^l;  logprob = l_id - lse;  H = -sum p l^  (l^ = l - lse, p = e^l^);  top k by (value descending, index ascending)
//   dx = t [ glp (d_id - p) + sum_j gtop_j (d_top_j - p) - gH p (l^ + H) ]
// Memory bound: the row is read once (backward: read once, written once).  One pass keeps, per thread, s = sum 2^(L - ref) and w = sum 2^(L - ref) (L - ref)
// of the logits in log2 units, L = x t log2 e, in fp32; ref is any float near the largest L and moves when a value passes it by 2^16, so lse =
// ln 2 (ref + log2 s), H = ln 2 (log2 s - w / s).  L - ref is one fused multiply-add, exact but for its rounding: offsets common to a row keep their digits
// as far as L has them.  Rows beyond +-2^28 (offsets of 1e30, masks of the type's lowest value everywhere) are summed again relative to their largest logit,
// x - m formed before the temperature and the base change (scan_huge).
// The alternatives ride along: a thread remembers the best value of its pairs of 16-byte groups (g, g + 256) with its pair, and the best value outside
// that pair.  The smallest of the k largest maxima of 64, 128 or 256 sets of threads (k up to 16, 32, 64) is a lower bound of the row's k-th largest value;
// only pairs that reach it are read again, a thread whose second value reaches it too is re-read whole, and the few candidates are ranked exactly.
// Rows with many equal values, NaN or +inf take an ordered scan of the row in the same kernel (select_ordered).
// A row may begin anywhere and be of any length.
// Measured: 2048 rows of 128000 bf16, 20 alternatives 118 us (4.5 TB/s; the vector unit is busy three quarters of the time: an exponential and some six more
// instructions an element), 106 without.  4112 rows of 16385 fp32 in a training step, inputs from memory: 88 us with 8 alternatives (3.1 TB/s: the waves wait
// three quarters of the time, and a row of 64 KB ends in reductions and the ranking, under which no load of its own runs; called over and over on
// one input, mostly from the 256 MB cache, 53), gradients 98 us (5.5 TB/s; 120 if the forward pass was long ago; 2048 rows of 128000 bf16 226, 4.7).
// 4 rows of 32000: 8 + 4 us in parts.
#include <float.h>
#include "elem.h"

namespace {

constexpr int NT = 256, NW = NT / 64;
constexpr int KMAX = 64;                 // alternatives
constexpr int CAP = 1024;                // candidates of the fast selection
constexpr int RESCAN = 64;               // threads re-read whole before the ordered scan is cheaper
constexpr int SMAX = 32;                 // parts of a row
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Sums of a set of logits in log2 units, L = x c with c = t log2 e: s = sum 2^(L - ref), w = sum 2^(L - ref) (L - ref).  The reference is any float
// near the largest L - d = fma(x, c, -ref) is exact but for its own rounding - so it moves only when a value passes it by 2^16.  Logits beyond
// +-2^28 (masks of the type's lowest value everywhere, offsets of 1e30) have no such reference: s comes out 0, infinite or NaN, and the
// row is summed again relative to its own largest logit (scan_huge), where L - ref = (x - m) c.
struct Soft { float ref, s, w; };
__device__ __forceinline__ void soft_shift(Soft& a, float d) {              // to a reference higher by -d; clamped: 2^-1e4 = 0 and no 0 * inf
    d = fmaxf(d, -1e4f);
    const float f = __builtin_amdgcn_exp2f(d);
    a.w = f * (a.w + a.s * d);
    a.s *= f;
}
__device__ __forceinline__ Soft soft_join(Soft a, Soft b, float c) {          // c: log2 units of a reference's unit
    const float ref = fmaxf(a.ref, b.ref);
    soft_shift(a, (a.ref - ref) * c);
    soft_shift(b, (b.ref - ref) * c);
    return Soft{ref, a.s + b.s, a.w + b.w};
}
constexpr float REF_MAX = 268435456.f;                                       // 2^28

// total order of floats as whole numbers: -0 = +0, every NaN above +inf
__device__ __forceinline__ uint32_t okey(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b >> 31) ? ~b : b | 0x80000000u;
}

struct LogpP {
    const void* x;
    const int64_t* ids;
    float *logprob, *entropy, *lse, *stats;          // stats [rows][4]: reference, log2 s, H, 1 if the reference is a logit (else log2 units)
    int64_t* top_ids;
    float* top_lp;
    long rows, ld, V;
    int k, splits;
    float t;
    float* part;                                      // [rows][splits][4 + 2 k]: ref, s, w, huge ; values ; indices (as int32 bits, within V < 2^30)
    // backward
    const float *dlp, *dent, *dtop;
    const int64_t* tids;
    void* dx;
    long ldd;
};

// The groups of VEC elements (16 bytes, at any address) of elements [v0, v1) of a row.  The last one is read up to v1 and overlaps the one before
// where it would stick out: holds() says which elements are its own.  Every load is whole and unconditional.
template <typename T> struct Groups {
    static constexpr int VEC = Elem<T>::VEC;
    typedef typename VecOf<T, VEC>::type Raw;
    const T* base;                                           // element v0
    long first;
    int len, n;
    __device__ Groups(const T* row, long v0, long v1) : base(row + v0), first(v0), len((int)(v1 - v0)), n((len + VEC - 1) / VEC) {}
    __device__ __forceinline__ int at(int g) const { return min(g * VEC, max(len - VEC, 0)); }
    __device__ __forceinline__ bool whole(int g) const { return (g + 1) * VEC <= len; }
    __device__ __forceinline__ bool holds(int g, int j) const { return at(g) + j >= g * VEC && at(g) + j < len; }
    __device__ __forceinline__ long index(int g, int j) const { return first + at(g) + j; }
    __device__ __forceinline__ const T* ptr(int g) const { return (const T*)((const char*)base + (unsigned)at(g) * (unsigned)sizeof(T)); }   // (rows of less than 4 GB)
    __device__ __forceinline__ Raw raw(int g) const {
        if (len >= VEC) return *(const typename MemVec<T, VEC>::type*)ptr(g);
        Raw r;
#pragma unroll
        for (int j = 0; j < VEC; ++j) r[j] = base[min(j, len - 1)];
        return r;
    }
    __device__ __forceinline__ void load(int g, float* f) const {                        // elements that are not group g's own: -inf
        const Raw r = raw(g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = holds(g, j) ? (float)r[j] : -INFINITY;
    }
};

struct __attribute__((aligned(16))) Shared {
    uint32_t key[NT];
    uint64_t cand[CAP];                   // candidates
    int rescan[RESCAN];
    Soft soft[NW];
    uint32_t tau;                         // (candidates of the fast selection reach it)
    int ncand, nrescan, any;
    uint64_t best[2][KMAX];               // the k best, sorted; running best of the ordered scan
};

// A candidate as one whole number that orders by value, then by the lower index
__device__ __forceinline__ uint64_t cand(uint32_t key, int idx) { return (uint64_t)key << 32 | (uint32_t)~idx; }
__device__ __forceinline__ uint32_t cand_key(uint64_t c) { return (uint32_t)(c >> 32); }
__device__ __forceinline__ int cand_idx(uint64_t c) { return (int)~(uint32_t)c; }
// Number of entries of list[0, n) that beat c; list is 16-byte aligned
__device__ __forceinline__ int rank_of(const uint64_t* list, int n, uint64_t c) {
    int r = 0;
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    const u64x2* two = (const u64x2*)list;
#pragma unroll 4
    for (int j = 0; j < n / 2; ++j) {
        const u64x2 q = two[j];
        r += (q[0] > c) + (q[1] > c);
    }
    if (n & 1) r += list[n - 1] > c;
    return r;
}
__device__ __forceinline__ int rank_of_thread(const uint32_t* key, uint32_t k, int t) {
    int r = 0;
    for (int j = 0; j < NT; ++j) r += key[j] > k || (key[j] == k && j < t);
    return r;
}

// Exact selection by one ordered scan: 256 groups at a time in index order; a chunk is looked at only if one of its values beats the k-th of
// the best so far.  Of a chunk only the k threads with the best (largest, then leftmost) maxima can hold winners: every element of another
// thread is beaten by those k maxima.  Leaves the k best, sorted, in sh.best[return value].
template <typename T>
__device__ int select_ordered(const Groups<T>& gr, int k, Shared& sh) {
    constexpr int VEC = Elem<T>::VEC;
    const int tid = threadIdx.x;
    int cur = 0;
    long have = 0;
    for (int g0 = 0; g0 < gr.n; g0 += NT) {
        const int g = g0 + tid;
        float f[VEC];
        uint32_t best = 0;                                     // 0: below every float's key
        if (g < gr.n) {
            gr.load(g, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (gr.holds(g, j)) best = max(best, okey(f[j]));
        }
        __syncthreads();
        if (tid == 0) { sh.any = 0; sh.ncand = 0; }
        sh.key[tid] = best;
        __syncthreads();
        const uint32_t bar = have >= k ? cand_key(sh.best[cur][k - 1]) : 0;
        if (best > bar) sh.any = 1;
        __syncthreads();
        if (!sh.any) continue;
        if (best > bar && rank_of_thread(sh.key, best, tid) < k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (gr.holds(g, j) && okey(f[j]) > bar) {
                    const int at = atomicAdd(&sh.ncand, 1);     // at most k * VEC <= 512: fits
                    sh.cand[at] = cand(okey(f[j]), (int)gr.index(g, j));
                }
        }
        __syncthreads();
        const int n = sh.ncand, old = (int)min((long)k, have);
        // ranks within the union of the old best (all of them left of the chunk) and the new candidates
        for (int i = tid; i < n + old; i += NT) {
            const uint64_t c = i < n ? sh.cand[i] : sh.best[cur][i - n];
            const int r = rank_of(sh.cand, n, c) + rank_of(sh.best[cur], old, c);
            if (r < k) sh.best[cur ^ 1][r] = c;
        }
        have += n;
        cur ^= 1;
        __syncthreads();
    }
    __syncthreads();
    return cur;
}

// The workgroup's sum of its threads' sums; c as in soft_join
__device__ __forceinline__ Soft block_join(Soft t, float c, Soft* soft) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Soft u{__shfl_xor(t.ref, o, 64), __shfl_xor(t.s, o, 64), __shfl_xor(t.w, o, 64)};
        t = soft_join(t, u, c);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) soft[threadIdx.x >> 6] = t;
    __syncthreads();
    t = soft[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) t = soft_join(t, soft[i], c);
    return t;
}

// Rows without a reference in log2 units: relative to the largest logit itself
template <typename T>
__device__ Soft scan_huge(const Groups<T>& gr, float c, Soft* soft) {
    constexpr int VEC = Elem<T>::VEC;
    Soft a{-FLT_MAX, 0.f, 0.f};
    for (int g = threadIdx.x; g < gr.n; g += NT) {
        float f[VEC], m = a.ref;
        gr.load(g, f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = fmaxf(m, f[j]);
        soft_shift(a, (a.ref - m) * c);
        a.ref = m;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float d = (f[j] - m) * c, e = __builtin_amdgcn_exp2f(d);
            a.s += e;
            a.w += e * fmaxf(d, -150.f);
        }
    }
    return block_join(a, c, soft);
}

// Sums and the k best (sorted) of elements [v0, v1) of one row by one workgroup; k <= v1 - v0.
template <typename T>
__device__ Soft scan_row(const T* row, long v0, long v1, float c, int k, Shared& sh, int& best_set, bool& huge) {
    constexpr int VEC = Elem<T>::VEC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Groups<T> gr(row, v0, v1);
    Soft a{-REF_MAX, 0.f, 0.f};
    float b1 = -INFINITY, b2 = -INFINITY;                 // best value, best value outside the best pair of groups (g, g + NT)
    int bg = -1;
    const int n = gr.n;
    typename Groups<T>::Raw r0 = gr.raw(min(tid, n - 1)), r1 = gr.raw(min(tid + NT, n - 1));
    for (int g0 = 0; g0 < n; g0 += 2 * NT) {
        const int g = g0 + tid;
        float f[2 * VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) { f[j] = (float)r0[j]; f[VEC + j] = (float)r1[j]; }
        if (g0 + 2 * NT < n) {                             // (the next pair is in flight while this one is summed)
            r0 = gr.raw(min(g + 2 * NT, n - 1));
            r1 = gr.raw(min(g + 3 * NT, n - 1));
        }
        if (g0 + 2 * NT >= n) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                f[j] = g < n && gr.holds(g, j) ? f[j] : -INFINITY;
                f[VEC + j] = g + NT < n && gr.holds(g + NT, j) ? f[VEC + j] : -INFINITY;
            }
        }
        float vm = f[0];
#pragma unroll
        for (int j = 1; j < 2 * VEC; ++j) vm = fmaxf(vm, f[j]);
        b2 = fmaxf(b2, fminf(b1, vm));
        bg = g < n && (vm > b1 || bg < 0) ? g : bg;
        b1 = fmaxf(b1, vm);
        const float top = fminf(vm * c, REF_MAX);
        if (__any(top > a.ref + 16.f)) {
            const float ref = fmaxf(top, a.ref);
            soft_shift(a, a.ref - ref);
            a.ref = ref;
        }
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) {
            const float d = fmaf(f[j], c, -a.ref), e = __builtin_amdgcn_exp2f(d);
            a.s += e;
            a.w += e * fmaxf(d, -150.f);                  // 2^-150 = 0: e is 0 wherever the clamp acts, and 0 * -inf does not arise
        }
    }
    const uint32_t mine = bg < 0 ? 0u : okey(b1);
    // a bound of the k-th value from the maxima of 64, 128 or 256 sets of threads: the smallest of the k largest maxima
    const int sets = k <= 16 ? 64 : (k <= 32 ? 128 : 256);
    if (k) {
        uint32_t best = mine;
        if (sets <= 128) best = max(best, (uint32_t)__shfl_xor((int)best, 1, 64));
        if (sets == 64) best = max(best, (uint32_t)__shfl_xor((int)best, 2, 64));
        if (tid % (NT / sets) == 0) sh.key[tid / (NT / sets)] = best;
        if (tid == 0) { sh.ncand = 0; sh.nrescan = 0; sh.any = 0; sh.tau = 0xFFFFFFFFu; }
    }
    Soft t = block_join(a, 1.f, sh.soft);
    huge = !(t.s > 0.f && t.s < INFINITY);
    if (huge) t = scan_huge(gr, c, sh.soft);
    best_set = 0;
    if (k == 0) return t;

    if (!huge) {                                           // (no NaN, no +inf)
        if (tid < sets) {
            const uint4* keys = (const uint4*)sh.key;
            const uint32_t x = sh.key[tid];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < sets / 4; ++j) {
                const uint4 q = keys[j];
                above += (q.x > x) + (q.y > x) + (q.z > x) + (q.w > x);
            }
            if (above < k) atomicMin(&sh.tau, x);
        }
        __syncthreads();
        const uint32_t tau = sh.tau;                       // 0: fewer than k sets hold elements - every element is a candidate
        auto push = [&](int g) {                            // a group's elements that reach the bound
            if (g >= n) return;
            float f[VEC];
            gr.load(g, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (gr.holds(g, j) && okey(f[j]) >= tau) {
                    const int at = atomicAdd(&sh.ncand, 1);
                    if (at < CAP) sh.cand[at] = cand(okey(f[j]), (int)gr.index(g, j));
                }
        };
        if (bg >= 0 && mine >= tau) {
            const bool more = n > 2 * NT && okey(b2) >= tau;   // (with one pair a thread there is no value outside it)
            if (more && b2 == -INFINITY) {
                sh.any = 1;                                 // the bound itself is -inf: too few finite values
            } else if (more) {
                const int at = atomicAdd(&sh.nrescan, 1);
                if (at < RESCAN) sh.rescan[at] = tid;
            } else {
                push(bg);
                push(bg + NT);
            }
        }
        __syncthreads();
        const int nr = sh.nrescan;
        if (nr <= RESCAN && !sh.any) {
            for (int i = wave; i < nr; i += NW)
                for (int gg = sh.rescan[i] + lane * NT; gg < n; gg += 64 * NT) push(gg);
            __syncthreads();
            const int nc = sh.ncand;
            if (nc <= CAP) {
                for (int i = tid; i < nc; i += NT) {
                    const uint64_t c = sh.cand[i];
                    const int r = rank_of(sh.cand, nc, c);
                    if (r < k) sh.best[0][r] = c;
                }
                __syncthreads();
                return t;
            }
        }
    }
    best_set = select_ordered(gr, k, sh);
    return t;
}

__device__ __forceinline__ float key_value(uint32_t k) {
    return k == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k);
}

// log p of a value from the row's reference and log2 s (a masked value near the type's lowest has no log2 units in fp32's range: natural ones).  Of a token
// that decides its row the two cancel but for their roundings: not above 0 (NaN stays).
__device__ __forceinline__ float value_lp(float x, float ref, float logs, bool huge, float t) {
    const float lp = huge ? (x - ref) * t - LN2 * logs
                          : (fabsf(x) > 1e30f ? x * t - LN2 * (ref + logs) : LN2 * (fmaf(x, t * LOG2E, -ref) - logs));
    return lp > 0.f ? 0.f : lp;
}

// A row without any finite value has no distribution: log probabilities -inf, entropy 0.
template <typename T>
__device__ void finish_row(const LogpP& p, long r, Soft a, bool huge, const uint64_t* best) {
    const float logs = a.s > 0.f || a.s != a.s ? log2f(a.s) : -INFINITY;
    const bool none = logs == -INFINITY;
    if (threadIdx.x == 0) {
        float H = none ? 0.f : LN2 * (logs - a.w / a.s);
        if (H < 0.f) H = 0.f;                                  // (the same rounding of a decided row)
        const int64_t id = p.ids ? p.ids[r] : -1;
        float lp = 0.f;
        if (id >= 0 && id < p.V) lp = none ? -INFINITY : value_lp((float)((const T*)p.x)[r * p.ld + id], a.ref, logs, huge, p.t);
        p.logprob[r] = lp;
        p.entropy[r] = H;
        p.lse[r] = none ? -INFINITY : (huge ? a.ref * p.t + LN2 * logs : LN2 * (a.ref + logs));
        *(float4*)(p.stats + 4 * r) = make_float4(a.ref, logs, H, huge ? 1.f : 0.f);
    }
    for (int j = threadIdx.x; j < p.k; j += NT) {
        p.top_ids[r * p.k + j] = cand_idx(best[j]);
        p.top_lp[r * p.k + j] = none ? -INFINITY : value_lp(key_value(cand_key(best[j])), a.ref, logs, huge, p.t);
    }
}

template <typename T>
__global__ __launch_bounds__(NT) void k_token_logprobs(LogpP p) {
    __shared__ Shared sh;
    const long r = blockIdx.x;
    int set;
    bool huge;
    const Soft a = scan_row((const T*)p.x + r * p.ld, 0, p.V, p.t * LOG2E, p.k, sh, set, huge);
    finish_row<T>(p, r, a, huge, sh.best[set]);
}

// Few rows: `splits` workgroups a row, each with its part's sums and its k best; k_token_logprobs_join puts them together.
template <typename T>
__global__ __launch_bounds__(NT) void k_token_logprobs_part(LogpP p) {
    __shared__ Shared sh;
    const long r = blockIdx.x / p.splits, i = blockIdx.x % p.splits;
    const long v0 = p.V * i / p.splits, v1 = p.V * (i + 1) / p.splits;
    int set;
    bool huge;
    const Soft a = scan_row((const T*)p.x + r * p.ld, v0, v1, p.t * LOG2E, p.k, sh, set, huge);
    float* o = p.part + (long)blockIdx.x * (4 + 2 * p.k);
    if (threadIdx.x == 0) { o[0] = a.ref; o[1] = a.s; o[2] = a.w; o[3] = huge ? 1.f : 0.f; }
    for (int j = threadIdx.x; j < p.k; j += NT) {
        o[4 + j] = __uint_as_float(cand_key(sh.best[set][j]));
        o[4 + p.k + j] = __int_as_float(cand_idx(sh.best[set][j]));
    }
}

template <typename T>
__global__ __launch_bounds__(NT) void k_token_logprobs_join(LogpP p) {
    __shared__ __attribute__((aligned(16))) uint64_t list[SMAX * KMAX], best[KMAX];
    __shared__ uint64_t bound;
    __shared__ int n;
    __shared__ Soft soft[NW];
    const long r = blockIdx.x;
    const float *q = p.part + r * p.splits * (4 + 2 * p.k), c = p.t * LOG2E;
    // Parts summed relative to a logit (sum 0: nothing finite in them) do not mix with the others; far below them (a part that is masked with
    // the type's lowest value) they add nothing, else the row is summed again here.  A lane a part, every wave the same.
    const int i = threadIdx.x & 63;
    const float* o = q + (i < p.splits ? i : 0) * (4 + 2 * p.k);
    const float o0 = o[0], o1 = o[1], o2 = o[2], o3 = o[3];
    const bool in = i < p.splits, odd = in && o3 != 0.f && o1 != 0.f, low = odd && o1 < INFINITY && o0 < 0.f;
    Soft a = in && o3 == 0.f ? Soft{o0, o1, o2} : Soft{-REF_MAX, 0.f, 0.f};
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) {
        a = soft_join(a, Soft{__shfl_xor(a.ref, x, 64), __shfl_xor(a.s, x, 64), __shfl_xor(a.w, x, 64)}, 1.f);
    }
    const bool huge = __any(odd && !low) || (__any(low) && a.ref < -0.5f * REF_MAX);
    if (huge) a = scan_huge(Groups<T>((const T*)p.x + r * p.ld, 0, p.V), c, soft);
    if (p.k == 0) return finish_row<T>(p, r, a, huge, best);
    // the k-th best of the first few of every part (at least 2 k in all) bounds the row's k-th from below: few candidates are left to rank
    auto entry = [&](int part, int j) {
        const float* e = q + part * (4 + 2 * p.k) + 4;
        return cand(__float_as_uint(e[j]), __float_as_int(e[p.k + j]));
    };
    const int few = min(p.k, (2 * p.k + p.splits - 1) / p.splits + 1), nf = p.splits * few;
    for (int j = threadIdx.x; j < nf; j += NT) list[j] = entry(j / few, j % few);
    if (threadIdx.x == 0) n = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < nf; j += NT)
        if (rank_of(list, nf, list[j]) == p.k - 1) bound = list[j];
    __syncthreads();
    const uint64_t tau = bound;
    for (int j = threadIdx.x; j < p.splits * p.k; j += NT) {
        const uint64_t c = entry(j / p.k, j % p.k);
        if (c >= tau) list[atomicAdd(&n, 1)] = c;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += NT) {
        const int rk = rank_of(list, n, list[j]);
        if (rk < p.k) best[rk] = list[j];
    }
    __syncthreads();
    finish_row<T>(p, r, a, huge, best);
}

// One pass: reads a part of a row, writes its gradient.  The tokens that carry gradients of their own (the given one, the alternatives) are read
// before the pass and written after it by the part that holds them, each once with all it gets; so dx may be x itself.
template <typename T>
__global__ __launch_bounds__(NT) void k_token_logprobs_bwd(LogpP p) {
    constexpr int VEC = Elem<T>::VEC;
    __shared__ long sid[KMAX + 1];
    __shared__ float sg[KMAX + 1];
    __shared__ float gsum;
    const int tid = threadIdx.x;
    const long r = blockIdx.x / p.splits, i = blockIdx.x % p.splits;
    const long v0 = p.V * i / p.splits, v1 = p.V * (i + 1) / p.splits;
    const T* row = (const T*)p.x + r * p.ld;
    T* out = (T*)p.dx + r * p.ldd;
    const float4 st = *(const float4*)(p.stats + 4 * r);
    const float c = p.t * LOG2E, off = st.w != 0.f ? st.x : 0.f, ref = st.w != 0.f ? 0.f : st.x, logs = st.y, H = st.z, gH = p.dent ? p.dent[r] : 0.f;
    if (tid <= p.k) {
        const long id = tid == 0 ? (p.ids ? (long)p.ids[r] : -1) : (long)p.tids[r * p.k + tid - 1];
        const bool in = id >= 0 && id < p.V;
        const float* src = tid == 0 ? p.dlp : p.dtop;
        sid[tid] = in ? id : -1;
        sg[tid] = in && src ? (tid == 0 ? src[r] : src[r * p.k + tid - 1]) : 0.f;
    }
    __syncthreads();
    if (tid == 0) {
        float s = 0.f;
        for (int j = 0; j <= p.k; ++j) s += sg[j];
        gsum = s;
    }
    // this thread's special token, if it is the first of its index and lies in this part
    long mine = -1;
    float xm = 0.f, gm = 0.f;
    if (tid <= p.k && sid[tid] >= v0 && sid[tid] < v1) {
        mine = sid[tid];
        for (int j = 0; j <= p.k; ++j)
            if (sid[j] == mine) {
                if (j < tid) mine = -1;
                gm += sg[j];
                if (mine < 0) break;
            }
        if (mine >= 0) xm = (float)row[mine];
    }
    __syncthreads();
    const float A = gsum;
    const bool none = logs == -INFINITY;
    auto grad = [&](float x, float g) {
        const float l2 = fmaf(x - off, c, -ref) - logs, pr = __builtin_amdgcn_exp2f(l2);
        return none ? 0.f : p.t * (g - pr * (A + gH * (LN2 * fmaxf(l2, -300.f) + H)));      // 2^-300 = 0 in fp32: no 0 * inf
    };
    const Groups<T> gr(row, v0, v1);
    for (int g = tid; g < gr.n; g += NT) {
        const typename Groups<T>::Raw raw = gr.raw(g);
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = grad((float)raw[j], 0.f);
        T* const o = (T*)((char*)(out + v0) + (unsigned)gr.at(g) * (unsigned)sizeof(T));
        if (gr.whole(g)) {
            st_elems<T, VEC>(o, f);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (gr.holds(g, j)) o[j] = (T)f[j];
        }
    }
    __syncthreads();                                        // (orders this workgroup's stores: the special tokens are written last)
    if (mine >= 0) out[mine] = (T)grad(xm, gm);
}

int check_common(const dua_token_logprobs_args* a, const char* who) {
    DUA_REQUIRE(a, "%s: null arguments", who);
    DUA_REQUIRE(dua_dtype_ok(a->dtype), "%s: dtype must be fp32, bf16 or fp16", who);
    DUA_REQUIRE(a->rows >= 0 && a->rows < (1L << 24) && a->V >= 1 && a->V < (1L << 30) && a->ld >= a->V, "%s: rows in [0, 2^24), V in [1, 2^30), ld >= V", who);
    DUA_REQUIRE(a->k >= 0 && a->k <= KMAX && a->k <= a->V, "%s: k must be in [0, %d] and at most V", who, KMAX);
    DUA_REQUIRE(a->inv_temperature > 0.f && a->inv_temperature * LOG2E < INFINITY, "%s: inv_temperature must be positive and finite, also times log2 e", who);
    DUA_REQUIRE(a->rows == 0 || (a->logits && a->stats && ((uintptr_t)a->stats & 15) == 0), "%s: null logits / stats, or stats not 16-byte aligned", who);
    return DUA_OK;
}

// Parts of a row: enough workgroups for the chip, at least 4096 elements (more than k) each.  Rows from 192 KB on are dealt up to 512 rows, where a workgroup a
// row still leaves CUs waiting for the last ones: 256 / 384 / 512 rows of 128000 bf16 27 / 38 / 39 us whole, 21 / 29 / 33 in 4 / 3 / 2 parts, of 65536 fp32
// (384) 29 and 26; 600 rows of 128000 fp32 60 and 61.  Shorter rows only below 256 (256 / 512 rows of 65536 bf16 18 / 18 us whole, 20 / 21 in parts).
int plan_splits(long rows, long V, int dtype) {
    const bool big = V * (long)dua_dtype_size(dtype) >= 192 * 1024;
    if (rows == 0 || rows > (big ? 512 : 255)) return 1;
    const long want = rows < 256 ? 512 : 1024;
    long s = (want + rows - 1) / rows, most = V / 4096;
    if (s > most) s = most;
    if (s > SMAX) s = SMAX;
    return s < 1 ? 1 : (int)s;
}
LogpP pack(const dua_token_logprobs_args* a) {
    LogpP p{};
    p.x = a->logits; p.ids = a->ids; p.logprob = a->logprob; p.entropy = a->entropy; p.lse = a->lse; p.stats = a->stats;
    p.top_ids = a->top_ids; p.top_lp = a->top_logprobs; p.rows = a->rows; p.ld = a->ld; p.V = a->V; p.k = a->k; p.t = a->inv_temperature;
    return p;
}

}  // namespace

extern "C" size_t dua_token_logprobs_workspace_bytes(const dua_token_logprobs_args* a) {
    if (!a || a->rows < 0 || a->V < 1 || a->k < 0) return 0;
    const int s = plan_splits(a->rows, a->V, a->dtype);
    return s > 1 ? (size_t)a->rows * s * (4 + 2 * a->k) * sizeof(float) : 0;
}

extern "C" int dua_token_logprobs(const dua_token_logprobs_args* a, void* stream) {
    if (int rc = check_common(a, "dua_token_logprobs")) return rc;
    if (a->rows == 0) return DUA_OK;
    DUA_REQUIRE(a->logprob && a->entropy && a->lse && (a->k == 0 || (a->top_ids && a->top_logprobs)), "dua_token_logprobs: null output");
    LogpP p = pack(a);
    p.splits = plan_splits(a->rows, a->V, a->dtype);
    p.part = (float*)a->workspace;
    DUA_REQUIRE(p.splits == 1 || (a->workspace && a->workspace_bytes >= dua_token_logprobs_workspace_bytes(a)),
                "dua_token_logprobs: workspace smaller than dua_token_logprobs_workspace_bytes");
    hipStream_t st = as_stream(stream);
#define GO(T)                                                                                                              \
    if (p.splits == 1) hipLaunchKernelGGL(k_token_logprobs<T>, (unsigned)p.rows, NT, 0, st, p);                             \
    else {                                                                                                                  \
        hipLaunchKernelGGL(k_token_logprobs_part<T>, (unsigned)(p.rows * p.splits), NT, 0, st, p);                          \
        hipLaunchKernelGGL(k_token_logprobs_join<T>, (unsigned)p.rows, NT, 0, st, p);                                       \
    }
    if (a->dtype == DUA_DTYPE_F32) { GO(float) } else if (a->dtype == DUA_DTYPE_BF16) { GO(bf16_t) } else { GO(f16_t) }
#undef GO
    return dua_check_launch("dua_token_logprobs");
}

extern "C" int dua_token_logprobs_bwd(const dua_token_logprobs_args* a, void* stream) {
    if (int rc = check_common(a, "dua_token_logprobs_bwd")) return rc;
    if (a->rows == 0) return DUA_OK;
    DUA_REQUIRE(a->dlogits && a->ldd >= a->V && (!a->dlogprob || a->ids) && (a->k == 0 || (a->dtop && a->top_ids)),
                "dua_token_logprobs_bwd: null operand (k > 0 needs dtop and top_ids, dlogprob needs ids)");
    DUA_REQUIRE(a->dlogits != a->logits || a->ldd == a->ld, "dua_token_logprobs_bwd: in place needs one row stride");
    LogpP p = pack(a);
    p.dlp = a->dlogprob; p.dent = a->dentropy; p.dtop = a->dtop; p.tids = a->top_ids; p.dx = a->dlogits; p.ldd = a->ldd;
    long s = (4096 + a->rows - 1) / a->rows;                 // parts of at least 4096 elements, about 4096 workgroups
    if (s > a->V / 4096) s = a->V / 4096;
    p.splits = s < 1 ? 1 : (s > 1024 ? 1024 : (int)s);
    hipStream_t st = as_stream(stream);
    const unsigned grid = (unsigned)(p.rows * p.splits);
    if (a->dtype == DUA_DTYPE_F32) hipLaunchKernelGGL(k_token_logprobs_bwd<float>, grid, NT, 0, st, p);
    else if (a->dtype == DUA_DTYPE_BF16) hipLaunchKernelGGL(k_token_logprobs_bwd<bf16_t>, grid, NT, 0, st, p);
    else hipLaunchKernelGGL(k_token_logprobs_bwd<f16_t>, grid, NT, 0, st, p);
    return dua_check_launch("dua_token_logprobs_bwd");
}
