/* Expert routing (le_moe_route, le_moe_sort, le_moe_permute, le_moe_combine and their gradients, include/le_qmm.h). */
#include <hip/hip_runtime.h>

#include "le_f32_types.h"
#include "le_route_args.h"

static __device__ __forceinline__ int as_int(float v) { return __builtin_bit_cast(int, v); }
static __device__ __forceinline__ float as_float(int v) { return __builtin_bit_cast(float, v); }

/* The value of the lane D away (1, 2), or of the mirrored lane of the 8 (4) or 16 (8) where all lanes of a 4 or 8 hold the same value by
 * then, or of the row or half 16 or 32 away: the steps of a butterfly over up to 64 lanes without LDS. */
template <int D> static __device__ __forceinline__ int across(int v) {
    if constexpr (D == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xf, 0xf, true);
    else if constexpr (D == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xf, 0xf, true);
    else if constexpr (D == 4) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);
    else if constexpr (D == 8) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true);
    else if constexpr (D == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
/* Sum over groups of L lanes, in every lane of them. */
template <int L, int D = 1> static __device__ __forceinline__ float group_sum(float v) {
    if constexpr (D < L) {
        v += as_float(across<D>(as_int(v)));
        return group_sum<L, 2 * D>(v);
    } else {
        return v;
    }
}
/* Largest and smallest over groups of L lanes, in every lane of them (one instruction a step up to 16 lanes). */
template <int L, int D = 1> static __device__ __forceinline__ int group_max(int v) {
    if constexpr (D < L) return group_max<L, 2 * D>(max(v, across<D>(v)));
    else return v;
}
template <int L, int D = 1> static __device__ __forceinline__ int group_min(int v) {
    if constexpr (D < L) return group_min<L, 2 * D>(min(v, across<D>(v)));
    else return v;
}

/* ---- router ----
 * Top-k by groups of L lanes, a token each, lane l holding experts l, l + L, ... (V of them) as integers that order as the logits do (-0
 * as 0; NaN and -infinity below all). k rounds of a maximum, then the lowest expert that has it. Lane s < k keeps selection s. Reads
 * the logits once; bound by the rounds' instructions for many tokens (16384 of 128 experts, 8 of them: L = 16, whose wave serves
 * four tokens with a round), by their latency for few (L = 64, ballots instead of the second reduction). */
constexpr int kNone = (int)0x80000000;
static __device__ __forceinline__ int order_key(float x) {
    const int b = as_int(x + 0.f);
    return x > -INFINITY ? b ^ ((b >> 31) & 0x7FFFFFFF) : kNone;
}
static __device__ __forceinline__ float key_value(int k) { return as_float(k ^ ((k >> 31) & 0x7FFFFFFF)); }
template <int TY, int L, int V> __device__ __forceinline__ void route_body(const RouteArgs &a) {
    const int l = threadIdx.x & (L - 1);
    for (long long t0 = (long long)blockIdx.x * (256 / L); t0 < a.n_tok; t0 += (long long)gridDim.x * (256 / L)) {
        const long long t = t0 + threadIdx.x / L;
        const bool there = t < a.n_tok; /* lanes of a token behind the last go along, and write nothing */
        const typename XT<TY>::raw *lg = (const typename XT<TY>::raw *)a.logits + (there ? t : a.n_tok - 1) * a.n_exp;
        int v[V];
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = l + L * j < a.n_exp ? order_key(XT<TY>::up(lg[l + L * j])) : kNone;
        int my_e = -1, my_v = kNone;
        for (int r = 0; r < a.k; r++) {
            int mx = v[0];
#pragma unroll
            for (int j = 1; j < V; j++) mx = max(mx, v[j]);
            mx = group_max<L>(mx);
            int e = 0x7FFFFFFF;
            if constexpr (L == 64) {
#pragma unroll
                for (int j = V - 1; j >= 0; j--) {
                    const unsigned long long b = __ballot(v[j] == mx);
                    e = b ? 64 * j + __ffsll((long long)b) - 1 : e;
                }
            } else {
#pragma unroll
                for (int j = V - 1; j >= 0; j--) e = v[j] == mx ? l + L * j : e;
                e = group_min<L>(e);
            }
#pragma unroll
            for (int j = 0; j < V; j++) v[j] = e == l + L * j ? kNone : v[j];
            if (l == r && mx != kNone) my_e = e, my_v = mx;
        }
        const float top = key_value(__builtin_amdgcn_ds_bpermute((threadIdx.x & 63 & ~(L - 1)) * 4, my_v));
        const float ex = my_e >= 0 ? expf(key_value(my_v) - top) : 0.f;
        const float tot = group_sum<L>(ex);
        if (there && l < a.k) {
            a.idx[t * a.k + l] = my_e;
            a.w[t * a.k + l] = my_e >= 0 ? ex / tot : 0.f;
        }
    }
}

/* Gradient: one wave a token, its selections in lanes s < k; each value is then added where its expert is: no scatter, every logit written
 * once. */
template <int TY> __device__ __forceinline__ void route_bwd_body(const RouteBwdArgs &a) {
    const int l = threadIdx.x & 63;
    for (long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); t < a.n_tok; t += (long long)gridDim.x * 4) {
        int e = -1;
        float w = 0.f, dw = 0.f;
        if (l < a.k) {
            e = a.idx[t * a.k + l];
            w = a.w[t * a.k + l], dw = a.dw[t * a.k + l];
            if (e < 0 || e >= a.n_exp) e = -1, w = 0.f, dw = 0.f;
        }
        const float g = w * (dw - group_sum<16>(w * dw)); /* the selections lie in the first 16 lanes */
        typename XT<TY>::raw *d = (typename XT<TY>::raw *)a.dlogits + t * a.n_exp;
        for (int e0 = 0; e0 < a.n_exp; e0 += 256) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < a.k; s++) {
                const int es = __builtin_amdgcn_readlane(e, s) - e0 - l;
                const float gs = as_float(__builtin_amdgcn_readlane(as_int(g), s));
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] += es == 64 * j ? gs : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (e0 + l + 64 * j < a.n_exp) d[e0 + l + 64 * j] = XT<TY>::down(v[j]);
        }
    }
}

/* ---- sort ----
 * A stable counting sort. A block takes a run of the pairs, each of its waves 64 J of them in a row (lane, then step), so that pair
 * order is (block, wave, step, lane) order. Counts per wave and expert in LDS give every wave its first place for every expert; a
 * pair's place is that, the wave's pairs of the expert in earlier steps, and those in lower lanes of the step, which ballots
 * over the bits of the expert's number find. One block does all of up to 4096 pairs; more run as two launches, the first of which
 * writes every block's counts to the workspace (at most 256 blocks, so that each can add up what all have). */
static __device__ __forceinline__ int expert_of(const SortArgs &a, long long p) {
    if (p >= a.np) return -2; /* no pair */
    const int e = a.idx[p];
    return e >= 0 && e < a.n_exp ? e : -1;
}
extern "C" __global__ void __launch_bounds__(1024) le_rt_count(SortArgs a) {
    extern __shared__ int hist[];
    const long long p0 = ((long long)blockIdx.x * a.waves + (threadIdx.x >> 6)) * 64 * a.steps + (threadIdx.x & 63);
    const int first = expert_of(a, p0); /* on its way while LDS is cleared */
    for (int e = threadIdx.x; e < a.n_exp; e += 1024) hist[e] = 0;
    __syncthreads();
    if (first >= 0) atomicAdd(&hist[first], 1);
#pragma unroll 4
    for (int j = 1; j < a.steps; j++) {
        const int e = expert_of(a, p0 + 64ll * j);
        if (e >= 0) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.n_exp; e += 1024) a.ws[blockIdx.x * a.n_exp + e] = hist[e];
}
extern "C" __global__ void __launch_bounds__(1024) le_rt_sort(SortArgs a) {
    extern __shared__ int hist[]; /* [wave][expert], then [expert] all pairs, [expert] those of earlier blocks, [16] */
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nt = 64 * a.waves, ne = a.n_exp;
    int *all = hist + a.waves * ne, *before = all + ne, *wsum = before + ne;
    const long long p0 = ((long long)blockIdx.x * a.waves + wave) * 64 * a.steps + lane;
    const int first = expert_of(a, p0); /* on its way while LDS is cleared; the other blocks' counts, too */
    const int c0 = a.blocks > 1 && (int)threadIdx.x < a.blocks * ne ? a.ws[threadIdx.x] : 0;
    for (int i = threadIdx.x; i < a.waves * ne + 2 * ne; i += nt) hist[i] = 0;
    __syncthreads();
    if (first >= 0) atomicAdd(&hist[wave * ne + first], 1);
#pragma unroll 4
    for (int j = 1; j < a.steps; j++) {
        const int e = expert_of(a, p0 + 64ll * j);
        if (e >= 0) atomicAdd(&hist[wave * ne + e], 1);
    }
    if (a.blocks > 1) { /* integer sums: their order does not matter */
#pragma unroll 4
        for (int i = threadIdx.x; i < a.blocks * ne; i += nt) {
            const int c = i == (int)threadIdx.x ? c0 : a.ws[i], e = i % ne;
            if (c) {
                atomicAdd(&all[e], c);
                if (i / ne < (int)blockIdx.x) atomicAdd(&before[e], c);
            }
        }
    }
    __syncthreads();
    /* offsets: an exclusive scan over the experts, one a thread and round */
    int carry = 0;
    for (int e0 = 0; e0 < ne; e0 += nt) {
        const int e = e0 + threadIdx.x, busy = min(a.waves, (ne - e0 + 63) >> 6); /* waves that have experts */
        int c[16], own = 0; /* the waves' counts, all read before the first is replaced */
#pragma unroll
        for (int w = 0; w < 16; w++) c[w] = e < ne && w < a.waves ? hist[w * ne + e] : 0;
        if (a.blocks > 1) {
            own = e < ne ? all[e] : 0;
        } else {
#pragma unroll
            for (int w = 0; w < 16; w++) own += c[w];
        }
        int incl = own;
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(incl, d);
            if (lane >= d) incl += y;
        }
        __syncthreads();
        if (lane == 63) wsum[wave] = incl;
        __syncthreads();
        int at = carry + incl - own;
        for (int w = 0; w < busy; w++) {
            if (w < wave) at += wsum[w];
            carry += wsum[w];
        }
        if (e < ne) {
            if (blockIdx.x == 0) a.off[e] = at;
            at += before[e];
#pragma unroll
            for (int w = 0; w < 16; w++) { /* counts to places */
                if (w < a.waves) hist[w * ne + e] = at;
                at += c[w];
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.off[ne] = carry;
    __syncthreads();
    const int bits = 32 - __clz(ne - 1);
    const unsigned long long lower = (1ull << lane) - 1ull;
    for (int j = 0; j < a.steps; j++) {
        const long long p = p0 + 64ll * j;
        const int e = j == 0 ? first : expert_of(a, p);
        unsigned long long same = __ballot(e >= 0);
        for (int b = 0; b < bits; b++) {
            const unsigned long long m = __ballot(e >> b & 1);
            same &= e >> b & 1 ? m : ~m;
        }
        if (e >= 0) {
            int *next = &hist[wave * ne + e];
            const int q = *next + __popcll(same & lower);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if ((same & ~lower) >> lane == 1ull) *next = q + 1; /* the step's last of this expert */
            if (a.in_idx) a.in_idx[q] = (int)(p / a.k);
            if (a.out_idx) a.out_idx[q] = (int)p;
            if (a.pos) a.pos[p] = q;
        } else if (e == -1 && a.pos) {
            a.pos[p] = -1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

/* ---- rows between token order and expert order ----
 * Bound by memory: every row is read once and written once (4096 tokens of 8 pairs by 2048 bf16: copied 136 MB in 30.5 us, summed 26.6,
 * gradient of the sum 285 MB in 58; a copy of 256 MB runs at 5.4 TB/s). Stores stay in the caches for whoever reads the rows next
 * (non-temporal, the copy alone takes 26 us, but with a sum behind it 60 against 55). A token is taken by a group of L lanes (16 to 256), 16 bytes a lane and step (rows
 * need not be aligned: the unaligned forms of the loads and stores), the last values of a row one by one. The places and weights of a
 * token's pairs are loaded by 16 lanes at once. */
typedef unsigned v4 __attribute__((ext_vector_type(4)));
typedef unsigned v4u __attribute__((ext_vector_type(4), aligned(2))); /* at any value's address */
template <int TY> struct Oct { /* 16 bytes of values */
    static constexpr int N = TY == 0 ? 4 : 8;
    using raw = typename XT<TY>::raw;
    raw v[N];
    /* n values are there. NT: past the caches' replacement order, for rows that are read once and are more than the L2s hold: */
    template <bool NT = false> __device__ __forceinline__ void load(const raw *p, int n) {
        if (n >= N) {
            const v4 w = NT ? __builtin_nontemporal_load((const v4u *)p) : *(const v4u *)p;
            __builtin_memcpy(v, &w, 16);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = i < n ? p[i] : (raw)0;
        }
    }
    __device__ __forceinline__ void store(raw *p, int n) const {
        if (n >= N) {
            v4 w;
            __builtin_memcpy(&w, v, 16);
            *(v4u *)p = w;
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < n) p[i] = v[i];
        }
    }
};
/* The pairs of a token: lane i of each 16 holds pair i's row (-1: none) and weight. */
template <int L> struct Pairs {
    int row;
    float w;
    __device__ __forceinline__ void load(const RowsArgs &a, long long t) {
        const int i = threadIdx.x & 15;
        row = -1;
        w = 1.f;
        if (t < a.n_tok && i < a.k) {
            const long long p = t * a.k + i;
            row = a.pos ? a.pos[p] : (int)p;
            if (row < 0 || row >= a.n_row) row = -1;
            if (a.w) w = a.w[p];
        }
    }
    template <class T> static __device__ __forceinline__ T of(T v, int s) {
        const int b = __builtin_bit_cast(int, v);
        if constexpr (L >= 64) return __builtin_bit_cast(T, __builtin_amdgcn_readlane(b, s)); /* one token a wave */
        else return __builtin_bit_cast(T, __builtin_amdgcn_ds_bpermute((((int)threadIdx.x & 48) + s) * 4, b));
    }
};
/* Group of L lanes, and the tokens it goes over. */
#define GROUP_TOKENS(L) \
    const int l = threadIdx.x & (L - 1); \
    for (long long t0 = (long long)blockIdx.x * (256 / L), t; t = t0 + threadIdx.x / L, t0 < a.n_tok; t0 += (long long)gridDim.x * (256 / L))

/* e[row of pair] = x[t]; blockIdx.y: 16 L bytes of the columns. */
template <int TY, int L> __device__ __forceinline__ void permute_body(const RowsArgs &a) {
    using O = Oct<TY>;
    GROUP_TOKENS(L) {
        const int c = ((int)blockIdx.y * L + l) * O::N, n = t < a.n_tok ? a.cols - c : 0;
        Pairs<L> pr;
        pr.load(a, t);
        O o;
        if (n > 0) o.load((const typename O::raw *)a.src + t * a.ldt + c, n);
        for (int s = 0; s < a.k; s++) {
            const int r = Pairs<L>::of(pr.row, s);
            if (r >= 0 && n > 0) o.store((typename O::raw *)a.dst + r * a.lde + c, n);
        }
    }
}

/* out[t] = sum of weight * e[row], in selection order; the rows' loads eight at a time. */
template <int TY, int L, bool NT> __device__ __forceinline__ void combine_body(const RowsArgs &a) {
    using O = Oct<TY>;
    GROUP_TOKENS(L) {
        const int c = ((int)blockIdx.y * L + l) * O::N, n = t < a.n_tok ? a.cols - c : 0;
        Pairs<L> pr;
        pr.load(a, t);
        float sum[O::N] = {};
        for (int s0 = 0; s0 < a.k; s0 += 8) {
            O o[8];
            int r[8];
#pragma unroll
            for (int s = 0; s < 8; s++) {
                r[s] = Pairs<L>::of(pr.row, s0 + s); /* -1 from k on */
                if (r[s] >= 0 && n > 0) o[s].template load<NT>((const typename O::raw *)a.src + r[s] * a.lde + c, n);
            }
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const float w = Pairs<L>::of(pr.w, s0 + s);
#pragma unroll
                for (int i = 0; i < O::N; i++) sum[i] = r[s] >= 0 ? __builtin_fmaf(w, XT<TY>::up(o[s].v[i]), sum[i]) : sum[i];
            }
        }
        if (n > 0) {
            O o;
#pragma unroll
            for (int i = 0; i < O::N; i++) o.v[i] = XT<TY>::down(sum[i]);
            o.store((typename O::raw *)a.dst + t * a.ldt + c, n);
        }
    }
}

/* de[row] = weight * dout[t], dw = dout[t] . e[row]: a lane's products over its columns, then the lanes', then the waves'. */
template <int TY, int L, bool NT> __device__ __forceinline__ void combine_bwd_body(const RowsArgs &a) {
    using O = Oct<TY>;
    __shared__ float part[4][8];
    GROUP_TOKENS(L) {
        Pairs<L> pr;
        pr.load(a, t);
        for (int s0 = 0; s0 < a.k; s0 += 8) {
            int r[8];
            float w[8], dot[8] = {};
#pragma unroll
            for (int s = 0; s < 8; s++) {
                r[s] = Pairs<L>::of(pr.row, s0 + s);
                w[s] = Pairs<L>::of(pr.w, s0 + s);
            }
            for (int c = l * O::N; c < (t < a.n_tok ? a.cols : 0); c += L * O::N) {
                const int n = a.cols - c;
                O d, e[8];
                d.load((const typename O::raw *)a.src + t * a.ldt + c, n);
                if (a.dw) {
#pragma unroll
                    for (int s = 0; s < 8; s++)
                        if (r[s] >= 0) e[s].template load<NT>((const typename O::raw *)a.e + r[s] * a.lde + c, n);
                }
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    if (r[s] < 0) continue;
                    if (a.dw) {
#pragma unroll
                        for (int i = 0; i < O::N; i++) dot[s] = __builtin_fmaf(XT<TY>::up(d.v[i]), XT<TY>::up(e[s].v[i]), dot[s]);
                    }
                    if (a.dst) {
                        O o;
#pragma unroll
                        for (int i = 0; i < O::N; i++) o.v[i] = XT<TY>::down(w[s] * XT<TY>::up(d.v[i]));
                        o.store((typename O::raw *)a.dst + r[s] * a.lde + c, n);
                    }
                }
            }
            if (!a.dw) continue;
#pragma unroll
            for (int s = 0; s < 8; s++) dot[s] = group_sum<(L < 64 ? L : 64)>(dot[s]);
            if constexpr (L > 64) {
                __syncthreads(); /* every thread of the block is here as often: L > 64 gives a block whole tokens, and k is one */
                if ((threadIdx.x & 63) == 0)
#pragma unroll
                    for (int s = 0; s < 8; s++) part[threadIdx.x >> 6][s] = dot[s];
                __syncthreads();
                const int w0 = threadIdx.x / L * (L / 64);
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    dot[s] = part[w0][s];
                    for (int i = 1; i < L / 64; i++) dot[s] += part[w0 + i][s];
                }
            }
            if (t < a.n_tok && l < 8 && s0 + l < a.k) {
                float v = 0.f;
#pragma unroll
                for (int s = 0; s < 8; s++) v = l == s && r[s] >= 0 ? dot[s] : v;
                a.dw[t * a.k + s0 + l] = v;
            }
        }
    }
}

#define LE_RT_ROUTE(TY, L, V) \
    extern "C" __global__ void __launch_bounds__(256) le_rt_route_##TY##_l##L##_v##V(RouteArgs a) { route_body<TY, L, V>(a); }
#define LE_RT_ROWS(TY, L) \
    extern "C" __global__ void __launch_bounds__(256) le_rt_permute_##TY##_l##L(RowsArgs a) { permute_body<TY, L>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_##TY##_l##L(RowsArgs a) { combine_body<TY, L, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_##TY##_l##L##_nt(RowsArgs a) { combine_body<TY, L, true>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_bwd_##TY##_l##L(RowsArgs a) { combine_bwd_body<TY, L, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) le_rt_combine_bwd_##TY##_l##L##_nt(RowsArgs a) { combine_bwd_body<TY, L, true>(a); }
#define LE_RT(TY) \
    LE_RT_ROUTE(TY, 16, 2) LE_RT_ROUTE(TY, 16, 4) LE_RT_ROUTE(TY, 16, 8) LE_RT_ROUTE(TY, 32, 8) \
    LE_RT_ROUTE(TY, 64, 1) LE_RT_ROUTE(TY, 64, 2) LE_RT_ROUTE(TY, 64, 4) LE_RT_ROUTE(TY, 64, 8) LE_RT_ROUTE(TY, 64, 16) \
    extern "C" __global__ void __launch_bounds__(256) le_rt_route_bwd_##TY(RouteBwdArgs a) { route_bwd_body<TY>(a); } \
    LE_RT_ROWS(TY, 16) LE_RT_ROWS(TY, 64) LE_RT_ROWS(TY, 256)
LE_RT(0) LE_RT(1) LE_RT(30)
