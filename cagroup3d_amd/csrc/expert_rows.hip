// expert_rows.hip -- rows sorted by expert and back (gfx950): the plan of a routing (a stable counting sort of the (token, slot)
// pairs by their expert), the gather of the tokens' rows into that order, the weighted combination back to tokens, and the
// gradients of both.
//
//   p = t * k + s;  e(p) = experts[t, s];  a pair whose id is outside [0, E) has no row
//   row of p   = #{ q : e(q) < e(p) } + #{ q < p : e(q) = e(p) }             (experts ascending, pairs ascending inside one)
//   gather       r[row(t, s)] = x[t]                    its gradient   dx[t] = sum_s dr[row(t, s)]
//   combine      o[t] = sum_s w[t, s] y[row(t, s)]      its gradient   dy[row(t, s)] = w[t, s] do[t],  dw[t, s] = <do[t], y[row(t, s)]>
//
// All four passes run token by token: a token's own row is read (written) once for its k slots, the rows in expert order are
// whole lines at arbitrary places, and no sum needs an atomic -- every result is the same from run to run.  The T * k - offsets[E]
// rows behind the last are given to the pairs without a row (pos = ~row, negative), so that the pass that writes rows clears them
// too.  Sums are held in fp32 in slot order and rounded once.
#include "cg3d_common.h"

#define EX_MAX_EXPERTS 1024

// ---------------------------------------------------------------- element types
struct ex_bf16 {
    uint16_t v;
    static __device__ __forceinline__ float to(ex_bf16 a) { return __uint_as_float((uint32_t)a.v << 16); }
    static __device__ __forceinline__ ex_bf16 from(float f) { ex_bf16 r; r.v = __builtin_bit_cast(uint16_t, (__bf16)f); return r; }
};
struct ex_f16 {
    uint16_t v;
    static __device__ __forceinline__ float to(ex_f16 a) { return (float)__builtin_bit_cast(_Float16, a.v); }
    static __device__ __forceinline__ ex_f16 from(float f) { ex_f16 r; r.v = __builtin_bit_cast(uint16_t, (_Float16)f); return r; }
};
struct ex_f32 {
    float v;
    static __device__ __forceinline__ float to(ex_f32 a) { return a.v; }
    static __device__ __forceinline__ ex_f32 from(float f) { ex_f32 r; r.v = f; return r; }
};
// V elements of a row that starts at any multiple of the element's size (16-byte accesses at any alignment of 2 are single
// instructions on gfx950)
template <typename T, int V> struct __attribute__((packed, aligned(2))) ex_vec { T e[V]; };

static __device__ __forceinline__ float ex_weight(const void *w, int32_t wtype, int64_t p) {
    if (!w) return 1.f;
    if (wtype == CG3D_DT_F32) return reinterpret_cast<const float *>(w)[p];
    if (wtype == CG3D_DT_BF16) return ex_bf16::to(reinterpret_cast<const ex_bf16 *>(w)[p]);
    return ex_f16::to(reinterpret_cast<const ex_f16 *>(w)[p]);
}

// ---------------------------------------------------------------- plan
// A wave takes 64 consecutive pairs at a time.  Lanes with equal keys find each other by one ballot per bit of the key; a lane's
// rank among them is the number of earlier lanes, the wave's running count of the key is kept in LDS (only this wave touches it).
static __device__ __forceinline__ int ex_key(const void *ids, int32_t wide, int64_t p, int E) {
    if (wide) {
        const int64_t v = reinterpret_cast<const int64_t *>(ids)[p];
        return (uint64_t)v < (uint64_t)E ? (int)v : E;
    }
    const int32_t v = reinterpret_cast<const int32_t *>(ids)[p];
    return (uint32_t)v < (uint32_t)E ? v : E;
}
static __device__ __forceinline__ uint64_t ex_peers(int key, bool in, int bits) {
    uint64_t m = __ballot(in);
    for (int b = 0; b < bits; b++) {
        const bool one = (key >> b) & 1;
        const uint64_t v = __ballot(one);
        m &= one ? v : ~v;
    }
    return m;
}
static __device__ __forceinline__ uint64_t ex_below(int lane) { return (1ull << lane) - 1; }

// counts of the keys of pairs [p0, p1) into the wave's row h[0 .. E]
static __device__ __forceinline__ void ex_wave_count(const void *ids, int32_t wide, int64_t p0, int64_t p1, int E, int bits, int lane,
                                                     int32_t *h) {
    for (int64_t p = p0; p < p1; p += 64) {
        const bool in = p + lane < p1;
        const int key = in ? ex_key(ids, wide, p + lane, E) : E;
        const uint64_t m = ex_peers(key, in, bits);
        if (in && (m & ex_below(lane)) == 0) atomicAdd(&h[key], __popcll(m));    // (the first of its peers; no other wave's row)
    }
}
// the rows of the pairs [p0, p1): h[key] holds the next row of each key and is moved on
static __device__ __forceinline__ void ex_wave_place(const void *ids, int32_t wide, int64_t p0, int64_t p1, int E, int bits, int lane,
                                                     int32_t *h, int32_t k, int32_t *__restrict__ rows, int32_t *__restrict__ pos) {
    for (int64_t p = p0; p < p1; p += 64) {
        const bool in = p + lane < p1;
        const int key = in ? ex_key(ids, wide, p + lane, E) : E;
        const uint64_t m = ex_peers(key, in, bits);
        int base = 0;
        if (in && (m & ex_below(lane)) == 0) base = atomicAdd(&h[key], __popcll(m));
        const int first = in ? __ffsll((unsigned long long)m) - 1 : lane;
        base = __shfl(base, first);
        if (in) {
            const int row = base + __popcll(m & ex_below(lane));
            pos[p + lane] = key < E ? row : ~row;
            rows[row] = key < E ? (int32_t)((p + lane) / k) : -1;
        }
    }
}
// exclusive prefix sums over keys [0, E] of tot[], in place, by the whole block (nt threads, scr: nt / 64 ints)
static __device__ __forceinline__ void ex_block_scan(int32_t *tot, int n, int32_t *scr) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6;
    int carry = 0;
    for (int b = 0; b < n; b += nt) {
        const int i = b + tid;
        const int v = i < n ? tot[i] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s, d); if (lane >= d) s += o; }
        if (lane == 63) scr[wave] = s;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < (nt >> 6); w++) { if (w < wave) before += scr[w]; all += scr[w]; }
        if (i < n) tot[i] = before + s - v;
        carry += all;
        __syncthreads();
    }
}

// up to EX_ONE pairs: everything in one workgroup of 16 waves
#define EX_ONE 16384
__global__ __launch_bounds__(1024) void k_expert_plan_one(const void *__restrict__ ids, int32_t wide, int32_t n, int32_t k, int32_t E,
                                                          int32_t bits, int32_t *__restrict__ offsets, int32_t *__restrict__ rows,
                                                          int32_t *__restrict__ pos) {
    extern __shared__ int32_t ex_sm[];
    const int nw = blockDim.x >> 6, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int32_t *const hist = ex_sm, *const tot = ex_sm + nw * (E + 1), *const scr = tot + (E + 1);
    for (int i = tid; i < nw * (E + 1); i += blockDim.x) hist[i] = 0;
    __syncthreads();
    const int per = ((n + nw - 1) / nw + 63) & ~63;
    const int p0 = min(n, wave * per), p1 = min(n, p0 + per);
    ex_wave_count(ids, wide, p0, p1, E, bits, lane, hist + wave * (E + 1));
    __syncthreads();
    for (int e = tid; e <= E; e += blockDim.x) {
        int s = 0;
        for (int w = 0; w < nw; w++) { const int c = hist[w * (E + 1) + e]; hist[w * (E + 1) + e] = s; s += c; }
        tot[e] = s;
    }
    __syncthreads();
    ex_block_scan(tot, E + 1, scr);
    for (int e = tid; e <= E; e += blockDim.x) {
        offsets[e] = tot[e];                             // tot[E]: the first row without a pair = the number of rows
        for (int w = 0; w < nw; w++) hist[w * (E + 1) + e] += tot[e];
    }
    __syncthreads();
    ex_wave_place(ids, wide, p0, p1, E, bits, lane, hist + wave * (E + 1), k, rows, pos);
}

// more pairs: workgroup b owns the pairs [b * per_block, (b + 1) * per_block); counts [nblk][E + 1] go through memory, and every
// workgroup of the second launch adds up the columns it needs itself (at most EX_BLOCKS rows)
#define EX_BLOCKS 256
__global__ __launch_bounds__(256) void k_expert_plan_count(const void *__restrict__ ids, int32_t wide, int64_t n, int32_t E, int32_t bits,
                                                           int64_t per_wave, int32_t *__restrict__ counts) {
    extern __shared__ int32_t ex_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i <= E; i += 256) ex_sm[i] = 0;
    __syncthreads();
    const int64_t p0 = min(n, ((int64_t)blockIdx.x * 4 + wave) * per_wave), p1 = min(n, p0 + per_wave);
    ex_wave_count(ids, wide, p0, p1, E, bits, lane, ex_sm);       // (one row for the workgroup: whole numbers add up in any order)
    __syncthreads();
    for (int i = tid; i <= E; i += 256) counts[(int64_t)blockIdx.x * (E + 1) + i] = ex_sm[i];
}
__global__ __launch_bounds__(256) void k_expert_plan_place(const void *__restrict__ ids, int32_t wide, int64_t n, int32_t k, int32_t E,
                                                           int32_t bits, int64_t per_wave, const int32_t *__restrict__ counts,
                                                           int32_t *__restrict__ offsets, int32_t *__restrict__ rows,
                                                           int32_t *__restrict__ pos) {
    extern __shared__ int32_t ex_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nblk = gridDim.x, me = blockIdx.x;
    int32_t *const hist = ex_sm, *const tot = ex_sm + 4 * (E + 1), *const mine = tot + (E + 1), *const scr = mine + (E + 1);
    for (int i = tid; i < 4 * (E + 1); i += 256) hist[i] = 0;
    for (int e = tid; e <= E; e += 256) {
        int all = 0, before = 0;
        for (int b = 0; b < nblk; b++) { const int c = counts[(int64_t)b * (E + 1) + e]; all += c; before += b < me ? c : 0; }
        tot[e] = all;
        mine[e] = before;
    }
    __syncthreads();
    const int64_t p0 = min(n, ((int64_t)me * 4 + wave) * per_wave), p1 = min(n, p0 + per_wave);
    ex_wave_count(ids, wide, p0, p1, E, bits, lane, hist + wave * (E + 1));
    ex_block_scan(tot, E + 1, scr);                      // (starts and ends with barriers of its own for scr; tot is complete above)
    __syncthreads();
    for (int e = tid; e <= E; e += 256) {
        if (me == 0) offsets[e] = tot[e];
        int s = tot[e] + mine[e];
        for (int w = 0; w < 4; w++) { const int c = hist[w * (E + 1) + e]; hist[w * (E + 1) + e] = s; s += c; }
    }
    __syncthreads();
    ex_wave_place(ids, wide, p0, p1, E, bits, lane, hist + wave * (E + 1), k, rows, pos);
}

static int64_t ex_blocks(int64_t n) { return n <= EX_ONE ? 0 : (cg3d_divup(n, 4 * 512) < EX_BLOCKS ? cg3d_divup(n, 4 * 512) : EX_BLOCKS); }

extern "C" int64_t cg3d_expert_plan_ws_bytes(int64_t n_tokens, int32_t k, int32_t n_experts) {
    if (n_tokens < 0 || k < 1 || n_experts < 1 || n_experts > EX_MAX_EXPERTS || n_tokens > 0x7fffffffll / k) return CG3D_ERR_ARG;
    return ex_blocks(n_tokens * k) * (n_experts + 1) * (int64_t)sizeof(int32_t);
}
extern "C" int cg3d_expert_plan(const void *experts, int32_t wide, int64_t n_tokens, int32_t k, int32_t n_experts, int32_t *offsets,
                                int32_t *rows, int32_t *pos, void *ws, cg3d_stream_t stream) {
    if (cg3d_expert_plan_ws_bytes(n_tokens, k, n_experts) < 0 || (wide != 0 && wide != 1) || !offsets) return CG3D_ERR_ARG;
    const int64_t n = n_tokens * k;
    if (n > 0 && (!experts || !rows || !pos || ((uintptr_t)experts & (wide ? 7 : 3)))) return CG3D_ERR_ARG;
    const int64_t nblk = ex_blocks(n);
    if (nblk > 0 && !ws) return CG3D_ERR_ARG;
    int bits = 1;
    while ((n_experts >> bits) != 0) bits++;
    hipStream_t s = cg3d_hs(stream);
    if (nblk == 0) {
        int nt = n <= 64 ? 64 : n >= 1024 ? 1024 : (int)((n + 63) & ~63ll);
        const size_t lds = ((size_t)(nt / 64 + 1) * (n_experts + 1) + 16) * sizeof(int32_t);
        if (lds > 64 * 1024) {
            if (hipFuncSetAttribute(reinterpret_cast<const void *>(&k_expert_plan_one), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
                return CG3D_ERR_LAUNCH;
        }
        hipLaunchKernelGGL(k_expert_plan_one, dim3(1), dim3(nt), lds, s, experts, wide, (int32_t)n, k, n_experts, bits, offsets, rows, pos);
        CG3D_CHECK_LAUNCH();
        return CG3D_OK;
    }
    const int64_t per_wave = (cg3d_divup(n, nblk * 4) + 63) & ~63ll;
    int32_t *counts = reinterpret_cast<int32_t *>(ws);
    hipLaunchKernelGGL(k_expert_plan_count, dim3((unsigned)nblk), dim3(256), (n_experts + 1) * sizeof(int32_t), s, experts, wide, n,
                       n_experts, bits, per_wave, counts);
    CG3D_CHECK_LAUNCH();
    hipLaunchKernelGGL(k_expert_plan_place, dim3((unsigned)nblk), dim3(256), (6 * (n_experts + 1) + 4) * sizeof(int32_t), s, experts, wide,
                       n, k, n_experts, bits, per_wave, counts, offsets, rows, pos);
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

// ---------------------------------------------------------------- rows
static __device__ __forceinline__ int64_t ex_div(int64_t i, int32_t d) {
    return (i >> 32) ? i / d : (int64_t)((uint32_t)i / (uint32_t)d);
}
// A thread owns V elements (16 bytes) of one token's row; the last vector of a row whose width V does not divide is moved back to
// end with the row (its first elements are then computed twice, with the same result).  Rows shorter than a vector: V = 1.
template <typename T, int V>
__global__ __launch_bounds__(256) void k_expert_gather(const T *__restrict__ x, const int32_t *__restrict__ pos, int64_t n_tokens,
                                                       int32_t k, int32_t c, int32_t nv, T *__restrict__ out) {
    typedef ex_vec<T, V> vec;
    const int64_t P = n_tokens * k;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n_tokens * nv; i += gridDim.x * 256ll) {
        const int64_t t = ex_div(i, nv);
        int a = (int)(i - t * nv) * V;
        if (a + V > c) a = c - V;
        const vec v = *reinterpret_cast<const vec *>(x + t * c + a);
        vec z;
#pragma unroll
        for (int j = 0; j < V; j++) z.e[j] = T::from(0.f);
        for (int s = 0; s < k; s++) {
            const int32_t r = pos[t * k + s];
            const int64_t j = r < 0 ? ~r : r;
            if (j < P) *reinterpret_cast<vec *>(out + j * c + a) = r < 0 ? z : v;
        }
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void k_expert_combine(const T *__restrict__ y, const int32_t *__restrict__ pos, const void *__restrict__ w,
                                                        int32_t wtype, int64_t n_tokens, int32_t k, int32_t c, int32_t nv,
                                                        T *__restrict__ out) {
    typedef ex_vec<T, V> vec;
    const int64_t P = n_tokens * k;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n_tokens * nv; i += gridDim.x * 256ll) {
        const int64_t t = ex_div(i, nv);
        int a = (int)(i - t * nv) * V;
        if (a + V > c) a = c - V;
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = 0.f;
        for (int s = 0; s < k; s++) {
            const int32_t r = pos[t * k + s];
            if (r < 0 || r >= P) continue;
            const float ws = ex_weight(w, wtype, t * k + s);
            const vec v = *reinterpret_cast<const vec *>(y + (int64_t)r * c + a);
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] += ws * T::to(v.e[j]);
        }
        vec o;
#pragma unroll
        for (int j = 0; j < V; j++) o.e[j] = T::from(acc[j]);
        *reinterpret_cast<vec *>(out + t * c + a) = o;
    }
}

// L lanes (a power of two, at most a wave) own one token: slot by slot dy = w do and the lanes' shares of <do, y>, joined by shuffles
template <typename T, int V>
__global__ __launch_bounds__(256) void k_expert_combine_bwd(const T *__restrict__ dout, const T *__restrict__ y, const int32_t *__restrict__ pos,
                                                            const void *__restrict__ w, int32_t wtype, int64_t n_tokens, int32_t k,
                                                            int32_t c, int32_t nv, int32_t lshift, T *__restrict__ dy, void *__restrict__ dw) {
    typedef ex_vec<T, V> vec;
    const int L = 1 << lshift, lane = threadIdx.x & (L - 1);
    const int64_t P = n_tokens * k;
    // (whole groups of L lanes take a token and leave together)
    for (int64_t t = (blockIdx.x * 256ll + threadIdx.x) >> lshift; t < n_tokens; t += (gridDim.x * 256ll) >> lshift)
    for (int s = 0; s < k; s++) {
        const int32_t r = pos[t * k + s];
        const int64_t j = r < 0 ? ~(int64_t)r : (int64_t)r;
        const bool there = r >= 0 && j < P;
        const float ws = there ? ex_weight(w, wtype, t * k + s) : 0.f;
        float dot = 0.f;
        if (j < P) {
            for (int q = lane; q < nv; q += L) {
                const int a0 = q * V, a = a0 + V > c ? c - V : a0;
                vec g, o;
                if (there) g = *reinterpret_cast<const vec *>(dout + t * c + a);
                if (dw && there) {
                    const vec v = *reinterpret_cast<const vec *>(y + j * c + a);
#pragma unroll
                    for (int u = 0; u < V; u++) dot += a + u >= a0 ? T::to(g.e[u]) * T::to(v.e[u]) : 0.f;
                }
                if (dy) {
#pragma unroll
                    for (int u = 0; u < V; u++) o.e[u] = T::from(there ? ws * T::to(g.e[u]) : 0.f);
                    *reinterpret_cast<vec *>(dy + j * c + a) = o;
                }
            }
        }
        if (dw) {
            for (int d = L >> 1; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
            if (lane == 0) {
                if (wtype == CG3D_DT_F32) reinterpret_cast<float *>(dw)[t * k + s] = dot;
                else if (wtype == CG3D_DT_BF16) reinterpret_cast<ex_bf16 *>(dw)[t * k + s] = ex_bf16::from(dot);
                else reinterpret_cast<ex_f16 *>(dw)[t * k + s] = ex_f16::from(dot);
            }
        }
    }
}

static bool ex_bad(int32_t dtype, int32_t wtype, int64_t n_tokens, int32_t k, int32_t c) {
    return dtype < CG3D_DT_F32 || dtype > CG3D_DT_F16 || wtype < CG3D_DT_F32 || wtype > CG3D_DT_F16 || n_tokens < 0 || k < 1 || c < 1 ||
           n_tokens > 0x7fffffffll / k;
}
static bool ex_odd(const void *p, int32_t dtype) { return ((uintptr_t)p & (dtype == CG3D_DT_F32 ? 3 : 1)) != 0; }

static int64_t ex_grid(int64_t nb) { return nb < (1 << 22) ? nb : (1 << 22); }      // (fewer than 2^32 threads; the kernels loop)

#define EX_DISPATCH(LAUNCH)                                                                                        \
    do {                                                                                                           \
        if (dtype == CG3D_DT_F32) { if (c >= 4) LAUNCH(ex_f32, 4); else LAUNCH(ex_f32, 1); }                       \
        else if (dtype == CG3D_DT_BF16) { if (c >= 8) LAUNCH(ex_bf16, 8); else LAUNCH(ex_bf16, 1); }               \
        else { if (c >= 8) LAUNCH(ex_f16, 8); else LAUNCH(ex_f16, 1); }                                            \
    } while (0)

extern "C" int cg3d_expert_gather(const void *x, int32_t dtype, const int32_t *pos, int64_t n_tokens, int32_t k, int32_t c, void *out,
                                  cg3d_stream_t stream) {
    if (ex_bad(dtype, CG3D_DT_F32, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!x || !pos || !out || ex_odd(x, dtype) || ex_odd(out, dtype)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH(T, V)                                                                                            \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens * nv, 256));                                                \
        hipLaunchKernelGGL((k_expert_gather<T, V>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(x), pos, n_tokens, k, \
                           c, nv, reinterpret_cast<T *>(out));                                                     \
    } while (0)
    EX_DISPATCH(EX_LAUNCH);
#undef EX_LAUNCH
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

extern "C" int cg3d_expert_combine(const void *y, int32_t dtype, const int32_t *pos, const void *w, int32_t wtype, int64_t n_tokens,
                                   int32_t k, int32_t c, void *out, cg3d_stream_t stream) {
    if (ex_bad(dtype, wtype, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!y || !pos || !out || ex_odd(y, dtype) || ex_odd(out, dtype) || ex_odd(w, wtype)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH(T, V)                                                                                            \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens * nv, 256));                                                \
        hipLaunchKernelGGL((k_expert_combine<T, V>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(y), pos, w, wtype, \
                           n_tokens, k, c, nv, reinterpret_cast<T *>(out));                                        \
    } while (0)
    EX_DISPATCH(EX_LAUNCH);
#undef EX_LAUNCH
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

extern "C" int cg3d_expert_combine_bwd(const void *dout, const void *y, int32_t dtype, const int32_t *pos, const void *w, int32_t wtype,
                                       int64_t n_tokens, int32_t k, int32_t c, void *dy, void *dw, cg3d_stream_t stream) {
    if (ex_bad(dtype, wtype, n_tokens, k, c) || (!dy && !dw)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!dout || !pos || (dw && (!y || !w)) || ex_odd(dout, dtype) || ex_odd(y, dtype) || ex_odd(dy, dtype) || ex_odd(w, wtype) || ex_odd(dw, wtype))
        return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH(T, V)                                                                                            \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        int32_t ls = 0;                                                                                            \
        while ((1 << ls) < nv && ls < 6) ls++;                                                                     \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens << ls, 256));                                               \
        hipLaunchKernelGGL((k_expert_combine_bwd<T, V>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(dout),   \
                           reinterpret_cast<const T *>(y), pos, w, wtype, n_tokens, k, c, nv, ls, reinterpret_cast<T *>(dy), dw);  \
    } while (0)
    EX_DISPATCH(EX_LAUNCH);
#undef EX_LAUNCH
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}
