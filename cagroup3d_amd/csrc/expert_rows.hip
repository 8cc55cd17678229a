// expert_rows.hip -- rows sorted by expert and back (gfx950): the plan of a routing (a stable counting sort of the (token, slot)
// pairs by their expert), the gather of the tokens' rows into that order, the weighted combination back to tokens, and the
// gradients of both.
//
//   p = t * k + s;  e(p) = experts[t, s];  a pair whose id is outside [0, E) has no row
//   row of p   = #{ q : e(q) < e(p) } + #{ q < p : e(q) = e(p) }             (experts ascending, pairs ascending inside one)
//   gather       r[row(t, s)] = x[t]                    its gradient   dx[t] = sum_s dr[row(t, s)]
//   combine      o[t] = sum_s w[t, s] y[row(t, s)]      its gradient   dy[row(t, s)] = w[t, s] do[t],  dw[t, s] = <do[t], y[row(t, s)]>
//
// Every pass runs over what it WRITES, row by row or token by token, so that writes are streamed and only reads jump (the gather of
// 155 773 x 2 rows of 256 bytes: 41 us token by token, 29 us row by row), and no sum needs an atomic: results are the same from run to
// run.  The T * k - offsets[E] rows behind the last belong to the pairs without a row (pos = ~row, pairs = ~pair, negative), so that
// the passes that write rows clear them, and their weights' gradients.  Sums are held in fp32 in slot order and rounded once.
#include "cg3d_common.h"

#define EX_MAX_EXPERTS 1024
#define EX_STEPS 2                   // ids of a lane in flight

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
typedef uint32_t ex_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t ex_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
// results are streamed past the caches (non-temporal): they are larger than a die's 4 MB of L2 where it matters (combination of
// 155 773 x 2 rows of 256 bytes 27.2 -> 24.5 us, of 20 011 x 8 rows of 502 bytes 28.1 -> 22.4 us; nothing at 2.5 MB)
template <typename vec> static __device__ __forceinline__ void ex_put(vec *p, const vec &v) {
    if constexpr (sizeof(vec) == 16) { __builtin_nontemporal_store(__builtin_bit_cast(ex_u32x4, v), reinterpret_cast<ex_u32x4 *>(p)); return; }
    if constexpr (sizeof(vec) == 8) { __builtin_nontemporal_store(__builtin_bit_cast(ex_u32x2, v), reinterpret_cast<ex_u32x2 *>(p)); return; }
    *p = v;
}

static __device__ __forceinline__ float ex_weight(const void *w, int32_t wtype, int64_t p) {
    if (!w) return 1.f;
    if (wtype == CG3D_DT_F32) return reinterpret_cast<const float *>(w)[p];
    if (wtype == CG3D_DT_BF16) return ex_bf16::to(reinterpret_cast<const ex_bf16 *>(w)[p]);
    return ex_f16::to(reinterpret_cast<const ex_f16 *>(w)[p]);
}

// ---------------------------------------------------------------- plan
// A wave takes 64 consecutive pairs at a time.  Lanes with equal keys find each other by one ballot per bit of the key; a lane's
// rank among them is the number of earlier lanes, the wave's running count of the key is kept in LDS (only this wave touches it).
// Bound by the chain ids - counts - offsets - rows, each a trip to memory, not by its 20 bytes a pair: 82 107 x 2 ids of 18 experts count
// 3.3 + place 6.7 us, 155 773 x 2 4.6 + 8.5 us; one token 3 us, a launch.
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

// exclusive prefix sums of tot[0 .. n) in place, by the whole workgroup (scr: an int for each wave)
static __device__ __forceinline__ void ex_block_scan(int32_t *tot, int n, int32_t *scr) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x >> 6;
    int carry = 0;
    for (int b = 0; b < n; b += blockDim.x) {
        const int i = b + tid;
        const int v = i < n ? tot[i] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s, d); if (lane >= d) s += o; }
        if (lane == 63) scr[wave] = s;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < nw; w++) { const int c = scr[w]; if (w < wave) before += c; all += c; }
        if (i < n) tot[i] = before + s - v;
        carry += all;
        __syncthreads();
    }
}

// A chunk of blockDim * EX_STEPS pairs belongs to a workgroup: wave w takes the EX_STEPS * 64 pairs behind w of those, all its ids in
// flight at once.  Chunks of one workgroup follow each other, so that any number of pairs needs at most ex_shape's workgroups.
// ex_chunk_ranks: counts of the keys in the wave's row h[0 .. E] of LDS and each pair's rank in the wave.
static __device__ __forceinline__ void ex_chunk_keys(const void *ids, int32_t wide, int64_t p, int64_t n, int E, int (&key)[EX_STEPS]) {
#pragma unroll
    for (int i = 0; i < EX_STEPS; i++) {
        const int64_t q = p + i * 64;
        key[i] = ex_key(ids, wide, q < n ? q : n - 1, E);
    }
}
static __device__ __forceinline__ void ex_chunk_ranks(const int (&key)[EX_STEPS], int64_t p, int64_t n, int bits, int lane, int32_t *h,
                                                      int (&rank)[EX_STEPS]) {
#pragma unroll
    for (int i = 0; i < EX_STEPS; i++) {
        const bool in = p + i * 64 < n;
        if (!__any(in)) break;
        const uint64_t m = ex_peers(key[i], in, bits);
        int base = 0;
        if (in && (m & ex_below(lane)) == 0) base = atomicAdd(&h[key[i]], __popcll(m));      // (the first of its peers)
        base = __shfl(base, in ? __ffsll((unsigned long long)m) - 1 : lane);
        rank[i] = base + __popcll(m & ex_below(lane));
    }
}
static __device__ __forceinline__ void ex_chunk_count(const int (&key)[EX_STEPS], int64_t p, int64_t n, int bits, int lane, int32_t *h) {
#pragma unroll
    for (int i = 0; i < EX_STEPS; i++) {
        const bool in = p + i * 64 < n;
        if (!__any(in)) break;
        const uint64_t m = ex_peers(key[i], in, bits);
        if (in && (m & ex_below(lane)) == 0) atomicAdd(&h[key[i]], __popcll(m));             // (whole numbers: any order)
    }
}

// more than one workgroup: counts [nblk][W4] of the workgroups' pairs go through memory (W4: E + 1 up to a multiple of 4)
__global__ __launch_bounds__(1024) void k_expert_plan_count(const void *__restrict__ ids, int32_t wide, int64_t n, int32_t E,
                                                                  int32_t bits, int32_t chunks, int32_t *__restrict__ counts) {
    extern __shared__ int32_t ex_sm[];
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6, W4 = (E + 4) & ~3;
    const int64_t chunk = (int64_t)nt * EX_STEPS, p = blockIdx.x * chunks * chunk + wave * (EX_STEPS * 64) + lane;
    int key[EX_STEPS];
    ex_chunk_keys(ids, wide, p, n, E, key);
    for (int i = tid; i < W4; i += nt) ex_sm[i] = 0;
    __syncthreads();
    ex_chunk_count(key, p, n, bits, lane, ex_sm);
    for (int c = 1; c < chunks; c++) {
        ex_chunk_keys(ids, wide, p + c * chunk, n, E, key);
        ex_chunk_count(key, p + c * chunk, n, bits, lane, ex_sm);
    }
    __syncthreads();
    for (int i = tid; i < W4; i += nt) counts[(int64_t)blockIdx.x * W4 + i] = ex_sm[i];
}
// The first row of each key for this workgroup, from the counts of all of them (the workgroup adds their rows up
// itself, four columns of a thread at a time), or from its own pairs when it is the only one; then chunk by chunk the rows of the pairs.
__global__ __launch_bounds__(1024) void k_expert_plan_place(const void *__restrict__ ids, int32_t wide, int64_t n, int32_t k,
                                                                  int32_t E, int32_t bits, int32_t chunks, const int32_t *__restrict__ counts,
                                                                  int32_t *__restrict__ offsets, int32_t *__restrict__ rows,
                                                                  int32_t *__restrict__ pairs, int32_t *__restrict__ pos) {
    extern __shared__ int32_t ex_sm[];
    const int tid = threadIdx.x, nt = blockDim.x, nw = nt >> 6, lane = tid & 63, wave = tid >> 6, nblk = gridDim.x, me = blockIdx.x;
    const int W4 = (E + 4) & ~3, W = E + 1;
    int32_t *const hist = ex_sm, *const tot = ex_sm + nw * W4, *const next = tot + W4, *const scr = next + W4;
    const int64_t chunk = (int64_t)nt * EX_STEPS;
    const int64_t p0 = (int64_t)me * chunks * chunk + wave * (EX_STEPS * 64) + lane;
    int key[EX_STEPS], rank[EX_STEPS];
    if (n > 0) ex_chunk_keys(ids, wide, p0, n, E, key);              // (the first chunk's ids travel while the counts are added up)
    for (int i = tid; i < (nw + 2) * W4; i += nt) ex_sm[i] = 0;
    __syncthreads();
    if (counts) {
        const int nv = W4 >> 2;
        int width = 1;
        while (width < nv && width < nt) width <<= 1;
        const int part = tid / width, parts = nt / width;
        for (int v = tid & (width - 1); v < nv; v += width) {
            int4 all = make_int4(0, 0, 0, 0), before = all;
#pragma unroll 4
            for (int b = part; b < nblk; b += parts) {
                const int4 c = *reinterpret_cast<const int4 *>(counts + (int64_t)b * W4 + v * 4);
                all.x += c.x; all.y += c.y; all.z += c.z; all.w += c.w;
                if (b < me) { before.x += c.x; before.y += c.y; before.z += c.z; before.w += c.w; }
            }
            atomicAdd(&tot[v * 4], all.x); atomicAdd(&tot[v * 4 + 1], all.y); atomicAdd(&tot[v * 4 + 2], all.z); atomicAdd(&tot[v * 4 + 3], all.w);
            atomicAdd(&next[v * 4], before.x); atomicAdd(&next[v * 4 + 1], before.y); atomicAdd(&next[v * 4 + 2], before.z); atomicAdd(&next[v * 4 + 3], before.w);
        }
    } else if (chunks > 1)                                           // the only workgroup, several chunks: counted first
        for (int c = 0; c < chunks; c++) {
            int later[EX_STEPS];
            ex_chunk_keys(ids, wide, p0 + c * chunk, n, E, later);
            ex_chunk_count(later, p0 + c * chunk, n, bits, lane, tot);
        }
    if (n > 0) ex_chunk_ranks(key, p0, n, bits, lane, hist + wave * W4, rank);
    __syncthreads();
    if (!counts && chunks == 1) {
        for (int e = tid; e < W; e += nt) {
            int s = 0;
            for (int w = 0; w < nw; w++) s += hist[w * W4 + e];
            tot[e] = s;
        }
        __syncthreads();
    }
    ex_block_scan(tot, W, scr);
    for (int e = tid; e < W; e += nt) {
        if (me == 0) offsets[e] = tot[e];                            // (tot[E]: the first row without a pair = the number of rows)
        next[e] += tot[e];
    }
    for (int c = 0; c < chunks; c++) {
        const int64_t p = p0 + c * chunk;
        if (c > 0) {
            ex_chunk_keys(ids, wide, p, n, E, key);
            __syncthreads();                                         // (the rows of hist have been read by everyone)
            for (int i = lane; i < W; i += 64) hist[wave * W4 + i] = 0;
            ex_chunk_ranks(key, p, n, bits, lane, hist + wave * W4, rank);
            __syncthreads();
        }
        for (int e = tid; e < W; e += nt) {
            int at = next[e];
            for (int w = 0; w < nw; w++) { const int q = hist[w * W4 + e]; hist[w * W4 + e] = at; at += q; }
            next[e] = at;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EX_STEPS; i++) {
            const int64_t q = p + i * 64;
            if (q < n) {
                const int row = hist[wave * W4 + key[i]] + rank[i];
                const bool there = key[i] < E;
                pos[q] = there ? row : ~row;
                rows[row] = there ? (int32_t)((uint32_t)q / (uint32_t)k) : -1;
                pairs[row] = there ? (int32_t)q : ~(int32_t)q;
            }
        }
    }
}

// Threads, chunks of a workgroup and workgroups for n pairs.  Up to 4096 pairs one workgroup of up to 1024 threads does it, in one
// launch (1200 / 2000 pairs of 18 experts: 7.2 / 7.8 us, with two workgroups of 512 8.9 / 9.5).  Above, 512 threads and at most 512
// workgroups (164 214 pairs of 18 experts, both kernels: 10.6 us; 12.0 with 1024 and at most 256, 12.3 with twice the ids of a lane), but
// every workgroup adds up the counts of all of them, so that many experts in many workgroups want fewer and larger ones (311 546 pairs
// of 128 experts 16.5 against 21.8 us, of 1024 experts 30 / 72; about the same where workgroups x experts = 20 000).
struct ex_shape {
    int32_t threads, chunks;
    int64_t blocks;
    ex_shape(int64_t n, int32_t n_experts) {
        const int64_t small = cg3d_divup(n, 512 * EX_STEPS) < 512 ? cg3d_divup(n, 512 * EX_STEPS) : 512;
        const bool one = n <= 2 * 1024 * EX_STEPS, wide = one || (n_experts > 64 && small * n_experts > 20480);
        threads = wide ? 1024 : 512;
        const int64_t least = n > n_experts / 4 ? n : n_experts / 4;              // (2 pairs of 1024 experts: 15.6 us with 64 threads, 9.6 with 256)
        if (least < threads) threads = least <= 64 ? 64 : (int32_t)((least + 63) & ~63ll);
        const int64_t all = cg3d_divup(n, threads * EX_STEPS);
        chunks = one ? (all > 1 ? 2 : 1) : (int32_t)cg3d_divup(all, wide ? 256 : 512);
        blocks = one ? 1 : cg3d_divup(all, chunks);
    }
};

extern "C" int64_t cg3d_expert_plan_ws_bytes(int64_t n_tokens, int32_t k, int32_t n_experts) {
    if (n_tokens < 0 || k < 1 || n_experts < 1 || n_experts > EX_MAX_EXPERTS || n_tokens > 0x7fffffffll / k) return CG3D_ERR_ARG;
    const int64_t nblk = ex_shape(n_tokens * k, n_experts).blocks;
    return nblk == 1 ? 0 : nblk * ((n_experts + 4) & ~3) * (int64_t)sizeof(int32_t);
}
extern "C" int cg3d_expert_plan(const void *experts, int32_t wide, int64_t n_tokens, int32_t k, int32_t n_experts, int32_t *offsets,
                                int32_t *rows, int32_t *pairs, int32_t *pos, void *ws, cg3d_stream_t stream) {
    const int64_t need = cg3d_expert_plan_ws_bytes(n_tokens, k, n_experts);
    if (need < 0 || (wide != 0 && wide != 1) || !offsets) return CG3D_ERR_ARG;
    const int64_t n = n_tokens * k;
    if (n > 0 && (!experts || !rows || !pairs || !pos || ((uintptr_t)experts & (wide ? 7 : 3)))) return CG3D_ERR_ARG;
    if (need > 0 && (!ws || ((uintptr_t)ws & 15))) return CG3D_ERR_ARG;
    const ex_shape shape(n, n_experts);
    const int64_t nblk = shape.blocks;
    const int32_t chunks = shape.chunks, nt = shape.threads;
    int bits = 1;
    while ((n_experts >> bits) != 0) bits++;
    hipStream_t s = cg3d_hs(stream);
    const int W4 = (n_experts + 4) & ~3;
    const int lds = ((nt / 64 + 2) * W4 + nt / 64) * (int)sizeof(int32_t);          // (at most 72.4 KB)
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(&k_expert_plan_place), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return CG3D_ERR_LAUNCH;
    int32_t *counts = need > 0 ? reinterpret_cast<int32_t *>(ws) : nullptr;
    if (counts) {
        hipLaunchKernelGGL(k_expert_plan_count, dim3((unsigned)nblk), dim3(nt), W4 * sizeof(int32_t), s, experts, wide, n,
                           n_experts, bits, chunks, counts);
        CG3D_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(k_expert_plan_place, dim3((unsigned)nblk), dim3(nt), lds, s, experts, wide, n, k, n_experts, bits, chunks, counts,
                       offsets, rows, pairs, pos);
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

// ---------------------------------------------------------------- rows
// A thread owns V elements (16 bytes) of one token's row; the last vector of a row whose width V does not divide is moved back to
// end with the row (its first elements are then computed twice, with the same result).  Rows shorter than a vector: V = 1.  The
// combination takes a token's slots EX_SLOTS at a time: their rows are looked up, and then read, together.
// Bound by memory: 155 773 x 2 rows of 256 bytes gather 28 us (120 MB, 4.3 TB/s), combine 24.6 us (4.9 TB/s), its gradient 43.5 us (201 MB, 4.6
// TB/s); 20 011 x 8 rows of 502 bytes 24.8, 22.4 and 41.3 us (90, 90 and 171 MB).  A copy of 512 MB reaches 5.4 TB/s.
#define EX_SLOTS 4
// i / nv by a multiplication: magic = ceil(2^64 / nv), exact while i * nv < 2^64 (i counts 16-byte pieces of memory)
static __device__ __forceinline__ int64_t ex_div(int64_t i, int32_t nv, uint64_t magic) {
    return nv == 1 ? i : (int64_t)__umul64hi((uint64_t)i, magic);
}
template <typename T, int V>
__global__ __launch_bounds__(256) void k_expert_gather(const T *__restrict__ x, const int32_t *__restrict__ rows, int64_t n_tokens,
                                                       int64_t P, int32_t c, int32_t nv, uint64_t magic, T *__restrict__ out) {
    typedef ex_vec<T, V> vec;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < P * nv; i += gridDim.x * 256ll) {
        const int64_t j = ex_div(i, nv, magic);
        const int a = min((int)(i - j * nv) * V, c - V);
        const int32_t t = rows[j];
        vec v;
        if (t >= 0 && t < n_tokens) v = *reinterpret_cast<const vec *>(x + (int64_t)t * c + a);
        else {
#pragma unroll
            for (int u = 0; u < V; u++) v.e[u] = T::from(0.f);
        }
        ex_put(reinterpret_cast<vec *>(out + j * c + a), v);
    }
}

template <typename T, int V, typename O>
__global__ __launch_bounds__(256) void k_expert_combine(const T *__restrict__ y, const int32_t *__restrict__ pos, const void *__restrict__ w,
                                                        int32_t wtype, int64_t n_tokens, int32_t k, int32_t c, int32_t nv, uint64_t magic,
                                                        O *__restrict__ out) {
    typedef ex_vec<T, V> vec;
    const int64_t P = n_tokens * k;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n_tokens * nv; i += gridDim.x * 256ll) {
        const int64_t t = ex_div(i, nv, magic);
        const int a = min((int)(i - t * nv) * V, c - V);
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] = 0.f;
        for (int s0 = 0; s0 < k; s0 += EX_SLOTS) {
            int32_t r[EX_SLOTS];
            float ws[EX_SLOTS];
            vec v[EX_SLOTS];
#pragma unroll
            for (int s = 0; s < EX_SLOTS; s++) {
                const bool in = s0 + s < k;
                r[s] = in ? pos[t * k + s0 + s] : -1;
                ws[s] = in ? ex_weight(w, wtype, t * k + s0 + s) : 0.f;
            }
#pragma unroll
            for (int s = 0; s < EX_SLOTS; s++)
                if (r[s] >= 0 && r[s] < P) v[s] = *reinterpret_cast<const vec *>(y + (int64_t)r[s] * c + a);
#pragma unroll
            for (int s = 0; s < EX_SLOTS; s++)
                if (r[s] >= 0 && r[s] < P) {
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] += ws[s] * T::to(v[s].e[j]);
                }
        }
        ex_vec<O, V> o;
#pragma unroll
        for (int j = 0; j < V; j++) o.e[j] = O::from(acc[j]);
        ex_put(reinterpret_cast<ex_vec<O, V> *>(out + t * c + a), o);
    }
}

// L lanes (a power of two, at most a wave) own one row: dy = w do and the lanes' shares of <do, y>, joined by shuffles.  (Two or four
// rows of a group at a time, all their loads in flight together: 45.0 -> 48.0 -> 54.4 us at 155 773 x 2 rows of 256 bytes, not kept.)
template <typename T, int V>
__global__ __launch_bounds__(256) void k_expert_combine_bwd(const T *__restrict__ dout, const T *__restrict__ y, const int32_t *__restrict__ pairs,
                                                            const void *__restrict__ w, int32_t wtype, int64_t P, int32_t k, int32_t c,
                                                            int32_t nv, int32_t lshift, T *__restrict__ dy, void *__restrict__ dw) {
    typedef ex_vec<T, V> vec;
    const int L = 1 << lshift, lane = threadIdx.x & (L - 1);
    // (whole groups of L lanes take a row and leave together)
    for (int64_t j = (blockIdx.x * 256ll + threadIdx.x) >> lshift; j < P; j += (gridDim.x * 256ll) >> lshift) {
        const int32_t pr = pairs[j];
        const bool there = pr >= 0 && pr < P;
        const int32_t p = pr < 0 ? ~pr : pr;
        const int64_t t = there ? (int64_t)((uint32_t)p / (uint32_t)k) : 0;
        const float ws = there ? ex_weight(w, wtype, p) : 0.f;
        float dot = 0.f;
        for (int q = lane; q < nv; q += L) {
            const int a0 = q * V, a = min(a0, c - V);
            vec g, v, o;
            if (there) {
                g = *reinterpret_cast<const vec *>(dout + t * c + a);
                if (dw) v = *reinterpret_cast<const vec *>(y + j * c + a);
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                o.e[i] = T::from(there ? ws * T::to(g.e[i]) : 0.f);
                if (dw) dot += there && a + i >= a0 ? T::to(g.e[i]) * T::to(v.e[i]) : 0.f;
            }
            if (dy) ex_put(reinterpret_cast<vec *>(dy + j * c + a), o);
        }
        if (dw) {
            for (int d = L >> 1; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
            if (lane == 0 && p < P) {
                if (wtype == CG3D_DT_F32) reinterpret_cast<float *>(dw)[p] = dot;
                else if (wtype == CG3D_DT_BF16) reinterpret_cast<ex_bf16 *>(dw)[p] = ex_bf16::from(dot);
                else reinterpret_cast<ex_f16 *>(dw)[p] = ex_f16::from(dot);
            }
        }
    }
}

static bool ex_bad(int32_t dtype, int32_t wtype, int64_t n_tokens, int32_t k, int32_t c) {
    return dtype < CG3D_DT_F32 || dtype > CG3D_DT_F16 || wtype < CG3D_DT_F32 || wtype > CG3D_DT_F16 || n_tokens < 0 || k < 1 || c < 1 || c > (1 << 30) ||
           n_tokens > 0x7fffffffll / k;
}
static bool ex_odd(const void *p, int32_t dtype) { return ((uintptr_t)p & (dtype == CG3D_DT_F32 ? 3 : 1)) != 0; }

static uint64_t ex_magic(int32_t nv) { return nv > 1 ? ~0ull / (uint64_t)nv + 1 : 0; }      // ceil(2^64 / nv)
static int64_t ex_grid(int64_t nb) { return nb < (1 << 22) ? nb : (1 << 22); }      // (fewer than 2^32 threads; the kernels loop)

#define EX_DISPATCH(LAUNCH)                                                                                        \
    do {                                                                                                           \
        if (dtype == CG3D_DT_F32) { if (c >= 4) LAUNCH(ex_f32, 4); else LAUNCH(ex_f32, 1); }                       \
        else if (dtype == CG3D_DT_BF16) { if (c >= 8) LAUNCH(ex_bf16, 8); else LAUNCH(ex_bf16, 1); }               \
        else { if (c >= 8) LAUNCH(ex_f16, 8); else LAUNCH(ex_f16, 1); }                                            \
    } while (0)

extern "C" int cg3d_expert_gather(const void *x, int32_t dtype, const int32_t *rows, int64_t n_tokens, int32_t k, int32_t c, void *out,
                                  cg3d_stream_t stream) {
    if (ex_bad(dtype, CG3D_DT_F32, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!x || !rows || !out || ex_odd(x, dtype) || ex_odd(out, dtype)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH(T, V)                                                                                            \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens * k * nv, 256));                                                \
        hipLaunchKernelGGL((k_expert_gather<T, V>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(x), rows, n_tokens, n_tokens * k, \
                           c, nv, ex_magic(nv), reinterpret_cast<T *>(out));                                                     \
    } while (0)
    EX_DISPATCH(EX_LAUNCH);
#undef EX_LAUNCH
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

extern "C" int cg3d_expert_combine(const void *y, int32_t dtype, const int32_t *pos, const void *w, int32_t wtype, int64_t n_tokens,
                                   int32_t k, int32_t c, void *out, int32_t out_dtype, cg3d_stream_t stream) {
    if (ex_bad(dtype, wtype, n_tokens, k, c) || out_dtype < CG3D_DT_F32 || out_dtype > CG3D_DT_F16 || (dtype != CG3D_DT_F32 && out_dtype != dtype))
        return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!y || !pos || !out || ex_odd(y, dtype) || ex_odd(out, out_dtype) || ex_odd(w, wtype)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH_O(T, V, O)                                                                                       \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens * nv, 256));                                                \
        hipLaunchKernelGGL((k_expert_combine<T, V, O>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(y), pos, w, \
                           wtype, n_tokens, k, c, nv, ex_magic(nv), reinterpret_cast<O *>(out));                   \
    } while (0)
#define EX_LAUNCH(T, V) EX_LAUNCH_O(T, V, T)
    if (out_dtype == dtype) EX_DISPATCH(EX_LAUNCH);
    else if (out_dtype == CG3D_DT_BF16) { if (c >= 4) EX_LAUNCH_O(ex_f32, 4, ex_bf16); else EX_LAUNCH_O(ex_f32, 1, ex_bf16); }
    else { if (c >= 4) EX_LAUNCH_O(ex_f32, 4, ex_f16); else EX_LAUNCH_O(ex_f32, 1, ex_f16); }
#undef EX_LAUNCH
#undef EX_LAUNCH_O
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

extern "C" int cg3d_expert_combine_bwd(const void *dout, const void *y, int32_t dtype, const int32_t *pairs, const void *w, int32_t wtype,
                                       int64_t n_tokens, int32_t k, int32_t c, void *dy, void *dw, cg3d_stream_t stream) {
    if (ex_bad(dtype, wtype, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;                               // (empty tensors have no address)
    if ((!dy && !dw) || !dout || !pairs || (dw && (!y || !w)) || ex_odd(dout, dtype) || ex_odd(y, dtype) || ex_odd(dy, dtype) || ex_odd(w, wtype) || ex_odd(dw, wtype))
        return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
#define EX_LAUNCH(T, V)                                                                                            \
    do {                                                                                                           \
        const int32_t nv = (int32_t)cg3d_divup(c, V);                                                              \
        int32_t ls = 0;                                                                                            \
        while ((1 << ls) < nv && ls < 6) ls++;                                                                     \
        const int64_t nb = ex_grid(cg3d_divup(n_tokens * k << ls, 256));                                           \
        hipLaunchKernelGGL((k_expert_combine_bwd<T, V>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const T *>(dout),   \
                           reinterpret_cast<const T *>(y), pairs, w, wtype, n_tokens * k, k, c, nv, ls, reinterpret_cast<T *>(dy), dw);  \
    } while (0)
    EX_DISPATCH(EX_LAUNCH);
#undef EX_LAUNCH
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}
