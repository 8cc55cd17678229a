// int8_linear.hip -- Y = (Q @ W) * sx * sw + b in 8-bit integers with a scale for each row and each output channel (gfx950), dense or
// with a matrix of its own for each expert's rows, and the quantisation of rows and weights.
//
//   y[r, n] = (sum_k q[r, k] w[k, n]) * sx[r] * sw[n] + b[n]      the sum is exact: int32, fewer than 2^17 terms of at most 2^14
//   sx[r]   = max_k |x[r, k]| / 127,   q[r, k] = 127 x[r, k] / max |x[r, .]| rounded to the nearest, ties to even
//
// The rounding of q is decided exactly, not up to the error of a reciprocal.  With c = 127 / max rounded UP to fp32, t' = c x lies
// between the true t and t (1 + 2^-23), so that a wrong nearest level needs t' on or just above a half (by at most 127 * 2^-23 <
// 2^-16).  t' enters one fused multiply-add with 1.5 * 2^23 (its low byte is then the level) and is never rounded by itself.
//   fp32 rows: where t' falls into that strip the two sides 127 |x| and (n - 1/2) max are compared, each as an fp32 product and its
//   exact error.
//   16-bit rows: x = mx 2^i and max = ma 2^(i + s) with whole mx, ma < 2^11, so a t that is no half is off it by 1 / (2 ma 2^s) or more
//   -- over 2^-12 2^-s, against an error below 2^-15 2^-s: only true halves can go wrong, 254 mx = (2 n + 1) ma 2^s.  127 divides one
//   side's 2 n + 1 (n = 63: t' lands on 64, the even side, as it should) or ma = 127 k: for k a power of two c is exact and so is the
//   rounding, and only for the other k (fp16; bf16 has none, ma < 2^8) a row's elements are looked at like those of fp32 rows.
// A row that holds an infinity or a NaN gets the scale NaN (and so a row of NaN as its result); a row of zeros the scale 0.
//
// A tile of the product is v_mfma_i32_16x16x64_i8 with the rows as A and the weights as B operand.  The weights are laid out once
// (cg3d_int8_weight): [expert][panel of 64 channels][chunk of 64 contraction steps][tile nb of 4][lane][16 bytes]; lane (g = lane / 16,
// m = lane % 16) of tile nb holds contraction steps 16 g .. 16 g + 15 of channel 4 m + nb of the panel, so that a lane's results of
// the four tiles are 4 neighbouring channels and 16 neighbouring lanes store a whole line of a row.  Channels and contraction steps
// past the end are zeros.
#include "cg3d_common.h"
#pragma clang fp contract(off)      // a result has the same bits on every path

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));      // a row may start at any multiple of its element
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

#define I8_MAX_CIN 131071            // 2^14 * 131071 < 2^31: -128 * -128 included
#define I8_MAX_EXPERTS 1024
#define I8_FUSED_CIN 512
#define I8_FUSED_LONG 832            // for many rows of 16 bits

template <typename T, int V> struct __attribute__((packed, aligned(1))) i8_vec { T e[V]; };

struct i8_bf16 { uint16_t v; };
struct i8_f16 { uint16_t v; };
static __device__ __forceinline__ float i8_f(float a) { return a; }
static __device__ __forceinline__ float i8_f(i8_bf16 a) { return __uint_as_float((uint32_t)a.v << 16); }
static __device__ __forceinline__ float i8_f(i8_f16 a) { return (float)__builtin_bit_cast(_Float16, a.v); }
static __device__ __forceinline__ uint32_t i8_abs(float f) { return __float_as_uint(f) & 0x7fffffffu; }   // ordered like |f|; infinity and NaN on top

// ---------------------------------------------------------------- pieces of rows: 16 bytes, i8_els<T> elements, in whole registers
template <typename T> static constexpr int i8_els = 16 / (int)sizeof(T);
template <typename T> static __device__ __forceinline__ float i8_el(const u32x4 &w, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else {
        const uint32_t d = w[j >> 1];
        if constexpr (__is_same(T, i8_bf16)) return __uint_as_float(j & 1 ? d & 0xffff0000u : d << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? d >> 16 : d));
    }
}
// the piece at element k0 of a row of cin, zeros behind its end
template <typename T> static __device__ __forceinline__ u32x4 i8_piece(const T *__restrict__ xr, int k0, int cin) {
    constexpr int N = i8_els<T>, PER = 4 / (int)sizeof(T);           // PER: elements of a register
    u32x4 w = {0, 0, 0, 0};
    if (k0 + N <= cin) w = *reinterpret_cast<const u32x4_any *>(xr + k0);
    else if (k0 < cin) {
#pragma unroll
        for (int j = 0; j < N - 1; j++)
            if (k0 + j < cin) {
                uint32_t d = 0;
                __builtin_memcpy(&d, xr + k0 + j, sizeof(T));
                w[j / PER] |= d << (j % PER * 8 * (int)sizeof(T));
            }
    }
    return w;
}
// the running maximum of |.|: fp32 bits, or for 16-bit floats two at a time (their bits are ordered like their magnitudes too)
template <typename T> struct i8_max {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    uint32_t v = 0;
    __device__ __forceinline__ void add(const u32x4 &w) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (sizeof(T) == 4) v = max(v, w[j] & 0x7fffffffu);
            else v = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, v), __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu)));
        }
    }
    __device__ __forceinline__ uint32_t bits() const {                // of the fp32 value
        if constexpr (sizeof(T) == 4) return v;
        else {
            T t;
            t.v = (uint16_t)max(v & 0xffffu, v >> 16);
            return i8_abs(i8_f(t));
        }
    }
};
template <int CTRL> static __device__ __forceinline__ uint32_t i8_dpp(uint32_t v) {      // from another lane of 4, 8 or 16
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// the maximum over L = 4, 8, 16 or 64 neighbouring lanes, in all of them
template <int L> static __device__ __forceinline__ uint32_t i8_max_of(uint32_t v) {
    v = max(v, i8_dpp<0xb1>(v));                                      // quad_perm: lane ^ 1
    v = max(v, i8_dpp<0x4e>(v));                                      // quad_perm: lane ^ 2
    if constexpr (L >= 8) v = max(v, i8_dpp<0x141>(v));               // row_half_mirror: 7 - lane of 8
    if constexpr (L >= 16) v = max(v, i8_dpp<0x140>(v));              // row_mirror: 15 - lane of 16
    if constexpr (L >= 64) {
        v = max(v, (uint32_t)__shfl_xor((int)v, 16));
        v = max(v, (uint32_t)__shfl_xor((int)v, 32));
    }
    return v;
}

// What a row's largest magnitude (its bits) makes of the row's elements.  Rows whose largest is below 2^-96 or from 2^112 on are
// shifted by a power of two first (`shift`, exact for every element that is not level 0), so that no product here leaves the range.
struct i8_level {
    float amax, c, shift, scale;
    uint32_t keep;                                       // 0: the row has no levels
    bool fine127;                                        // max / 127 is exact, 127 / max is not
    i8_level() = default;
    __device__ __forceinline__ explicit i8_level(uint32_t top) {
        const float a = __uint_as_float(top);
        const bool fine = top < 0x7f800000u;
        shift = a < 0x1p-96f ? 0x1p96f : fine && a >= 0x1p112f ? 0x1p-16f : 1.f;
        keep = fine && top ? ~0u : 0u;
        amax = keep ? a * shift : 1.f;
        c = 127.f / amax;
        const float off = __builtin_fmaf(c, amax, -127.f), s127 = amax / 127.f;
        if (off < 0.f) c = __uint_as_float(__float_as_uint(c) + 1);
        fine127 = off != 0.f && __builtin_fmaf(s127, 127.f, -amax) == 0.f;
        scale = fine ? a / 127.f : __uint_as_float(0x7fc00000u);
    }
    __device__ __forceinline__ bool shifted() const { return shift != 1.f; }
};
#define I8_MAGIC 12582912.f          // 1.5 * 2^23
// r = the fma's result for x whose t' is in the strip: the level one nearer to zero where that is the nearest, ties to even
static __device__ __forceinline__ float i8_decide(const i8_level &v, float x, float r) {
    const float n = fabsf(r - I8_MAGIC), h = n - 0.5f, ax = fabsf(x);
    const float s = ax * 127.f, b = h * v.amax;
    const float es = __builtin_fmaf(ax, 127.f, -s), eb = __builtin_fmaf(h, v.amax, -b);
    const bool less = s < b || (s == b && es < eb), same = s == b && es == eb;
    const bool down = less || (same && ((int)n & 1));
    return down ? r - copysignf(1.f, r - I8_MAGIC) : r;
}
// N elements (shifted) of one row -> N levels, 4 to a word.  T: what the elements were
template <typename T, int N>
static __device__ __forceinline__ void i8_quant(const i8_level &v, const float (&x)[N], uint32_t (&out)[N / 4]) {
    float r[N];
    bool look = false;
#pragma unroll
    for (int j = 0; j < N; j++) r[j] = __builtin_fmaf(x[j], v.c, I8_MAGIC);
    if constexpr (sizeof(T) == 4) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < N; j++) most = fmaxf(most, fabsf(__builtin_fmaf(x[j], v.c, I8_MAGIC - r[j])));
        look = most > 0.5f - 0x1p-16f;
    } else if constexpr (__is_same(T, i8_f16)) look = v.fine127;
    if (!__is_same(T, i8_bf16) && __builtin_expect(__any(look), 0)) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float n = r[j] - I8_MAGIC, d = __builtin_fmaf(x[j], v.c, -n);
            if (d * n < 0.f && fabsf(d) > 0.5f - 0x1p-16f) r[j] = i8_decide(v, x[j], r[j]);     // (n = 0 is nearest from either side)
        }
    }
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
        const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(r[4 * i + 1]), __float_as_uint(r[4 * i]), 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(r[4 * i + 3]), __float_as_uint(r[4 * i + 2]), 0x04000c0cu);
        out[i] = (lo | hi) & v.keep;
    }
}
// the levels of a piece: i8_els<T> bytes
template <typename T> struct i8_lev { uint32_t w[i8_els<T> / 4]; };
template <typename T>
static __device__ __forceinline__ i8_lev<T> i8_levels(const i8_level &lev, bool far, const u32x4 &w) {
    constexpr int N = i8_els<T>;
    i8_lev<T> o;
    if constexpr (sizeof(T) == 1) {
#pragma unroll
        for (int j = 0; j < 4; j++) o.w[j] = w[j];
    } else {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; j++) f[j] = i8_el<T>(w, j);
        if (far) {
#pragma unroll
            for (int j = 0; j < N; j++) f[j] *= lev.shift;
        }
        i8_quant<T, N>(lev, f, o.w);
    }
    return o;
}

// ---------------------------------------------------------------- weights (once per model)
// w [E][cin][cout]: a thread of 16 to a channel, reads along the contraction are rows of the matrix (18 x 1024 x 1024 fp32: 13 us,
// 5.7 TB/s; the packing 27 us = 3.5 TB/s: a lane's channels are 4 apart, so that four waves read each line.  Once for a model)
template <typename T>
__global__ __launch_bounds__(1024) void k_i8_weight_scale(const T *__restrict__ w, int32_t cin, int32_t cout, float *__restrict__ scale,
                                                          uint32_t *__restrict__ top) {
    __shared__ uint32_t sh[16][64];
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6, e = blockIdx.y;
    uint32_t m = 0;
    if (n < cout) {
        const T *p = w + (int64_t)e * cin * cout + n;
#pragma unroll 4
        for (int k = part; k < cin; k += 16) m = max(m, i8_abs(i8_f(p[(int64_t)k * cout])));
    }
    sh[part][threadIdx.x & 63] = m;
    __syncthreads();
    if (part || n >= cout) return;
#pragma unroll
    for (int i = 1; i < 16; i++) m = max(m, sh[i][threadIdx.x]);
    scale[(int64_t)e * cout + n] = i8_level(m).scale;
    top[(int64_t)e * cout + n] = m;
}
// a thread writes the 16 bytes of one lane of one fragment (top == NULL: w is in 8 bits already)
template <typename T>
__global__ __launch_bounds__(256) void k_i8_weight_pack(const T *__restrict__ w, const uint32_t *__restrict__ top, int32_t cin, int32_t cout,
                                                        int32_t panels, int32_t chunks, int64_t total, int8_t *__restrict__ out) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int lane = (int)(i & 63), nb = (int)((i >> 6) & 3);
        const int64_t u = i >> 8;
        const int c = (int)(u % chunks), p = (int)((u / chunks) % panels), e = (int)(u / chunks / panels);
        const int n = p * 64 + (lane & 15) * 4 + nb, k0 = c * 64 + (lane >> 4) * 16;
        const bool there = n < cout;
        const T *src = w + (int64_t)e * cin * cout + (there ? n : 0);
        union { int8_t b[16]; uint32_t w[4]; u32x4 v; } o;
        if constexpr (sizeof(T) == 1) {
#pragma unroll
            for (int j = 0; j < 16; j++) o.b[j] = there && k0 + j < cin ? (int8_t)src[(int64_t)(k0 + j) * cout] : 0;
        } else {
            const i8_level lev(there ? top[(int64_t)e * cout + n] : 0);
            float f[16];
#pragma unroll
            for (int j = 0; j < 16; j++) f[j] = there && k0 + j < cin ? i8_f(src[(int64_t)(k0 + j) * cout]) * lev.shift : 0.f;
            i8_quant<T, 16>(lev, f, o.w);
        }
        reinterpret_cast<u32x4 *>(out)[i] = o.v;
    }
}

static bool i8_bad_shape(int32_t n_experts, int32_t cin, int32_t cout) {
    return n_experts < 1 || n_experts > I8_MAX_EXPERTS || cin < 1 || cin > I8_MAX_CIN || cout < 1 || cout > (1 << 20);
}
static int64_t i8_panels(int32_t cout) { return cg3d_divup(cout, 64); }
static int64_t i8_chunks(int32_t cin) { return cg3d_divup(cin, 64); }

extern "C" int64_t cg3d_int8_weight_bytes(int32_t n_experts, int32_t cin, int32_t cout) {
    if (i8_bad_shape(n_experts, cin, cout)) return CG3D_ERR_ARG;
    return (int64_t)n_experts * i8_panels(cout) * i8_chunks(cin) * 4096;
}
extern "C" int cg3d_int8_weight(const void *w, int32_t dtype, int32_t n_experts, int32_t cin, int32_t cout, int8_t *packed, float *scale,
                                void *ws, cg3d_stream_t stream) {
    if (i8_bad_shape(n_experts, cin, cout) || dtype < CG3D_DT_F32 || dtype > CG3D_DT_I8 || !w || !packed || ((uintptr_t)packed & 15)) return CG3D_ERR_ARG;
    if (((uintptr_t)w & (dtype == CG3D_DT_F32 ? 3 : dtype == CG3D_DT_I8 ? 0 : 1)) || (dtype != CG3D_DT_I8 && (!scale || !ws))) return CG3D_ERR_ARG;
    const int64_t total = cg3d_int8_weight_bytes(n_experts, cin, cout) / 16;
    const int32_t panels = (int32_t)i8_panels(cout), chunks = (int32_t)i8_chunks(cin);
    const unsigned nb = (unsigned)(cg3d_divup(total, 256) < (1 << 20) ? cg3d_divup(total, 256) : (1 << 20));
    hipStream_t s = cg3d_hs(stream);
    uint32_t *top = reinterpret_cast<uint32_t *>(ws);
#define I8_W(T)                                                                                                                     \
    do {                                                                                                                            \
        hipLaunchKernelGGL((k_i8_weight_scale<T>), dim3((unsigned)cg3d_divup(cout, 64), (unsigned)n_experts), dim3(1024), 0, s,     \
                           reinterpret_cast<const T *>(w), cin, cout, scale, top);                                                  \
        CG3D_CHECK_LAUNCH();                                                                                                        \
        hipLaunchKernelGGL((k_i8_weight_pack<T>), dim3(nb), dim3(256), 0, s, reinterpret_cast<const T *>(w), top, cin, cout, panels, \
                           chunks, total, packed);                                                                                  \
    } while (0)
    if (dtype == CG3D_DT_F32) I8_W(float);
    else if (dtype == CG3D_DT_BF16) I8_W(i8_bf16);
    else if (dtype == CG3D_DT_F16) I8_W(i8_f16);
    else
        hipLaunchKernelGGL((k_i8_weight_pack<int8_t>), dim3(nb), dim3(256), 0, s, reinterpret_cast<const int8_t *>(w), nullptr, cin, cout,
                           panels, chunks, total, packed);
#undef I8_W
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

// ---------------------------------------------------------------- rows
template <typename T> static __device__ __forceinline__ void i8_put_levels(int8_t *__restrict__ dst, int64_t k0, int64_t pitch, const i8_lev<T> &o) {
    constexpr int N = i8_els<T>;
    if (k0 + N <= pitch) {
        if constexpr (N == 4) *reinterpret_cast<i8_vec<uint32_t, 1> *>(dst + k0) = __builtin_bit_cast(i8_vec<uint32_t, 1>, o);
        else *reinterpret_cast<u32x2_any *>(dst + k0) = __builtin_bit_cast(u32x2_any, o);
    } else {
        const i8_vec<int8_t, N> b = __builtin_bit_cast(i8_vec<int8_t, N>, o);
#pragma unroll
        for (int j = 0; j < N - 1; j++)
            if (k0 + j < pitch) dst[k0 + j] = b.e[j];
    }
}
// L lanes (a power of two, at most a wave) own one row of at most L * KEEP pieces and hold it in registers: as few lanes as KEEP
// pieces of each allow (with 64 lanes and one piece 100 000 x 512 bf16 took 39.5 us, with 16 and four 26.7: 5.8 TB/s, the memory's)
template <typename T>
__global__ __launch_bounds__(256) void k_i8_rows(const T *__restrict__ x, int64_t n, int32_t cin, int64_t pitch, int32_t lshift,
                                                 int8_t *__restrict__ q, float *__restrict__ scale) {
    constexpr int N = i8_els<T>, KEEP = 4;
    const int L = 1 << lshift, lane = threadIdx.x & (L - 1);
    for (int64_t r = (blockIdx.x * 256ll + threadIdx.x) >> lshift; r < n; r += (gridDim.x * 256ll) >> lshift) {
        const T *row = x + r * cin;
        u32x4 v[KEEP];
        i8_max<T> most;
#pragma unroll
        for (int i = 0; i < KEEP; i++) v[i] = i8_piece<T>(row, (i * L + lane) * N, cin);
#pragma unroll
        for (int i = 0; i < KEEP; i++) most.add(v[i]);
        uint32_t top = most.bits();
        for (int d = L >> 1; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        const i8_level lev(top);
        if (lane == 0) scale[r] = lev.scale;
        int8_t *dst = q + r * pitch;
#pragma unroll
        for (int i = 0; i < KEEP; i++) {
            const int k0 = (i * L + lane) * N;
            if (k0 < pitch) i8_put_levels<T>(dst, k0, pitch, i8_levels<T>(lev, lev.shifted(), v[i]));
        }
        for (int64_t a = (int64_t)KEEP * L * N + lane; a < pitch; a += L) dst[a] = 0;
    }
}
// Longer rows, one to a workgroup of B threads; rows of more than B * KEEP pieces are read again for their levels.  Bound by memory
// and, with a barrier between a row's reads and its writes, by the rows that a CU has under way: B and KEEP by the row's length, and for
// 16-bit rows by how many there are (4000 rows of 10 976 fp32 49.9 us with 1024 threads of 4 pieces, 37.9 with 512 of 8 = 5.8 TB/s; 512 rows
// of 43 904: fp32 26.1 us with 1024 threads = 4.3 TB/s, 30.6 with 512, bf16 17.4 and 15.8; 100 rows 6.9 and 7.9).
template <typename T, int B, int KEEP>
__global__ __launch_bounds__(B) void k_i8_long_rows(const T *__restrict__ x, int64_t n, int32_t cin, int64_t pitch, int8_t *__restrict__ q,
                                                    float *__restrict__ scale) {
    constexpr int N = i8_els<T>;
    __shared__ uint32_t sh[B / 64];
    const int tid = threadIdx.x, step = B * KEEP * N;
    for (int64_t r = blockIdx.x; r < n; r += gridDim.x) {
        const T *row = x + r * cin;
        u32x4 v[KEEP];
        i8_max<T> most;
        for (int a = 0; a < cin; a += step) {
#pragma unroll
            for (int i = 0; i < KEEP; i++) v[i] = i8_piece<T>(row, a + (i * B + tid) * N, cin);
#pragma unroll
            for (int i = 0; i < KEEP; i++) most.add(v[i]);
        }
        uint32_t top = i8_max_of<64>(most.bits());
        if ((tid & 63) == 0) sh[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < B / 64; w++) top = max(top, sh[w]);
        __syncthreads();
        const i8_level lev(top);
        if (tid == 0) scale[r] = lev.scale;
        int8_t *dst = q + r * pitch;
        for (int64_t a = 0; a < pitch; a += step) {
            if (cin > step) {
#pragma unroll
                for (int i = 0; i < KEEP; i++) v[i] = i8_piece<T>(row, (int)a + (i * B + tid) * N, cin);
            }
#pragma unroll
            for (int i = 0; i < KEEP; i++) {
                const int64_t k0 = a + (i * B + tid) * N;
                if (k0 < pitch) i8_put_levels<T>(dst, k0, pitch, i8_levels<T>(lev, lev.shifted(), a < cin ? v[i] : u32x4{0, 0, 0, 0}));
            }
        }
    }
}
template <typename T>
static void i8_launch_rows(const T *x, int64_t n, int32_t cin, int64_t pitch, int8_t *q, float *scale, hipStream_t s) {
    constexpr int N = i8_els<T>, F = (int)sizeof(T) / 2;             // F: an fp32 row has twice the pieces
    const int32_t np = (cin + N - 1) / N;
    int32_t ls = 0;
    while ((4 << ls) < np && ls < 6) ls++;
    const int64_t waves = cg3d_divup(n << ls, 256);
    const dim3 gw((unsigned)(waves < (1 << 22) ? waves : (1 << 22))), gb((unsigned)(n < (1 << 20) ? n : (1 << 20)));
    if (np <= 256) hipLaunchKernelGGL((k_i8_rows<T>), gw, dim3(256), 0, s, x, n, cin, pitch, ls, q, scale);
    else if (cin <= 2048) hipLaunchKernelGGL((k_i8_long_rows<T, 128, 2 * F>), gb, dim3(128), 0, s, x, n, cin, pitch, q, scale);
    else if (cin <= 4096) hipLaunchKernelGGL((k_i8_long_rows<T, 256, 2 * F>), gb, dim3(256), 0, s, x, n, cin, pitch, q, scale);
    else if (cin <= 8192) hipLaunchKernelGGL((k_i8_long_rows<T, 512, 2 * F>), gb, dim3(512), 0, s, x, n, cin, pitch, q, scale);
    else if (cin <= 16384) hipLaunchKernelGGL((k_i8_long_rows<T, 512, 4 * F>), gb, dim3(512), 0, s, x, n, cin, pitch, q, scale);
    else {
        if constexpr (F == 1)
            if (n >= 512 && cin <= 512 * 12 * N) {
                hipLaunchKernelGGL((k_i8_long_rows<T, 512, 12>), gb, dim3(512), 0, s, x, n, cin, pitch, q, scale);
                return;
            }
        if (cin <= 32768) {                                          // (two workgroups fit a CU: 3000 x 20 000 fp32 71.9 -> 67.5 us)
            hipLaunchKernelGGL((k_i8_long_rows<T, 1024, 4 * F>), gb, dim3(1024), 0, s, x, n, cin, pitch, q, scale);
            return;
        }
        hipLaunchKernelGGL((k_i8_long_rows<T, 1024, 6 * F>), gb, dim3(1024), 0, s, x, n, cin, pitch, q, scale);
    }
}
extern "C" int cg3d_int8_quantize_rows(const void *x, int32_t dtype, int64_t n, int32_t cin, int64_t pitch, int8_t *q, float *scale,
                                       cg3d_stream_t stream) {
    if (dtype < CG3D_DT_F32 || dtype > CG3D_DT_F16 || n < 0 || cin < 1 || cin > I8_MAX_CIN || pitch < cin || pitch > (1 << 30)) return CG3D_ERR_ARG;
    if (n == 0) return CG3D_OK;
    if (!x || !q || !scale || ((uintptr_t)x & (dtype == CG3D_DT_F32 ? 3 : 1)) || ((uintptr_t)scale & 3)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
    if (dtype == CG3D_DT_F32) i8_launch_rows(reinterpret_cast<const float *>(x), n, cin, pitch, q, scale, s);
    else if (dtype == CG3D_DT_BF16) i8_launch_rows(reinterpret_cast<const i8_bf16 *>(x), n, cin, pitch, q, scale, s);
    else i8_launch_rows(reinterpret_cast<const i8_f16 *>(x), n, cin, pitch, q, scale, s);
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}

// ---------------------------------------------------------------- the product
struct i8_args {
    const float *sx;                 // row scales
    const int8_t *w;                 // fragments
    const float *sw, *bias;          // [E][cout], bias [E or 1][cout] or NULL
    const int32_t *offsets, *rows;   // grouped: the experts' rows, and the row of x that each of them reads (NULL: itself)
    void *y;
    int64_t n_rows, n_x;
    int32_t cin, cout, n_experts, out_dtype, bias_step;
};

// tile `u` of BM rows: the rows of one expert (grouped; expert n_experts: the rows behind the last, which are cleared).
// Ends of lists are clamped to the rows there are.  Returns false behind the last tile.
template <int BM>
static __device__ __forceinline__ bool i8_tile(const i8_args &a, int64_t u, int &e, int64_t &row0, int &rows) {
    if (!a.offsets) {
        e = 0;
        row0 = u * BM;
        rows = (int)min((int64_t)BM, a.n_rows - row0);
        return row0 < a.n_rows;
    }
    const int lane = threadIdx.x & 63;
    int64_t before = 0;
    for (int b = 0; b <= a.n_experts; b += 64) {
        const int g = b + lane;
        int64_t lo = 0, hi = 0;
        if (g <= a.n_experts) {
            lo = min(max((int64_t)a.offsets[g], (int64_t)0), a.n_rows);
            hi = g < a.n_experts ? min(max((int64_t)a.offsets[g + 1], lo), a.n_rows) : a.n_rows;
        }
        const int tiles = (int)(((uint32_t)(hi - lo) + (uint32_t)BM - 1) / (uint32_t)BM);
        int s = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s, d); if (lane >= d) s += o; }
        const uint64_t hit = __ballot(u < before + s);
        if (hit) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)hit) - 1);      // (uniform, and so is all that follows)
            const int64_t first = before + __builtin_amdgcn_readlane(s - tiles, l);
            const int64_t base = (int64_t)__builtin_amdgcn_readlane((int)lo, l), end = (int64_t)__builtin_amdgcn_readlane((int)hi, l);
            e = b + l;
            row0 = base + (u - first) * BM;
            rows = (int)min((int64_t)BM, end - row0);
            return true;
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return false;
}
static __device__ __forceinline__ int64_t i8_source(const i8_args &a, int64_t row) {
    const int64_t src = a.rows ? (int64_t)a.rows[row] : row;
    return (uint64_t)src < (uint64_t)a.n_x ? src : 0;
}
// N neighbouring channels from c0 of one expert: their scales and biases (zeros behind the last channel)
template <int N> struct i8_chan {
    i8_vec<float, N> s, b;
    __device__ __forceinline__ i8_chan(const i8_args &a, int e, int c0) : s{}, b{} {
        const float *sw = a.sw + (int64_t)e * a.cout + c0, *bias = a.bias + (int64_t)e * a.bias_step + c0;
        if (c0 + N <= a.cout) {
            s = *reinterpret_cast<const i8_vec<float, N> *>(sw);
            if (a.bias) b = *reinterpret_cast<const i8_vec<float, N> *>(bias);
        } else {
#pragma unroll
            for (int j = 0; j < N - 1; j++)
                if (c0 + j < a.cout) {
                    s.e[j] = sw[j];
                    if (a.bias) b.e[j] = bias[j];
                }
        }
    }
};
// Whether sum * sx may leave the normal range where the result does not: scales from 2^96 on (|sum| < 2^31) and subnormal ones (a sum
// that is not 0 is at least 1).  Such a scale is brought in by 2^64 and the result taken back: with any channel's scale in between, what
// then overflows or underflows does so in the result.  Decided once for the rows of a wave: one product more for all of them took
// 60 000 x 64 -> 1024 from 30.0 to 32.8 us, significands and exponents apart 31.8, a decision for each store of a large tile
// 52 000 x 576 -> 1024 from 76.8 to 80.5 us.
static __device__ __forceinline__ bool i8_is_far(float sx) {
    const float size = fabsf(sx);
    return size >= 0x1p96f || (size > 0.f && size < 0x1p-126f);
}
// a lane's N sums of one row, scaled, as many of them as there are channels left (n); far: one of the wave's rows may be (the same for
// all lanes); live = 0: a row behind the last.  to: where the workgroup's first lane would store (the same for all lanes), at: this lane's
// elements behind it
template <int N>
static __device__ __forceinline__ void i8_store(const i8_args &a, int64_t to, uint32_t at, int n, float sx, bool far, bool live, const i8_chan<N> &ch,
                                                const int (&sum)[N]) {
    i8_vec<float, N> v;
    if (far) {
        const float by = !i8_is_far(sx) ? 1.f : fabsf(sx) >= 1.f ? 0x1p-64f : 0x1p64f, back = 1.f / by;
#pragma unroll
        for (int j = 0; j < N; j++) v.e[j] = (float)sum[j] * (sx * by) * ch.s.e[j] * back;
    } else {
#pragma unroll
        for (int j = 0; j < N; j++) v.e[j] = (float)sum[j] * sx * ch.s.e[j];
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (a.bias) v.e[j] += ch.b.e[j];
        if (!live) v.e[j] = 0.f;
    }
    // (streamed past the caches like the rows of expert_rows.hip)
    if (a.out_dtype == CG3D_DT_F32) {
        float *y = reinterpret_cast<float *>(a.y) + to + at;
        if (n >= N) {
            if constexpr (N == 4) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4_any *>(y));
            else *reinterpret_cast<i8_vec<float, N> *>(y) = v;
        } else {
#pragma unroll
            for (int j = 0; j < N - 1; j++) if (j < n) y[j] = v.e[j];
        }
    } else {
        uint16_t *y = reinterpret_cast<uint16_t *>(a.y) + to + at;
        i8_vec<uint16_t, N> o;
        if (a.out_dtype == CG3D_DT_BF16) {
#pragma unroll
            for (int j = 0; j < N; j++) o.e[j] = __builtin_bit_cast(uint16_t, (__bf16)v.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) o.e[j] = __builtin_bit_cast(uint16_t, (_Float16)v.e[j]);
        }
        if (n >= N) {
            if constexpr (N == 4) __builtin_nontemporal_store(__builtin_bit_cast(u32x2_any, o), reinterpret_cast<u32x2_any *>(y));
            else *reinterpret_cast<i8_vec<uint16_t, N> *>(y) = o;
        } else {
#pragma unroll
            for (int j = 0; j < N - 1; j++) if (j < n) y[j] = o.e[j];
        }
    }
}
// a wave's results of 16 rows x one panel: acc[nb][i] of lane (g, m) is row 4 g + i, channel 4 m + nb; sx: of the lane's four rows
static __device__ __forceinline__ void i8_store_panel(const i8_args &a, int e, int panel, int64_t row0, int rows, const float (&sx)[4], bool far,
                                                      bool live, const i32x4 (&acc)[4]) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, c0 = panel * 64 + m * 4, n = a.cout - c0;
    if (n <= 0) return;
    const i8_chan<4> ch(a, live ? e : 0, c0);
    const uint32_t at = (uint32_t)(g * 4) * (uint32_t)a.cout + m * 4;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (g * 4 + i < rows) {
            const int sum[4] = {acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
            i8_store<4>(a, (row0 + i) * a.cout + panel * 64, at, n, sx[i], far, live, ch, sum);
        }
}
// the scales of the lane's four rows of 16
static __device__ __forceinline__ void i8_scales(const i8_args &a, int64_t row0, int rows, bool live, float (&sx)[4]) {
    const int g = (threadIdx.x & 63) >> 4;
    if (live && !a.rows && g * 4 + 4 <= rows) {
        const i8_vec<float, 4> s = *reinterpret_cast<const i8_vec<float, 4> *>(a.sx + row0 + g * 4);
#pragma unroll
        for (int i = 0; i < 4; i++) sx[i] = s.e[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) sx[i] = live && g * 4 + i < rows ? a.sx[i8_source(a, row0 + g * 4 + i)] : 0.f;
}
// where piece p (16 bytes) of row r lies in a fragment of 16 rows x 64 bytes of LDS: whole rows to write, and the 16 lanes that read
// one piece of every row touch every bank once
static __device__ __forceinline__ int i8_place(int r, int p) { return r * 64 + ((p ^ (r >> 2)) << 4); }

// Rows of at most I8_FUSED_CIN columns (many: I8_FUSED_LONG): one pass over them.  A workgroup of 4 waves owns 64 rows; each wave brings 16 of them in,
// neighbouring lanes neighbouring pieces (a chunk of a row is 4, 8 or 16 lanes, so a load of the wave is whole lines), finds their
// maxima over those lanes, and leaves their levels in LDS in the order of the MFMA's operand.  A level's divisions are done once for a
// row: of the NI rows that a lane has pieces of, lane l sees to row l % NI and its neighbours get the factor from it.  Then wave
// (wm, wn) multiplies RG of the 4 row groups by panels wn, wn + RG, ... of its part of the channels, the weights streaming past from the
// caches, every fragment used RG times.  RG = 4 / 2 / 1 for at least 4 / 2 / 1 panels a part.  The first `whole` tiles are one workgroup
// each, the panels of every other are shared out to `parts`.
// Bound by memory where panels are few: 155 773 x 64 fp32 -> 64, 80 MB, 15.3 us among others where the 256 MB memory-side cache still has
// the rows, 19.2 us = 4.2 TB/s with 600 MB of rows in turn.  With many panels by what a workgroup does one after the other -- rows in,
// products, results out --, which the three others of its CU overlap only in part: 82 107 x 512 bf16 -> 512 46 - 52 us, 54.6 from memory
// = 3.1 TB/s and 0.8 POP/s (31 us to read and write, 18 us to multiply).  The library's bf16 product of these sizes: 20.0 and 63.8 us.
template <typename T, int RG, int KEEP>                  // KEEP: chunks of a row held in registers; longer rows are read again, from the caches
__global__ __launch_bounds__(256, RG == 4 || KEEP * sizeof(T) > 8 ? 4 : RG == 2 ? 5 : 6) void k_i8_fused(i8_args a, const T *__restrict__ x, int32_t whole, int32_t parts) {
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_sm[];
    constexpr int NI = sizeof(T), LPR = 4 * NI, RPI = 64 / LPR, N = i8_els<T>;     // lanes of a row's chunk, rows of a load, elements of a piece
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int panels = (a.cout + 63) >> 6, chunks = (a.cin + 63) >> 6;
    const int late = (int)blockIdx.x - whole, tile = late < 0 ? blockIdx.x : whole + late / parts, part = late < 0 ? 0 : late % parts;
    const int of = late < 0 ? 1 : parts, p_lo = panels * part / of, p_hi = panels * (part + 1) / of;
    float *const scales = reinterpret_cast<float *>(i8_sm + chunks * 4096);        // [64], behind [4 groups][chunks][1 KB]
    int e, rows;
    int64_t row0;
    if (!i8_tile<64>(a, tile, e, row0, rows)) return;                              // (the whole workgroup)
    const bool live = e < a.n_experts;
    if (live && wave * 16 < rows) {
        const int rl = lane / LPR, k0 = (lane % LPR) * N;
        const T *xr[NI];
        uint8_t *to[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = i * RPI + rl;
            const int64_t src = i8_source(a, row0 + min(wave * 16 + r, rows - 1));
            xr[i] = x + src * a.cin;
            to[i] = i8_sm + wave * chunks * 1024 + i8_place(r, k0 >> 4) + (k0 & 15);
            if constexpr (NI == 1) {
                if (lane % LPR == 0) scales[wave * 16 + r] = a.sx[src];
            }
        }
        if constexpr (NI == 1) {
#pragma unroll 8
            for (int c = 0; c < chunks; c++) *reinterpret_cast<u32x4 *>(to[0] + c * 1024) = i8_piece<T>(xr[0], c * 64 + k0, a.cin);
        } else {
            u32x4 v[KEEP][NI];
            i8_max<T> most[NI];
            for (int c0 = 0; c0 < chunks; c0 += KEEP) {
#pragma unroll
                for (int c = 0; c < KEEP; c++)
                    if (c0 + c < chunks)
#pragma unroll
                        for (int i = 0; i < NI; i++) v[c][i] = i8_piece<T>(xr[i], (c0 + c) * 64 + k0, a.cin);
#pragma unroll
                for (int c = 0; c < KEEP; c++)
                    if (c0 + c < chunks)
#pragma unroll
                        for (int i = 0; i < NI; i++) most[i].add(v[c][i]);
            }
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const uint32_t t = i8_max_of<LPR>(most[i].bits());
                top = lane % NI == i ? t : top;
            }
            const i8_level mine(top);
            const bool far = __any(mine.shifted());
            if (lane % LPR < NI) scales[wave * 16 + (lane % NI) * RPI + rl] = mine.scale;
            i8_level lev[NI];
#pragma unroll
            for (int i = 0; i < NI; i++) {                                         // (lane i of each NI neighbours)
                lev[i] = mine;
                constexpr int ALL[4] = {NI == 2 ? 0xa0 : 0x00, NI == 2 ? 0xf5 : 0x55, 0xaa, 0xff};
                auto from = [&](uint32_t w) {
                    return i == 0 ? i8_dpp<ALL[0]>(w) : i == 1 ? i8_dpp<ALL[1]>(w) : i == 2 ? i8_dpp<ALL[2]>(w) : i8_dpp<ALL[3]>(w);
                };
                lev[i].c = __uint_as_float(from(__float_as_uint(mine.c)));
                lev[i].amax = __uint_as_float(from(__float_as_uint(mine.amax)));
                lev[i].shift = __uint_as_float(from(__float_as_uint(mine.shift)));
                lev[i].keep = from(mine.keep);
                lev[i].fine127 = from(mine.fine127) != 0;
            }
            for (int c0 = 0; c0 < chunks; c0 += KEEP) {
                if (chunks > KEEP) {
#pragma unroll
                    for (int c = 0; c < KEEP; c++)
                        if (c0 + c < chunks)
#pragma unroll
                            for (int i = 0; i < NI; i++) v[c][i] = i8_piece<T>(xr[i], (c0 + c) * 64 + k0, a.cin);
                }
#pragma unroll
                for (int c = 0; c < KEEP; c++)
                    if (c0 + c < chunks)
#pragma unroll
                        for (int i = 0; i < NI; i++)
                            *reinterpret_cast<i8_lev<T> *>(to[i] + (c0 + c) * 1024) = i8_levels<T>(lev[i], far, v[c][i]);
            }
        }
    }
    const int wn = wave % RG, wm = wave / RG;
    // the weights' fragments of the next chunk are asked for as soon as those of this one are used (two or four chunks ahead: no gain)
    const int8_t *const w_e = a.w + (int64_t)(live ? e : 0) * panels * (chunks * 4096);             // (uniform: an address for all lanes)
    i32x4 wq[4];
    if (p_lo + wn < p_hi)                                                          // (the first ones travel over the barrier)
#pragma unroll
        for (int nb = 0; nb < 4; nb++) wq[nb] = reinterpret_cast<const i32x4 *>(w_e + (int64_t)(p_lo + wn) * chunks * 4096 + nb * 1024)[lane];
    __syncthreads();
    if (wm * RG * 16 >= rows) return;
    const uint8_t *const bq = i8_sm + wm * RG * chunks * 1024 + i8_place(m, g);
    const bool far = __any(lane < RG * 16 && i8_is_far(scales[wm * RG * 16 + lane % (RG * 16)]));      // (of rows that there are not: old bytes)
    for (int p = p_lo + wn; p < p_hi; p += RG) {
        i32x4 acc[RG][4];
#pragma unroll
        for (int h = 0; h < RG; h++)
#pragma unroll
            for (int nb = 0; nb < 4; nb++) acc[h][nb] = i32x4{0, 0, 0, 0};
        const int here = p * chunks, then = (p + RG < p_hi ? p + RG : p) * chunks;
        for (int c = 0; c < chunks; c++) {
            if (live) {
#pragma unroll
                for (int h = 0; h < RG; h++) {
                    const i32x4 q = *reinterpret_cast<const i32x4 *>(bq + (h * chunks + c) * 1024);     // (a group without rows: old bytes, never stored)
#pragma unroll
                    for (int nb = 0; nb < 4; nb++) acc[h][nb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(q, wq[nb], acc[h][nb], 0, 0, 0);
                }
            }
            const int8_t *const wf = w_e + (int64_t)(c + 1 < chunks ? here + c + 1 : then) * 4096;
#pragma unroll
            for (int nb = 0; nb < 4; nb++) wq[nb] = reinterpret_cast<const i32x4 *>(wf + nb * 1024)[lane];
        }
#pragma unroll
        for (int h = 0; h < RG; h++) {
            const int r = (wm * RG + h) * 16;
            const i8_vec<float, 4> sx = *reinterpret_cast<const i8_vec<float, 4> *>(scales + r + g * 4);
            i8_store_panel(a, e, p, row0 + r, rows - r, sx.e, far, live, acc[h]);
        }
    }
}

// Few rows: a workgroup of 8 waves owns 16 rows x 32 channels (tiles nb of a pair) and its waves share the contraction (chunk c belongs
// to wave c % 8), so that every weight is read once, by loads that are all under way before the rows are even looked at.  Rows in
// floats that fit (CHUNKS chunks of a wave) are quantised here, in the operand's own layout -- each workgroup finds the rows' maxima for
// itself, through LDS; the waves' sums are joined there too.  grid: (16-row tiles, pairs of tiles).  KEEP: chunks of a wave held at once;
// registers for no more than there are let up to three workgroups onto a CU (8 experts of 640 -> 256, 1000 rows: 24.4 us with 8, 10.9 with 2).
// Bound by the weights' way from memory: 1 x 4096 bf16 -> 4096 8.2 us = 2.0 TB/s of weights that the memory-side cache holds, 9.5 us from
// memory (the library in bf16: 17.1) -- its 128 workgroups are on half of the CUs, and the other half reads nothing.  Small ones by a
// launch and two trips to memory: 1003 x 200 fp16 -> 77 5.5 us, 8 rows of 64 experts 512 -> 512 4.8 us.
template <typename T> struct i8_few { static constexpr int CHUNKS = sizeof(T) == 4 ? 4 : 8; };
template <typename T, int KEEP>
__global__ __launch_bounds__(512, KEEP == 1 || (KEEP == 2 && !__is_same(T, float) && !__is_same(T, i8_f16)) ? 6 : KEEP * sizeof(T) <= 8 ? 4 : 2) void k_i8_few(i8_args a, const T *__restrict__ x, int64_t pitch) {
    __shared__ i32x4 part[8][2][64];
    __shared__ uint32_t tops[8][16];
    __shared__ float scales[16];
    constexpr int NI = sizeof(T), N = i8_els<T>;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int panels = (a.cout + 63) >> 6, chunks = (a.cin + 63) >> 6, panel = blockIdx.y >> 1, pair = blockIdx.y & 1;
    int e, rows;
    int64_t row0;
    if (!i8_tile<16>(a, blockIdx.x, e, row0, rows)) return;      // (the whole workgroup)
    const bool live = e < a.n_experts;
    const int64_t src = live ? i8_source(a, row0 + min(m, rows - 1)) : 0;
    const T *xr = x + src * pitch;
    const i32x4 *wf = reinterpret_cast<const i32x4 *>(a.w) + (((int64_t)(live ? e : 0) * panels + panel) * chunks * 4 + pair * 2) * 64 + lane;
    i32x4 acc[2] = {i32x4{0, 0, 0, 0}, i32x4{0, 0, 0, 0}};
    float sx = 0.f;
    if (live) {
        if constexpr (NI == 1) sx = a.sx[src];
        for (int c0 = 0; c0 < chunks; c0 += 8 * KEEP) {          // (rows in floats: once)
            i32x4 w[KEEP][2];
            u32x4 v[KEEP][NI];
#pragma unroll
            for (int i = 0; i < KEEP; i++) {
                const int c = c0 + i * 8 + wave;
                if (c < chunks) {
#pragma unroll
                    for (int j = 0; j < NI; j++) v[i][j] = i8_piece<T>(xr, c * 64 + g * 16 + j * N, a.cin);
                    w[i][0] = wf[(int64_t)c * 256];
                    w[i][1] = wf[(int64_t)c * 256 + 64];
                }
            }
            i8_level lev(0);
            bool far = false;
            if constexpr (NI != 1) {
                i8_max<T> most;
#pragma unroll
                for (int i = 0; i < KEEP; i++)
                    if (i * 8 + wave < chunks)
#pragma unroll
                        for (int j = 0; j < NI; j++) most.add(v[i][j]);
                uint32_t top = most.bits();
                top = max(top, (uint32_t)__shfl_xor((int)top, 16));
                top = max(top, (uint32_t)__shfl_xor((int)top, 32));
                if (g == 0) tops[wave][m] = top;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; i++) top = max(top, tops[i][m]);
                lev = i8_level(top);
                far = __any(lev.shifted());
                sx = lev.scale;
            }
#pragma unroll
            for (int i = 0; i < KEEP; i++)
                if (c0 + i * 8 + wave < chunks) {
                    struct { i8_lev<T> p[NI]; } q;
#pragma unroll
                    for (int j = 0; j < NI; j++) q.p[j] = i8_levels<T>(lev, far, v[i][j]);
                    acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, q), w[i][0], acc[0], 0, 0, 0);
                    acc[1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, q), w[i][1], acc[1], 0, 0, 0);
                }
        }
    }
    part[wave][0][lane] = acc[0];
    part[wave][1][lane] = acc[1];
    if (wave == 0 && g == 0) scales[m] = sx;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 1; i < 8; i++) {
        acc[0] += part[i][0][lane];
        acc[1] += part[i][1][lane];
    }
    const bool far = __any(i8_is_far(scales[m]));                // (before lanes without channels leave: m is a row here)
    const int c0 = panel * 64 + m * 4 + pair * 2, n = a.cout - c0;
    if (n <= 0) return;
    const i8_chan<2> ch(a, live ? e : 0, c0);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (g * 4 + i < rows) {
            const int sum[2] = {acc[0][i], acc[1][i]};
            const uint32_t at = (uint32_t)(g * 4) * (uint32_t)a.cout + c0;
            i8_store<2>(a, (row0 + i) * a.cout, at, n, scales[g * 4 + i], far, live, ch, sum);
        }
}

// Many rows and a long contraction, rows in 8 bits (pitch and address multiples of 16): tiles of WR * RG * 16 rows x WC * 64 channels
// of WR * WC waves.  Both operands reach LDS by direct loads, three chunks of 64 contraction steps ahead of their use; a wave's
// fragments of the next chunk are read from LDS while it multiplies those of this one.  The weights' fragments are whole kilobytes
// in memory and in LDS.  16 rows' pieces of a chunk are another, piece p of row r in place r * 4 + (p ^ (r / 4)): four lanes fetch a
// row's 64 bytes and the reads of a fragment touch every bank once.  blockIdx.z: a range of chunks; with more than one the sums go to
// `part` (one i32x4 of a lane after the other, as the tile holds them) and k_i8_join adds them up.
// The direct loads and their waits are written out, since the compiler waits for ALL of them before any read of LDS: a wave has
// issued the NL loads of each chunk in order, so vmcnt(NL) leaves only the newest chunk's in flight.
// 4096 x 4096 x 4096, rows in 8 bits: 64 us = 2.1 POP/s, as the library's product of these sizes (68 us, 2.0 POP/s); the matrix unit is busy
// 47 % of the cycles.  A chunk is 1024 cycles of matrix instructions on each SIMD, 96 KB of fragments from LDS and 32 KB into it, and what
// raises the traffic costs time: 256 x 128 tiles with three buffers, two workgroups on a CU, 80 against 71 us in one run.  128 x 128 a wave
// with 4 waves would read a third less but does not fit the registers (354 us).  Rows whose chunks lie together in memory: no difference.
// 16 bytes of each lane to lds + 16 lane.  (M0 holds the address; the compiler uses it for nothing in a kernel without other such loads.)
static __device__ __forceinline__ void i8_dma(const void *src, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"((uint64_t)(uintptr_t)src), "s"(lds) : "memory");
}
template <int RG, int WR, int WC> static constexpr bool i8_in_parts = WR * RG * 16 == 128;      // (the larger tiles are for whole contractions)
template <int RG, int WR, int WC>
__global__ __launch_bounds__(WR * WC * 64, 2) void k_i8_tile(i8_args a, const int8_t *__restrict__ q, int64_t pitch, int32_t ny, i32x4 *__restrict__ part) {
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_sm[];
    constexpr int NW = WR * WC, BM = WR * RG * 16, NA = WC * 4, NB = WR * RG, NL = (NA + NB) / NW, STAGE = (NA + NB) * 1024, NBUF = 4;
    constexpr bool PARTS = i8_in_parts<RG, WR, WC>;
    static_assert((NA + NB) % NW == 0 && NA % NL == 0, "a wave's loads are of one operand");
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave % WR, wc = wave / WR;
    const int panels = (a.cout + 63) >> 6, chunks = (a.cin + 63) >> 6;
    // tiles of one XCD (workgroup index mod 8) are neighbours: they share rows and weights in its L2
    const int total = gridDim.x, per = total >> 3, left = total & 7, xcd = blockIdx.x & 7;
    const int id = xcd * per + min(xcd, left) + (blockIdx.x >> 3);
    const int by = id % ny;
    int e, rows;
    int64_t row0;
    if (!i8_tile<BM>(a, id / ny, e, row0, rows)) return;            // (the whole workgroup)
    const bool live = e < a.n_experts;
    const int c_lo = PARTS ? (int)((int64_t)chunks * blockIdx.z / gridDim.z) : 0, nc = PARTS ? (int)((int64_t)chunks * (blockIdx.z + 1) / gridDim.z) - c_lo : chunks;
    i32x4 acc[RG][4];
#pragma unroll
    for (int h = 0; h < RG; h++)
#pragma unroll
        for (int nb = 0; nb < 4; nb++) acc[h][nb] = i32x4{0, 0, 0, 0};
    // the scales of the wave's rows, a lane's share of them, looked at after the products
    float mine[(RG + 3) / 4];
#pragma unroll
    for (int h = 0; h < (RG + 3) / 4; h++) {
        const int r = wr * RG * 16 + h * 64 + lane;
        mine[h] = live && r < rows ? a.sx[i8_source(a, row0 + r)] : 0.f;
    }
    if (live && nc > 0) {
        // this wave's loads of a chunk: fragments [wave * NL, + NL) of the stage, the weights' first
        const uint8_t *src[NL];
        const bool of_a = wave * NL < NA;
        const int piece = (lane & 3) ^ (lane >> 4);
        const int last = (int)((a.cin + 15) & ~15) - 16;            // (no piece starts behind this one; what is read twice meets zeros)
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int f = wave * NL + i;
            if (of_a) {
                const int panel = min(by * WC + (f >> 2), panels - 1);
                src[i] = reinterpret_cast<const uint8_t *>(a.w) + ((((int64_t)e * panels + panel) * chunks + c_lo) * 4 + (f & 3)) * 1024 + lane * 16;
            } else {
                const int r = (f - NA) * 16 + (lane >> 2);
                src[i] = reinterpret_cast<const uint8_t *>(q) + i8_source(a, row0 + min(r, rows - 1)) * pitch;
            }
        }
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)i8_sm;
        // chunk min(k, nc - 1) into buffer k % NBUF: three more chunks are always under way than have been multiplied, past the end
        // the last one again, into a buffer that nobody reads
        auto issue = [&](int k) {
            const uint32_t to = base + (uint32_t)(k % NBUF) * STAGE + wave * NL * 1024;
            const int c = min(k, nc - 1);
#pragma unroll
            for (int i = 0; i < NL; i++)
                i8_dma(of_a ? src[i] + (int64_t)c * 4096 : src[i] + min((c_lo + c) * 64 + piece * 16, last), to + i * 1024);
        };
        const uint8_t *const la = i8_sm + wc * 4096 + lane * 16, *const lb = i8_sm + NA * 1024 + wr * RG * 1024 + i8_place(m, g);
        i32x4 fa[2][4], fb[2][RG];
        auto fetch = [&](int k, i32x4 (&A)[4], i32x4 (&B)[RG]) {
            const int at = (k % NBUF) * STAGE;
#pragma unroll
            for (int nb = 0; nb < 4; nb++) A[nb] = *reinterpret_cast<const i32x4 *>(la + at + nb * 1024);
#pragma unroll
            for (int h = 0; h < RG; h++) B[h] = *reinterpret_cast<const i32x4 *>(lb + at + h * 1024);
        };
        auto multiply = [&](const i32x4 (&A)[4], const i32x4 (&B)[RG]) {
#pragma unroll
            for (int h = 0; h < RG; h++)
#pragma unroll
                for (int nb = 0; nb < 4; nb++) acc[h][nb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(B[h], A[nb], acc[h][nb], 0, 0, 0);
        };
        auto step = [&](int k, i32x4 (&A)[4], i32x4 (&B)[RG], i32x4 (&nA)[4], i32x4 (&nB)[RG]) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(NL) : "memory");      // chunk k + 1 is in LDS, for every wave
            fetch(k + 1, nA, nB);
            issue(k + 3);                                           // (its buffer held chunk k - 1: read by every wave before this barrier)
            multiply(A, B);
        };
        issue(0);
        issue(1);
        issue(2);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(2 * NL) : "memory");
        fetch(0, fa[0], fb[0]);
        for (int k = 0; k < nc; k += 2) {
            step(k, fa[0], fb[0], fa[1], fb[1]);
            if (k + 1 < nc) step(k + 1, fa[1], fb[1], fa[0], fb[0]);
        }
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");          // (nothing may land in LDS after the workgroup has ended)
    }
    if (PARTS && gridDim.z > 1) {
        i32x4 *to = part + ((((int64_t)blockIdx.z * total + id) * NW + wave) * (RG * 4)) * 64 + lane;
#pragma unroll
        for (int h = 0; h < RG; h++)
            if ((wr * RG + h) * 16 < rows)                          // (a group without rows is not joined either)
#pragma unroll
                for (int nb = 0; nb < 4; nb++) to[(h * 4 + nb) * 64] = acc[h][nb];
        return;
    }
    const int panel = by * WC + wc;
    if (panel >= panels) return;
    bool far = false;
#pragma unroll
    for (int h = 0; h < (RG + 3) / 4; h++) far |= i8_is_far(mine[h]);
    far = __any(far);
#pragma unroll
    for (int h = 0; h < RG; h++) {
        const int r = (wr * RG + h) * 16;
        if (r >= rows) break;
        float sx[4];
        i8_scales(a, row0 + r, rows - r, live, sx);
        if (far) i8_store_panel(a, e, panel, row0 + r, rows - r, sx, true, live, acc[h]);
        else i8_store_panel(a, e, panel, row0 + r, rows - r, sx, false, live, acc[h]);
    }
}
// The sums of a tile's ranges of chunks: a workgroup owns 16 rows x 64 channels, its 8 waves share the ranges (one wave for all of
// them: 64 waves on the whole chip for 512 x 128 results, 18.7 us at 85 ranges; now 5.2 us at 64 = 3.3 TB/s of sums).
template <int RG, int WR, int WC>
__global__ __launch_bounds__(512) void k_i8_join(i8_args a, int32_t ny, int32_t total, int32_t splits, const i32x4 *__restrict__ part) {
    constexpr int NW = WR * WC, BM = WR * RG * 16;
    __shared__ i32x4 sum[8][4][64];
    const int lane = threadIdx.x & 63, me = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % RG, wave = blockIdx.x / RG % NW, id = blockIdx.x / (RG * NW);
    int e, rows;
    int64_t row0;
    if (!i8_tile<BM>(a, id / ny, e, row0, rows)) return;             // (the whole workgroup)
    const bool live = e < a.n_experts;
    const int wr = wave % WR, wc = wave / WR, panel = id % ny * WC + wc, r = (wr * RG + h) * 16;
    if (panel >= (a.cout + 63) >> 6 || r >= rows) return;
    i32x4 acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; nb++) acc[nb] = i32x4{0, 0, 0, 0};
    const int64_t next = (int64_t)total * NW * (RG * 4) * 64;
    const i32x4 *from = part + (((int64_t)id * NW + wave) * (RG * 4) + h * 4) * 64 + lane;
#pragma unroll 2
    for (int z = me; z < splits; z += 8)
#pragma unroll
        for (int nb = 0; nb < 4; nb++) acc[nb] += from[z * next + nb * 64];
#pragma unroll
    for (int nb = 0; nb < 4; nb++) sum[me][nb][lane] = acc[nb];
    __syncthreads();
    if (me != 0) return;
#pragma unroll
    for (int w = 1; w < 8; w++)
#pragma unroll
        for (int nb = 0; nb < 4; nb++) acc[nb] += sum[w][nb][lane];
    float sx[4];
    i8_scales(a, row0 + r, rows - r, live, sx);
    const bool far = __any(i8_is_far(sx[0]) || i8_is_far(sx[1]) || i8_is_far(sx[2]) || i8_is_far(sx[3]));
    i8_store_panel(a, e, panel, row0 + r, rows - r, sx, far, live, acc);
}

// rows of 8 bits whose pitch or address 16 does not divide: a copy with pitch i8_pitch
__global__ __launch_bounds__(256) void k_i8_pad(const int8_t *__restrict__ x, int64_t n, int32_t cin, int64_t pitch, int8_t *__restrict__ out) {
    const int nv = (int)(pitch >> 4);
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n * nv; i += gridDim.x * 256ll) {
        const int64_t r = i / nv;
        const int k0 = (int)(i - r * nv) * 16;
        *reinterpret_cast<u32x4 *>(out + r * pitch + k0) = i8_piece<int8_t>(x + r * cin, k0, cin);
    }
}

// ---------------------------------------------------------------- which kernel
struct i8_plan {
    enum { FUSED, FEW, TILE } kind;
    bool big;                        // TILE: 256 x 256 tiles, else 128 x 128
    bool rows8;                      // the rows are in 8 bits, in the workspace
    int32_t ny, splits;              // TILE: tiles along the channels, ranges of the contraction
    int64_t tiles, scale_at, part_at, bytes;
};
static int64_t i8_pitch(int32_t cin) { return i8_chunks(cin) * 64; }
static i8_plan i8_choose(int32_t dtype, int64_t n_x, int32_t cin, int64_t n_rows, int32_t cout, int32_t n_experts, bool grouped, bool padded) {
    i8_plan p = {};
    if (n_rows == 0) return p;                                       // (nothing is launched)
    const int64_t chunks = i8_chunks(cin), panels = i8_panels(cout);
    // (a list of rows has at most one tile that is not full, and only lists with rows have tiles: at most so many, and those of the rows
    // behind the last)
    const int64_t lists = n_experts < n_rows ? n_experts : n_rows;
    auto tiles = [&](int bm) { return grouped ? n_rows / bm + lists + 1 : cg3d_divup(n_rows, bm); };
    // The kernel for few rows: at most three workgroups a CU where the rows are short, else by its weights' fragments (half as many for
    // rows of fp32, which take it twice as long) against the rounds of 128 x 128 tiles, one to a CU, that the others would need.  Its
    // time against theirs, bf16: 512 -> 512, 500 rows (512 workgroups) 6.2 / 8.7 us, 1000 rows (1008) 8.5 / 8.9, 2000 rows 12.6 / 9.3;
    // 128 -> 128, 2000 rows (504) 5.4 / 6.0, 4000 rows (1004) 6.8 / 6.1; 18 experts of it, 2000 rows (572) 6.5 / 6.8.  1024 -> 1024, 500
    // rows 10.8 / 16.7, 1000 rows (32 256 fragments) 17.5 / 16.8 (fp32, 500 rows 15.8 / 16.8); 2048 -> 2048, 250 rows (32 768) 17.1 / 21.2 (fp32,
    // 128 rows 17.6 / 21.1); 18 experts of 1024 -> 1024, 512 rows (25 600) 16.1 / 17.2, 1200 rows (47 616) 27.9 / 20.8; 64 experts of it, 64
    // rows (35 328, 2 rounds) 16.4 / 38.6, 1000 rows (64 512) 31.6 / 40.8, 2000 rows (96 768) 49.4 / 45.8.  Of very long rows each would read
    // too much by itself (512 x 43 904 -> 128: 38 us against 18).
    const int64_t few = (n_rows / 16 + (grouped ? lists : 1)) * panels * 2, rounds256 = tiles(128) * cg3d_divup(panels, 2);
    const int64_t most_few = (dtype == CG3D_DT_F32 ? 16500 : 33000) * (rounds256 > 256 ? rounds256 : 256) / 256;
    if (cin <= I8_FUSED_CIN ? few <= 768 : chunks <= 128 && (few <= 384 || few * chunks <= most_few)) {
        p.kind = i8_plan::FEW;
        p.tiles = tiles(16);
        p.rows8 = dtype != CG3D_DT_I8 && chunks > 8 * (dtype == CG3D_DT_F32 ? i8_few<float>::CHUNKS : i8_few<i8_bf16>::CHUNKS);
    } else if (cin <= I8_FUSED_CIN || (cin <= I8_FUSED_LONG && n_rows >= 20000 && (dtype == CG3D_DT_BF16 || dtype == CG3D_DT_F16))) {
        // (longer rows lose what quantising them in the product gains, to fewer workgroups on a CU: bf16, 30 000 rows 704 -> 128 20.7 us
        // against 26.0 in two passes, 704 -> 512 33.4 / 36.6, 832 -> 512 38.1 / 39.9, 960 -> 512 42.0 / 42.9; 82 107 rows 576 -> 64 36.6 / 52.1,
        // 960 -> 128 68.1 / 65.6; 10 000 rows 704 -> 512 25.3 / 22.3; fp32, 30 000 rows 704 -> 128 34.6 / 31.2)
        p.kind = i8_plan::FUSED;
        p.tiles = tiles(64);
    } else {
        p.kind = i8_plan::TILE;
        p.rows8 = dtype != CG3D_DT_I8 || padded;
        // a round of 256 x 256 tiles nearly full; with one or two panels half of each is empty (82 107 x 576 -> 64 39.6 us against 22.8)
        p.big = panels > 2 && tiles(256) * cg3d_divup(panels, 4) >= 200;
        p.ny = (int32_t)cg3d_divup(panels, p.big ? 4 : 2);
        p.tiles = tiles(p.big ? 256 : 128);
        const int64_t total = p.tiles * p.ny;
        p.splits = 1;
        if (!p.big && chunks > 32) {
            // The contraction is shared out while that fills CUs that have no tile, at 16 chunks or more.  Tile + join, rows in 8 bits: 4096 ->
            // 4096, 100 rows (32 tiles) 16.9 us in 4 parts, 19.0 in 2; 43 904 -> 128, 512 rows 18.0 us in 64, 19.5 in 21.  With 32 chunks or
            // fewer the join takes what the parts save: 2048 -> 2048, 1000 rows (128 tiles) 22.1 us in 2 parts, 18.4 in one; 1024 -> 1024, 2000
            // rows 23.0 and 13.0.
            const int64_t want = 256 / total, most = chunks / 16;
            p.splits = (int32_t)(want < 1 ? 1 : want < most ? want : most);
        }
    }
    int64_t at = 0;
    if (p.rows8) {
        p.scale_at = n_x * i8_pitch(cin);
        at = p.scale_at + ((n_x * 4 + 255) & ~255ll);
    }
    if (p.kind == i8_plan::TILE && p.splits > 1) {
        p.part_at = at;
        at += p.splits * p.tiles * p.ny * (128 * 128 * 4);
    }
    p.bytes = at;
    return p;
}
extern "C" int64_t cg3d_int8_linear_ws_bytes(int32_t dtype, int64_t n_x, int32_t cin, int64_t n_rows, int32_t cout, int32_t n_experts, int32_t flags) {
    if (dtype < CG3D_DT_F32 || dtype > CG3D_DT_I8 || i8_bad_shape(n_experts, cin, cout) || n_x < 0 || n_x > 0x7fffffffll || n_rows < 0 ||
        n_rows > 0x7fffffffll || (flags & ~3))
        return CG3D_ERR_ARG;
    return i8_choose(dtype, n_x, cin, n_rows, cout, n_experts, flags & 1, (cin & 15) || !(flags & 2)).bytes;
}
extern "C" int cg3d_int8_linear(const void *x, int32_t dtype, const float *sx, int64_t n_x, int32_t cin, const int8_t *w, const float *sw,
                                const float *bias, int32_t bias_per_expert, const int32_t *offsets, const int32_t *rows, void *y,
                                int32_t out_dtype, int64_t n_rows, int32_t cout, int32_t n_experts, void *ws, cg3d_stream_t stream) {
    const bool padded = (cin & 15) || ((uintptr_t)x & 15);
    const int64_t need = cg3d_int8_linear_ws_bytes(dtype, n_x, cin, n_rows, cout, n_experts, (offsets ? 1 : 0) | (padded ? 0 : 2));
    if (need < 0 || out_dtype < CG3D_DT_F32 || out_dtype > CG3D_DT_F16 || (bias_per_expert != 0 && bias_per_expert != 1)) return CG3D_ERR_ARG;
    if (offsets ? (!rows && n_x != n_rows) : (rows || n_x != n_rows || n_experts != 1)) return CG3D_ERR_ARG;
    if (n_rows == 0) return CG3D_OK;
    if (n_x == 0 || !x || !w || !sw || !y || (dtype == CG3D_DT_I8 && !sx) || (need > 0 && !ws)) return CG3D_ERR_ARG;
    if (((uintptr_t)x & (dtype == CG3D_DT_F32 ? 3 : dtype == CG3D_DT_I8 ? 0 : 1)) || ((uintptr_t)w & 15) || ((uintptr_t)y & (out_dtype == CG3D_DT_F32 ? 3 : 1)) ||
        (((uintptr_t)sx | (uintptr_t)sw | (uintptr_t)bias | (uintptr_t)offsets | (uintptr_t)rows) & 3) || ((uintptr_t)ws & 15))
        return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
    const i8_plan p = i8_choose(dtype, n_x, cin, n_rows, cout, n_experts, offsets != nullptr, padded);
    const int64_t panels = i8_panels(cout);
    if (p.tiles >= (1ll << 24) || (p.kind == i8_plan::TILE && p.tiles * p.ny >= (p.big ? 1ll << 23 : 1ll << 24))) return CG3D_ERR_ARG;      // (2^32 threads of a launch)
    i8_args a = {sx, w, sw, bias, offsets, rows, y, n_rows, n_x, cin, cout, n_experts, out_dtype, bias_per_expert ? cout : 0};
    const int8_t *q = reinterpret_cast<const int8_t *>(x);
    int64_t pitch = cin;
    if (p.rows8) {
        int8_t *lev = reinterpret_cast<int8_t *>(ws);
        pitch = i8_pitch(cin);
        if (dtype == CG3D_DT_I8) {
            const int64_t nb = cg3d_divup(n_x * (pitch / 16), 256);
            hipLaunchKernelGGL(k_i8_pad, dim3((unsigned)(nb < (1 << 22) ? nb : (1 << 22))), dim3(256), 0, s, q, n_x, cin, pitch, lev);
            CG3D_CHECK_LAUNCH();
        } else {
            float *scale = reinterpret_cast<float *>(lev + p.scale_at);
            const int rc = cg3d_int8_quantize_rows(x, dtype, n_x, cin, pitch, lev, scale, stream);
            if (rc != CG3D_OK) return rc;
            a.sx = scale;
            dtype = CG3D_DT_I8;
        }
        q = lev;
        x = lev;
    }
    if (p.kind == i8_plan::FEW) {
        const dim3 grid((unsigned)p.tiles, (unsigned)(panels * 2));      // (at most 2^15)
        if (p.rows8) a.cin = (int32_t)pitch;                         // (zeros behind the row: whole pieces)
        const int64_t each = cg3d_divup(i8_chunks(a.cin), 8);        // chunks of a wave
#define I8_FEW(T, KEEP) hipLaunchKernelGGL((k_i8_few<T, KEEP>), grid, dim3(512), 0, s, a, reinterpret_cast<const T *>(x), pitch)
#define I8_FEW_K(T) do { if (each <= 1) I8_FEW(T, 1); else if (each <= 2) I8_FEW(T, 2); else if (each <= 4) I8_FEW(T, 4); else I8_FEW(T, 8); } while (0)
        if (dtype == CG3D_DT_F32) { if (each <= 1) I8_FEW(float, 1); else if (each <= 2) I8_FEW(float, 2); else I8_FEW(float, 4); }
        else if (dtype == CG3D_DT_BF16) I8_FEW_K(i8_bf16);
        else if (dtype == CG3D_DT_F16) I8_FEW_K(i8_f16);
        else I8_FEW_K(int8_t);
#undef I8_FEW_K
#undef I8_FEW
        CG3D_CHECK_LAUNCH();
        return CG3D_OK;
    }
    if (p.kind == i8_plan::FUSED) {
        // enough workgroups for the chip: the panels of a row tile are shared out where there are fewer than 384 tiles, though each part
        // quantises the rows for itself (512 -> 512, 10 000 rows: 20.6 / 16.4 / 18.3 / 16.9 / 25.4 us at 128 / 256 / 384 / 512 / 1024
        // wanted, 20 000 rows 24.7 / 24.5 / 22.0 / 21.9 / 27.9; 512 -> 2048, 5000 rows 33.4 / 22.7 / 23.9 / 26.8 / 26.0)
        int64_t whole = 0, parts = cg3d_divup(384, p.tiles);
        parts = parts < panels ? parts : panels;
        const int32_t each = (int32_t)cg3d_divup(panels, parts);
        // and those of the last few tiles behind whole rounds of the chip -- four workgroups a CU, or the three that the levels of more than
        // 576 columns leave room for --, four panels or more to a part: 512 -> 512, 73 728 rows (128 tiles of 1152) 49.0 -> 44.9 us, 82 107
        // rows (259 of 1283) 52.3 -> 50.9; 256 -> 2048, 82 107 rows 118.9 -> 105.4; with 512 tiles left it loses (98 304 rows 55.4 -> 58.3).
        // Rounds of three: 704 -> 1024, 51 712 rows (40 tiles of 808) 91.7 -> 72.8, 64 512 rows (240 of 1008) 97.1 -> 93.6; 832 -> 512, 58 752
        // rows (150 of 918) 67.7 -> 66.5; with 300 left 704 -> 1024 102.1 -> 106.6
        const int64_t round = i8_chunks(cin) <= 9 ? 1024 : 768, late = p.tiles % round;
        if (p.tiles > round && late > 0 && late <= (round == 1024 ? 384 : 240) && panels >= 8) {
            whole = p.tiles - late;
            parts = cg3d_divup(768, late);
            parts = parts < panels / 4 ? parts : panels / 4;
        }
        const int64_t blocks = whole + (p.tiles - whole) * parts;
        const int lds = (int)i8_chunks(cin) * 4096 + 256;           // (at most 52.25 KB)
#define I8_F(T, RG, KEEP) hipLaunchKernelGGL((k_i8_fused<T, RG, KEEP>), dim3((unsigned)blocks), dim3(256), lds, s, a, reinterpret_cast<const T *>(x), (int32_t)whole, (int32_t)parts)
#define I8_FK(T, RG) do { if (chunks <= 1) I8_F(T, RG, 1); else if (chunks <= 2) I8_F(T, RG, 2); else I8_F(T, RG, (sizeof(T) == 4 ? 4 : 8)); } while (0)
#define I8_FC(T) do { if (each >= 4) I8_FK(T, 4); else if (each >= 2) I8_FK(T, 2); else I8_FK(T, 1); } while (0)
        const int64_t chunks = i8_chunks(cin);
        if (dtype == CG3D_DT_F32) I8_FC(float);
        else if (dtype == CG3D_DT_BF16) I8_FC(i8_bf16);
        else if (dtype == CG3D_DT_F16) I8_FC(i8_f16);
        else if (each >= 4) I8_F(int8_t, 4, 1);
        else if (each >= 2) I8_F(int8_t, 2, 1);
        else I8_F(int8_t, 1, 1);
#undef I8_FK
#undef I8_FC
#undef I8_F
        CG3D_CHECK_LAUNCH();
        return CG3D_OK;
    }
    if (p.rows8) a.cin = (int32_t)pitch;
    i32x4 *part = p.splits > 1 ? reinterpret_cast<i32x4 *>(reinterpret_cast<int8_t *>(ws) + p.part_at) : nullptr;
    const int32_t total = (int32_t)(p.tiles * p.ny);
#define I8_T(RG, WR, WC)                                                                                                            \
    do {                                                                                                                            \
        constexpr int lds = 4 * (WC * 4 + WR * RG) * 1024;                                                                          \
        if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(&k_i8_tile<RG, WR, WC>), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) \
            return CG3D_ERR_LAUNCH;                                                                                                 \
        hipLaunchKernelGGL((k_i8_tile<RG, WR, WC>), dim3((unsigned)total, 1, (unsigned)p.splits), dim3(WR * WC * 64), lds, s, a, q, pitch, p.ny, part); \
        CG3D_CHECK_LAUNCH();                                                                                                        \
    } while (0)
    if (p.big) I8_T(8, 2, 4);
    else {
        I8_T(4, 2, 2);
        if (part) {
            hipLaunchKernelGGL((k_i8_join<4, 2, 2>), dim3((unsigned)(total * 16)), dim3(512), 0, s, a, p.ny, total, p.splits, part);
            CG3D_CHECK_LAUNCH();
        }
    }
#undef I8_T
    return CG3D_OK;
}
