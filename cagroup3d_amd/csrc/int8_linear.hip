// int8_linear.hip -- Y = (Q @ W) * sx * sw + b in 8-bit integers with a scale for each row and each output channel (gfx950), dense or
// with a matrix of its own for each expert's rows, and the quantisation of rows and weights.
//
//   y[r, n] = (sum_k q[r, k] w[k, n]) * sx[r] * sw[n] + b[n]      the sum is exact: int32, fewer than 2^17 terms of at most 2^14
//   sx[r]   = max_k |x[r, k]| / 127,   q[r, k] = 127 x[r, k] / max |x[r, .]| rounded to the nearest, ties to even
//
// The rounding of q is decided exactly, not up to the error of a reciprocal: t = x * (127 / max) in fp32 is off by less than 2^-15,
// and where it falls within 2^-13 of a half the two sides 254 |x| and (2 n + 1) max are compared in 64 bits, where both are exact.
// A row that holds an infinity or a NaN gets the scale NaN (and so a row of NaN as its result); a row of zeros the scale 0.
//
// The weights are the MFMA's A operand and the rows its B operand (v_mfma_i32_16x16x64_i8), i.e. a tile of the product is
// D[channel][row]: a lane then holds neighbouring channels of ONE row, its row scale is one register, and the result leaves in
// 16-byte stores without a detour through LDS.  Weights are laid out once (cg3d_int8_weight): [expert][panel of 64 channels][chunk
// of 64 contraction steps][tile nb of 4][lane][16 bytes]; lane (g = lane / 16, m = lane % 16) holds contraction steps
// 16 g .. 16 g + 15 of the channel (nb / 2) * 32 + (m / 4) * 8 + (nb % 2) * 4 + m % 4 of the panel, so that the results of tiles nb = 0, 1
// (2, 3) in a lane are 8 consecutive channels.  Channels and contraction steps past the end are zeros.
#include "cg3d_common.h"

typedef int i32x4 __attribute__((ext_vector_type(4)));

#define I8_MAX_CIN 131071            // 2^14 * 131071 < 2^31: -128 * -128 included
#define I8_MAX_EXPERTS 1024

template <typename T, int V> struct __attribute__((packed, aligned(1))) i8_vec { T e[V]; };

struct i8_bf16 { uint16_t v; };
struct i8_f16 { uint16_t v; };
static __device__ __forceinline__ float i8_f(float a) { return a; }
static __device__ __forceinline__ float i8_f(i8_bf16 a) { return __uint_as_float((uint32_t)a.v << 16); }
static __device__ __forceinline__ float i8_f(i8_f16 a) { return (float)__builtin_bit_cast(_Float16, a.v); }
static __device__ __forceinline__ uint32_t i8_abs(float f) { return __float_as_uint(f) & 0x7fffffffu; }   // ordered like |f|; infinity and NaN on top

// what a row's largest magnitude (bits of |.|) makes of its elements: q = level(x), scale
struct i8_level {
    float amax, inv, up, scale;
    __device__ __forceinline__ explicit i8_level(uint32_t top) {
        const float a = __uint_as_float(top);
        const bool fine = top < 0x7f800000u;
        up = a < 0x1p-96f ? 0x1p96f : 1.f;               // (an exact shift of the whole row, so that 127 / max stays finite)
        amax = fine ? a * up : 0.f;
        inv = amax > 0.f ? 127.f / amax : 0.f;
        scale = fine ? a / 127.f : __uint_as_float(0x7fc00000u);
        if (!fine) up = 0.f;
    }
    __device__ __forceinline__ int operator()(float x) const {
        if (amax == 0.f) return 0;
        const float t = x * up * inv;
        const float n = rintf(t);
        if (__builtin_expect(fabsf(t - n) > 0.5f - 0x1p-13f, 0)) {
            const int lo = (int)floorf(fabsf(t));
            const double a = fabs((double)x * (double)up) * 254.0, b = (double)(2 * lo + 1) * (double)amax;
            const int m = a > b || (a == b && (lo & 1)) ? lo + 1 : lo;
            return t < 0.f ? -m : m;
        }
        return (int)n;
    }
};

// ---------------------------------------------------------------- weights (once per model)
// w [E][cin][cout]: a thread owns a channel, reads along the contraction are rows of the matrix
template <typename T>
__global__ __launch_bounds__(256) void k_i8_weight_scale(const T *__restrict__ w, int32_t cin, int32_t cout, float *__restrict__ scale,
                                                         uint32_t *__restrict__ top) {
    const int n = blockIdx.x * 256 + threadIdx.x, e = blockIdx.y;
    if (n >= cout) return;
    const T *p = w + (int64_t)e * cin * cout + n;
    uint32_t m = 0;
    for (int k = 0; k < cin; k++) m = max(m, i8_abs(i8_f(p[(int64_t)k * cout])));
    scale[(int64_t)e * cout + n] = i8_level(m).scale;
    top[(int64_t)e * cout + n] = m;
}
static __device__ __forceinline__ int i8_channel(int nb, int m) { return (nb >> 1) * 32 + (m >> 2) * 8 + (nb & 1) * 4 + (m & 3); }

// a thread writes the 16 bytes of one lane of one fragment (top == NULL: w is in 8 bits already)
template <typename T>
__global__ __launch_bounds__(256) void k_i8_weight_pack(const T *__restrict__ w, const uint32_t *__restrict__ top, int32_t cin, int32_t cout,
                                                        int32_t panels, int32_t chunks, int64_t total, int8_t *__restrict__ out) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int lane = (int)(i & 63), nb = (int)((i >> 6) & 3);
        const int64_t u = i >> 8;
        const int c = (int)(u % chunks), p = (int)((u / chunks) % panels), e = (int)(u / chunks / panels);
        const int n = p * 64 + i8_channel(nb, lane & 15), k0 = c * 64 + (lane >> 4) * 16;
        union { int8_t b[16]; i32x4 v; } o;
        o.v = i32x4{0, 0, 0, 0};
        if (n < cout) {
            const T *src = w + (int64_t)e * cin * cout + n;
            if constexpr (sizeof(T) == 1) {
                for (int j = 0; j < 16; j++)
                    if (k0 + j < cin) o.b[j] = (int8_t)src[(int64_t)(k0 + j) * cout];
            } else {
                const i8_level q(top[(int64_t)e * cout + n]);
                for (int j = 0; j < 16; j++)
                    if (k0 + j < cin) o.b[j] = (int8_t)q(i8_f(src[(int64_t)(k0 + j) * cout]));
            }
        }
        reinterpret_cast<i32x4 *>(out)[i] = o.v;
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
        hipLaunchKernelGGL((k_i8_weight_scale<T>), dim3((unsigned)cg3d_divup(cout, 256), (unsigned)n_experts), dim3(256), 0, s,     \
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
// A group of L lanes (a power of two) owns one row, 16 elements of a lane at a time; the row is read a second time (from the
// caches) for its levels.  Bytes [cin, pitch) are zeros.
template <typename T>
static __device__ __forceinline__ void i8_load16(const T *__restrict__ p, int left, float (&f)[16]) {   // left: elements before the row's end
    if (left >= 16) {
        const i8_vec<T, 16> v = *reinterpret_cast<const i8_vec<T, 16> *>(p);
#pragma unroll
        for (int j = 0; j < 16; j++) f[j] = i8_f(v.e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) f[j] = j < left ? i8_f(p[j]) : 0.f;
    }
}
template <typename T, int B>
__global__ __launch_bounds__(B) void k_i8_rows(const T *__restrict__ x, int64_t n, int32_t cin, int64_t pitch, int32_t lshift,
                                               int8_t *__restrict__ q, float *__restrict__ scale) {
    __shared__ uint32_t sh[B / 64];
    const int L = 1 << lshift, lane = threadIdx.x & (L - 1);
    const int nv = (cin + 15) >> 4;
    for (int64_t r = (blockIdx.x * (int64_t)B + threadIdx.x) >> lshift; r < n; r += ((int64_t)gridDim.x * B) >> lshift) {
        const T *row = x + r * cin;
        uint32_t top = 0;
        float f[16];
        for (int v = lane; v < nv; v += L) {
            i8_load16(row + v * 16, cin - v * 16, f);
#pragma unroll
            for (int j = 0; j < 16; j++) top = max(top, i8_abs(f[j]));
        }
        for (int d = (L < 64 ? L : 64) >> 1; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
        if (L > 64) {                                     // (L == B: the workgroup owns the row)
            if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < B / 64; w++) top = max(top, sh[w]);
            __syncthreads();
        }
        const i8_level lev(top);
        if (lane == 0) scale[r] = lev.scale;
        int8_t *dst = q + r * pitch;
        for (int v = lane; v < nv; v += L) {
            i8_load16(row + v * 16, cin - v * 16, f);
            i8_vec<int8_t, 16> o;
#pragma unroll
            for (int j = 0; j < 16; j++) o.e[j] = (int8_t)lev(f[j]);
            if (v * 16 + 16 <= pitch) *reinterpret_cast<i8_vec<int8_t, 16> *>(dst + v * 16) = o;
            else
                for (int j = 0; j < 16; j++)
                    if (v * 16 + j < pitch) dst[v * 16 + j] = o.e[j];
        }
        for (int64_t a = nv * 16ll + lane; a < pitch; a += L) dst[a] = 0;
    }
}
extern "C" int cg3d_int8_quantize_rows(const void *x, int32_t dtype, int64_t n, int32_t cin, int64_t pitch, int8_t *q, float *scale,
                                       cg3d_stream_t stream) {
    if (dtype < CG3D_DT_F32 || dtype > CG3D_DT_F16 || n < 0 || cin < 1 || cin > I8_MAX_CIN || pitch < cin) return CG3D_ERR_ARG;
    if (n == 0) return CG3D_OK;
    if (!x || !q || !scale || ((uintptr_t)x & (dtype == CG3D_DT_F32 ? 3 : 1)) || ((uintptr_t)scale & 3)) return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
    int32_t ls = 0;
    const int32_t nv = (cin + 15) / 16;
    while ((1 << ls) < nv && ls < 6) ls++;
    if (nv > 4 * 64) ls = 8;                              // a long row: the whole workgroup
    int64_t nb = cg3d_divup(n << ls, 256);
    if (nb > (1 << 22)) nb = 1 << 22;
    if (dtype == CG3D_DT_F32) hipLaunchKernelGGL((k_i8_rows<float, 256>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const float *>(x), n, cin, pitch, ls, q, scale);
    else if (dtype == CG3D_DT_BF16) hipLaunchKernelGGL((k_i8_rows<i8_bf16, 256>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const i8_bf16 *>(x), n, cin, pitch, ls, q, scale);
    else hipLaunchKernelGGL((k_i8_rows<i8_f16, 256>), dim3((unsigned)nb), dim3(256), 0, s, reinterpret_cast<const i8_f16 *>(x), n, cin, pitch, ls, q, scale);
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
        const int tiles = (int)((hi - lo + BM - 1) / BM);
        int s = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(s, d); if (lane >= d) s += o; }
        const uint64_t hit = __ballot(u < before + s);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            const int64_t first = before + __shfl(s - tiles, l);
            const int64_t base = (int64_t)__shfl((int)lo, l), end = (int64_t)__shfl((int)hi, l);
            e = b + l;
            row0 = base + (u - first) * BM;
            rows = (int)min((int64_t)BM, end - row0);
            return true;
        }
        before += __shfl(s, 63);
    }
    return false;
}
static int64_t i8_tiles(const i8_args &a, int bm) { return a.offsets ? a.n_rows / bm + a.n_experts + 1 : cg3d_divup(a.n_rows, bm); }

// a lane's results of one panel, acc[nb][i]: channels i8_channel(nb, 4 g + i) of row `row`; live = 0: rows behind the last
static __device__ __forceinline__ void i8_store(const i8_args &a, int e, int panel, int64_t row, float sx, bool live, const i32x4 (&acc)[4]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int c0 = panel * 64 + h * 32 + g * 8;
        if (c0 >= a.cout) continue;
        const bool whole = c0 + 8 <= a.cout;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int c = whole || c0 + j < a.cout ? c0 + j : a.cout - 1;
            v[j] = 0.f;
            if (live) {
                v[j] = (float)acc[2 * h + (j >> 2)][j & 3] * sx * a.sw[(int64_t)e * a.cout + c];
                if (a.bias) v[j] += a.bias[(int64_t)e * a.bias_step + c];
            }
        }
        if (a.out_dtype == CG3D_DT_F32) {
            float *y = reinterpret_cast<float *>(a.y) + row * a.cout + c0;
            if (whole) {
                i8_vec<float, 8> o;
#pragma unroll
                for (int j = 0; j < 8; j++) o.e[j] = v[j];
                *reinterpret_cast<i8_vec<float, 8> *>(y) = o;
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) if (c0 + j < a.cout) y[j] = v[j];
            }
        } else {
            uint16_t *y = reinterpret_cast<uint16_t *>(a.y) + row * a.cout + c0;
            i8_vec<uint16_t, 8> o;
#pragma unroll
            for (int j = 0; j < 8; j++)
                o.e[j] = a.out_dtype == CG3D_DT_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v[j]) : __builtin_bit_cast(uint16_t, (_Float16)v[j]);
            if (whole) *reinterpret_cast<i8_vec<uint16_t, 8> *>(y) = o;
            else {
#pragma unroll
                for (int j = 0; j < 8; j++) if (c0 + j < a.cout) y[j] = o.e[j];
            }
        }
    }
}

// The plainest form: a wave owns 16 rows x 64 channels, operands straight from memory (the fragments of the weights are whole
// kilobytes, a row's 64 bytes of a chunk belong to four lanes).
static __device__ __forceinline__ i32x4 i8_row16(const int8_t *__restrict__ p, int left) {
    if (left >= 16) return __builtin_bit_cast(i32x4, *reinterpret_cast<const i8_vec<int8_t, 16> *>(p));
    i8_vec<int8_t, 16> o;
#pragma unroll
    for (int j = 0; j < 16; j++) o.e[j] = j < left ? p[j] : 0;
    return __builtin_bit_cast(i32x4, o);
}
__global__ __launch_bounds__(256) void k_i8_wave(i8_args a, const int8_t *__restrict__ q, int64_t pitch) {
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int panels = (a.cout + 63) >> 6, chunks = (a.cin + 63) >> 6;
    const int64_t u = blockIdx.x * 4ll + (threadIdx.x >> 6);
    const int panel = (int)(u % panels);
    int e, rows;
    int64_t row0;
    if (!i8_tile<16>(a, u / panels, e, row0, rows)) return;
    const bool live = e < a.n_experts;
    const bool mine = m < rows;
    i32x4 acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; nb++) acc[nb] = i32x4{0, 0, 0, 0};
    float sx = 0.f;
    if (live) {
        int64_t src = row0 + (mine ? m : 0);
        if (a.rows) src = a.rows[src];
        if ((uint64_t)src >= (uint64_t)a.n_x) src = 0;
        sx = a.sx[src];
        const int8_t *xr = q + src * pitch;
        const i32x4 *wf = reinterpret_cast<const i32x4 *>(a.w) + ((int64_t)e * panels + panel) * chunks * 256 + lane;
        for (int c = 0; c < chunks; c++) {
            const int k0 = c * 64 + g * 16;
            const i32x4 b = k0 < a.cin ? i8_row16(xr + k0, a.cin - k0) : i32x4{0, 0, 0, 0};
#pragma unroll
            for (int nb = 0; nb < 4; nb++) acc[nb] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[(int64_t)(c * 4 + nb) * 64], b, acc[nb], 0, 0, 0);
        }
    }
    if (mine) i8_store(a, e, panel, row0 + m, sx, live, acc);
}

static int64_t i8_pitch(int32_t cin) { return i8_chunks(cin) * 64; }
extern "C" int64_t cg3d_int8_linear_ws_bytes(int32_t dtype, int64_t n_x, int32_t cin, int64_t n_rows, int32_t cout, int32_t n_experts) {
    if (dtype < CG3D_DT_F32 || dtype > CG3D_DT_I8 || i8_bad_shape(n_experts, cin, cout) || n_x < 0 || n_x > 0x7fffffffll || n_rows < 0 ||
        n_rows > 0x7fffffffll)
        return CG3D_ERR_ARG;
    return dtype == CG3D_DT_I8 ? 0 : ((n_x * 4 + 255) & ~255ll) + n_x * i8_pitch(cin);
}
extern "C" int cg3d_int8_linear(const void *x, int32_t dtype, const float *sx, int64_t n_x, int32_t cin, const int8_t *w, const float *sw,
                                const float *bias, int32_t bias_per_expert, const int32_t *offsets, const int32_t *rows, void *y,
                                int32_t out_dtype, int64_t n_rows, int32_t cout, int32_t n_experts, void *ws, cg3d_stream_t stream) {
    const int64_t need = cg3d_int8_linear_ws_bytes(dtype, n_x, cin, n_rows, cout, n_experts);
    if (need < 0 || out_dtype < CG3D_DT_F32 || out_dtype > CG3D_DT_F16 || (bias_per_expert != 0 && bias_per_expert != 1)) return CG3D_ERR_ARG;
    if (offsets ? (!rows && n_x != n_rows) : (rows || n_x != n_rows || n_experts != 1)) return CG3D_ERR_ARG;
    if (n_rows == 0) return CG3D_OK;
    if (n_x == 0 || !x || !w || !sw || !y || (dtype == CG3D_DT_I8 && !sx) || (need > 0 && !ws)) return CG3D_ERR_ARG;
    if (((uintptr_t)x & (dtype == CG3D_DT_F32 ? 3 : dtype == CG3D_DT_I8 ? 0 : 1)) || ((uintptr_t)w & 15) || ((uintptr_t)y & (out_dtype == CG3D_DT_F32 ? 3 : 1)) ||
        (((uintptr_t)sx | (uintptr_t)sw | (uintptr_t)bias) & 3) || ((uintptr_t)ws & 15))
        return CG3D_ERR_ARG;
    hipStream_t s = cg3d_hs(stream);
    i8_args a = {sx, w, sw, bias, offsets, rows, y, n_rows, n_x, cin, cout, n_experts, out_dtype, bias_per_expert ? cout : 0};
    const int8_t *q = reinterpret_cast<const int8_t *>(x);
    int64_t pitch = cin;
    if (dtype != CG3D_DT_I8) {
        float *scale = reinterpret_cast<float *>(ws);
        int8_t *lev = reinterpret_cast<int8_t *>(ws) + ((n_x * 4 + 255) & ~255ll);
        pitch = i8_pitch(cin);
        const int rc = cg3d_int8_quantize_rows(x, dtype, n_x, cin, pitch, lev, scale, stream);
        if (rc != CG3D_OK) return rc;
        a.sx = scale;
        q = lev;
    }
    const int64_t nb = cg3d_divup(i8_tiles(a, 16) * i8_panels(cout), 4);
    if (nb > (1ll << 23)) return CG3D_ERR_ARG;
    hipLaunchKernelGGL(k_i8_wave, dim3((unsigned)nb), dim3(256), 0, s, a, q, pitch);
    CG3D_CHECK_LAUNCH();
    return CG3D_OK;
}
