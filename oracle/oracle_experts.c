/* oracle_experts.c -- CPU restatement of the routed-row and 8-bit product entry points of include/cagroup3d_hip.h (test
 * infrastructure): the definitions written out row by row, sums in double. */
#include <math.h>
#include <stdint.h>
#include <string.h>
#include "../include/cagroup3d_hip.h"

/* ---- element types ---- */
static float ld(const void *p, int32_t dt, int64_t i) {
    if (dt == CG3D_DT_F32) return ((const float *)p)[i];
    const uint16_t h = ((const uint16_t *)p)[i];
    uint32_t u;
    float f;
    if (dt == CG3D_DT_BF16) {
        u = (uint32_t)h << 16;
        memcpy(&f, &u, 4);
        return f;
    }
    const uint32_t s = (uint32_t)(h >> 15) << 31, e = (h >> 10) & 31, m = h & 1023;
    if (e == 0) f = ldexpf((float)m, -24);
    else if (e == 31) f = m ? NAN : INFINITY;
    else f = ldexpf((float)(1024 + m), (int)e - 25);
    memcpy(&u, &f, 4);
    u |= s;
    memcpy(&f, &u, 4);
    return f;
}
static void st(void *p, int32_t dt, int64_t i, double d) {
    float f = (float)d;
    uint32_t u;
    if (dt == CG3D_DT_F32) { ((float *)p)[i] = f; return; }
    memcpy(&u, &f, 4);
    uint16_t h;
    if (f != f) h = dt == CG3D_DT_BF16 ? 0x7fc0 : 0x7e00;
    else if (dt == CG3D_DT_BF16) h = (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
    else {
        const uint16_t s = (uint16_t)((u >> 16) & 0x8000);
        const float a = fabsf(f);
        if (a >= 65520.f) h = s | 0x7c00;
        else if (a < 6.103515625e-05f) h = (uint16_t)(s | (uint16_t)rintf(a * 16777216.f));
        else {
            uint32_t v;
            memcpy(&v, &a, 4);
            v += 0xfff + ((v >> 13) & 1);
            h = (uint16_t)(s | ((v >> 13) - (112u << 10)));
        }
    }
    ((uint16_t *)p)[i] = h;
}
static int es(int32_t dt) { return dt == CG3D_DT_F32 ? 4 : dt == CG3D_DT_I8 ? 1 : 2; }
static int fl(int32_t dt) { return dt >= CG3D_DT_F32 && dt <= CG3D_DT_F16; }
static int odd(const void *p, int32_t dt) { return ((uintptr_t)p & (uintptr_t)(es(dt) - 1)) != 0; }

/* ---- rows sorted by expert ---- */
int64_t cg3d_expert_plan_ws_bytes(int64_t n_tokens, int32_t k, int32_t n_experts) {
    if (n_tokens < 0 || k < 1 || n_experts < 1 || n_experts > 1024 || n_tokens > 0x7fffffffll / k) return CG3D_ERR_ARG;
    return 0;
}
int cg3d_expert_plan(const void *experts, int32_t wide, int64_t n_tokens, int32_t k, int32_t n_experts, int32_t *offsets, int32_t *rows,
                     int32_t *pairs, int32_t *pos, void *ws, cg3d_stream_t stream) {
    (void)ws; (void)stream;
    if (cg3d_expert_plan_ws_bytes(n_tokens, k, n_experts) < 0 || (wide != 0 && wide != 1) || !offsets) return CG3D_ERR_ARG;
    const int64_t n = n_tokens * k;
    if (n > 0 && (!experts || !rows || !pairs || !pos || ((uintptr_t)experts & (wide ? 7 : 3)))) return CG3D_ERR_ARG;
    int64_t next[1025];
    memset(next, 0, sizeof next);
#define KEY(p) ({ const int64_t v = wide ? ((const int64_t *)experts)[p] : ((const int32_t *)experts)[p]; v < 0 || v >= n_experts ? n_experts : v; })
    for (int64_t p = 0; p < n; p++) next[KEY(p)]++;
    int64_t at = 0;
    for (int e = 0; e <= n_experts; e++) {
        const int64_t c = next[e];
        offsets[e] = (int32_t)at;
        next[e] = at;
        at += c;
    }
    for (int64_t p = 0; p < n; p++) {
        const int64_t e = KEY(p);
        const int32_t row = (int32_t)next[e]++;
        rows[row] = e < n_experts ? (int32_t)(p / k) : -1;
        pairs[row] = e < n_experts ? (int32_t)p : ~(int32_t)p;
        pos[p] = e < n_experts ? row : ~row;
    }
    return CG3D_OK;
}
static int bad(int32_t dt, int32_t wt, int64_t n, int32_t k, int32_t c) {
    return !fl(dt) || !fl(wt) || n < 0 || k < 1 || c < 1 || c > (1 << 30) || n > 0x7fffffffll / k;
}
int cg3d_expert_gather(const void *x, int32_t dtype, const int32_t *rows, int64_t n_tokens, int32_t k, int32_t c, void *out,
                       cg3d_stream_t stream) {
    (void)stream;
    if (bad(dtype, 0, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!x || !rows || !out || odd(x, dtype) || odd(out, dtype)) return CG3D_ERR_ARG;
    const int64_t w = (int64_t)c * es(dtype), P = n_tokens * k;
    for (int64_t j = 0; j < P; j++) {
        if (rows[j] < 0 || rows[j] >= n_tokens) memset((char *)out + j * w, 0, (size_t)w);
        else memcpy((char *)out + j * w, (const char *)x + rows[j] * w, (size_t)w);
    }
    return CG3D_OK;
}
int cg3d_expert_combine(const void *y, int32_t dtype, const int32_t *pos, const void *w, int32_t wtype, int64_t n_tokens, int32_t k,
                        int32_t c, void *out, int32_t out_dtype, cg3d_stream_t stream) {
    (void)stream;
    if (bad(dtype, wtype, n_tokens, k, c) || !fl(out_dtype) || (dtype != CG3D_DT_F32 && out_dtype != dtype)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if (!y || !pos || !out || odd(y, dtype) || odd(out, out_dtype) || odd(w, wtype)) return CG3D_ERR_ARG;
    for (int64_t t = 0; t < n_tokens; t++)
        for (int32_t a = 0; a < c; a++) {
            double acc = 0;
            for (int32_t s = 0; s < k; s++) {
                const int32_t r = pos[t * k + s];
                if (r >= 0 && r < n_tokens * k) acc += (w ? (double)ld(w, wtype, t * k + s) : 1.0) * ld(y, dtype, (int64_t)r * c + a);
            }
            st(out, out_dtype, t * c + a, acc);
        }
    return CG3D_OK;
}
int cg3d_expert_combine_bwd(const void *dout, const void *y, int32_t dtype, const int32_t *pairs, const void *w, int32_t wtype,
                            int64_t n_tokens, int32_t k, int32_t c, void *dy, void *dw, cg3d_stream_t stream) {
    (void)stream;
    if (bad(dtype, wtype, n_tokens, k, c)) return CG3D_ERR_ARG;
    if (n_tokens == 0) return CG3D_OK;
    if ((!dy && !dw) || !dout || !pairs || (dw && (!y || !w)) || odd(dout, dtype) || odd(y, dtype) || odd(dy, dtype) || odd(w, wtype) || odd(dw, wtype))
        return CG3D_ERR_ARG;
    const int64_t P = n_tokens * k;
    for (int64_t j = 0; j < P; j++) {
        const int there = pairs[j] >= 0 && pairs[j] < P;
        const int64_t p = pairs[j] < 0 ? ~pairs[j] : pairs[j], t = p / k;
        double dot = 0;
        for (int32_t a = 0; a < c; a++) {
            const double g = there ? ld(dout, dtype, t * c + a) : 0;
            if (dw && there) dot += g * ld(y, dtype, j * c + a);
            if (dy) st(dy, dtype, j * c + a, there ? (w ? (double)ld(w, wtype, p) : 1.0) * g : 0);
        }
        if (dw && p < P) st(dw, wtype, p, dot);
    }
    return CG3D_OK;
}

/* ---- products in 8-bit integers ---- */
static int level(float x, float amax) {                 /* 127 x / amax, nearest, ties to even, decided in 64 bits (all exact) */
    const double a = fabs((double)x) * 254.0, m = (double)amax;
    int n = (int)floor(a / m / 2);
    if (n > 0) n--;                                       /* (the quotient may be off in its last place) */
    while (a > (2 * n + 1) * m || (a == (2 * n + 1) * m && (n & 1))) n++;
    return x < 0 ? -n : n;
}
static int bad_shape(int32_t e, int32_t cin, int32_t cout) {
    return e < 1 || e > 1024 || cin < 1 || cin > 131071 || cout < 1 || cout > (1 << 20);
}
static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
/* where weight (e, k, n) lies in the packed form */
static int64_t place(int32_t e, int32_t k, int32_t n, int32_t cin, int32_t cout) {
    const int64_t panels = up(cout, 64), chunks = up(cin, 64);
    const int nb = n % 4, m = n % 64 / 4;
    const int lane = (k % 64) / 16 * 16 + m;
    return ((((int64_t)e * panels + n / 64) * chunks + k / 64) * 4 + nb) * 1024 + lane * 16 + k % 16;
}
int64_t cg3d_int8_weight_bytes(int32_t e, int32_t cin, int32_t cout) {
    return bad_shape(e, cin, cout) ? CG3D_ERR_ARG : (int64_t)e * up(cout, 64) * up(cin, 64) * 4096;
}
int cg3d_int8_weight(const void *w, int32_t dtype, int32_t E, int32_t cin, int32_t cout, int8_t *packed, float *scale, void *ws,
                     cg3d_stream_t stream) {
    (void)stream;
    if (bad_shape(E, cin, cout) || dtype < CG3D_DT_F32 || dtype > CG3D_DT_I8 || !w || !packed || ((uintptr_t)packed & 15)) return CG3D_ERR_ARG;
    if (odd(w, dtype) || (dtype != CG3D_DT_I8 && (!scale || !ws))) return CG3D_ERR_ARG;
    memset(packed, 0, (size_t)cg3d_int8_weight_bytes(E, cin, cout));
    for (int32_t e = 0; e < E; e++)
        for (int32_t n = 0; n < cout; n++) {
            float amax = 0;
            int fine = 1;
            if (dtype != CG3D_DT_I8) {
                for (int32_t k = 0; k < cin; k++) {
                    const float v = fabsf(ld(w, dtype, ((int64_t)e * cin + k) * cout + n));
                    if (!isfinite(v)) fine = 0;
                    if (v > amax) amax = v;
                }
                scale[(int64_t)e * cout + n] = fine ? amax / 127.f : NAN;
            }
            for (int32_t k = 0; k < cin; k++) {
                const int64_t i = ((int64_t)e * cin + k) * cout + n;
                const int q = dtype == CG3D_DT_I8 ? ((const int8_t *)w)[i] : fine && amax > 0 ? level(ld(w, dtype, i), amax) : 0;
                packed[place(e, k, n, cin, cout)] = (int8_t)q;
            }
        }
    return CG3D_OK;
}
int cg3d_int8_quantize_rows(const void *x, int32_t dtype, int64_t n, int32_t cin, int64_t pitch, int8_t *q, float *scale,
                            cg3d_stream_t stream) {
    (void)stream;
    if (!fl(dtype) || n < 0 || cin < 1 || cin > 131071 || pitch < cin || pitch > (1 << 30)) return CG3D_ERR_ARG;
    if (n == 0) return CG3D_OK;
    if (!x || !q || !scale || odd(x, dtype) || odd(scale, 0)) return CG3D_ERR_ARG;
    for (int64_t r = 0; r < n; r++) {
        float amax = 0;
        int fine = 1;
        for (int32_t k = 0; k < cin; k++) {
            const float v = fabsf(ld(x, dtype, r * cin + k));
            if (!isfinite(v)) fine = 0;
            if (v > amax) amax = v;
        }
        scale[r] = fine ? amax / 127.f : NAN;
        memset(q + r * pitch, 0, (size_t)pitch);
        if (fine && amax > 0)
            for (int32_t k = 0; k < cin; k++) q[r * pitch + k] = (int8_t)level(ld(x, dtype, r * cin + k), amax);
    }
    return CG3D_OK;
}
int64_t cg3d_int8_linear_ws_bytes(int32_t dtype, int64_t n_x, int32_t cin, int64_t n_rows, int32_t cout, int32_t n_experts, int32_t flags) {
    if (dtype < CG3D_DT_F32 || dtype > CG3D_DT_I8 || bad_shape(n_experts, cin, cout) || n_x < 0 || n_x > 0x7fffffffll || n_rows < 0 ||
        n_rows > 0x7fffffffll || (flags & ~3))
        return CG3D_ERR_ARG;
    return dtype == CG3D_DT_I8 ? 0 : n_x * (4 + (int64_t)cin);
}
int cg3d_int8_linear(const void *x, int32_t dtype, const float *sx, int64_t n_x, int32_t cin, const int8_t *w, const float *sw,
                     const float *bias, int32_t bias_per_expert, const int32_t *offsets, const int32_t *rows, void *y, int32_t out_dtype,
                     int64_t n_rows, int32_t cout, int32_t n_experts, void *ws, cg3d_stream_t stream) {
    const int64_t need = cg3d_int8_linear_ws_bytes(dtype, n_x, cin, n_rows, cout, n_experts, offsets != 0);
    if (need < 0 || !fl(out_dtype) || (bias_per_expert != 0 && bias_per_expert != 1)) return CG3D_ERR_ARG;
    if (offsets ? (!rows && n_x != n_rows) : (rows || n_x != n_rows || n_experts != 1)) return CG3D_ERR_ARG;
    if (n_rows == 0) return CG3D_OK;
    if (n_x == 0 || !x || !w || !sw || !y || (dtype == CG3D_DT_I8 && !sx) || (need > 0 && !ws)) return CG3D_ERR_ARG;
    if (odd(x, dtype) || ((uintptr_t)w & 15) || odd(y, out_dtype) || odd(sx, 0) || odd(sw, 0) || odd(bias, 0) || odd(offsets, 0) || odd(rows, 0) || ((uintptr_t)ws & 15))
        return CG3D_ERR_ARG;
    const int8_t *q = (const int8_t *)x;
    if (dtype != CG3D_DT_I8) {
        int8_t *lv = (int8_t *)ws + 4 * n_x;
        const int rc = cg3d_int8_quantize_rows(x, dtype, n_x, cin, cin, lv, (float *)ws, stream);
        if (rc) return rc;
        q = lv;
        sx = (const float *)ws;
    }
    for (int64_t r = 0; r < n_rows; r++) {
        int32_t e = 0;
        if (offsets)
            while (e < n_experts && r >= offsets[e + 1]) e++;
        const int64_t src = e < n_experts && rows ? rows[r] : r;
        for (int32_t n = 0; n < cout; n++) {
            float v = 0;
            if (e < n_experts) {
                int32_t sum = 0;
                for (int32_t k = 0; k < cin; k++) sum += (int32_t)q[src * cin + k] * w[place(e, k, n, cin, cout)];
                const float a = fabsf(sx[src]);               /* (scales at the range's ends: sum * sx is kept inside it) */
                const float by = a >= 0x1p96f ? 0x1p-64f : a < 0x1p-126f ? 0x1p64f : 1.f;
                v = (float)sum * (sx[src] * by) * sw[(int64_t)e * cout + n] * (1.f / by);
                if (bias) v += bias[(bias_per_expert ? (int64_t)e * cout : 0) + n];
            }
            st(y, out_dtype, r * cout + n, v);
        }
    }
    return CG3D_OK;
}
