// ds_ortho.hip -- an update matrix orthogonalised by Newton-Schulz products (ds_orthogonalize).
//
//   X = G / (|G|_F + eps);   steps times:  A = X X^T,  B = a I + b A + c A A,  X = B X      (m <= n; else the mirror image)
//
// A step is three products.  The first two have symmetric results: only tiles on and below the diagonal are formed, their
// mirror images written along.  Small singular values grow by a factor a = 3.4 per step, and with them whatever the products
// lost: with X, A and B rounded to bf16 the result is off by 1e-2 .. 6e-2, to fp16 by up to 8e-3 (matrices with a spectrum of
// three decades; measured against 64 bits), so all three are kept as two fp16 planes (22 bits; 1e-6) under fixed powers of
// two: entries of X and A are at most about 1.3, B's bound follows from the coefficients.
#include "ds_gemm.h"
#include "ds_internal.h"
#include "../../include/depthsynth.h"
#include <math.h>
#include <type_traits>

namespace ds {
namespace {

constexpr float kXs = 8192.f;    // stored X = 2^13 X, stored A = 2^13 A: 8x headroom in fp16
constexpr int kNormBlocks = 64;  // partial sums of squares per matrix


__global__ __launch_bounds__(256) void ortho_norm_kernel(const void* __restrict__ g, int dtype, long long mn,
                                                         double* __restrict__ part) {
    __shared__ double s[4];
    const long long base = blockIdx.y * mn;
    double a = 0.0;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < mn; i += kNormBlocks * 256ll) {
        const float x = dtype == DS_F32   ? static_cast<const float*>(g)[base + i]
                        : dtype == DS_F16 ? (float)static_cast<const f16*>(g)[base + i]
                                          : (float)static_cast<const bf16*>(g)[base + i];
        a += (double)x * x;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * kNormBlocks + blockIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
}

// G / (|G| + eps) as two planes, rows padded with zeros to np
__global__ __launch_bounds__(256) void ortho_load_kernel(const void* __restrict__ g, int dtype, int m, int n, int np, double eps,
                                                         const double* __restrict__ part, f16* __restrict__ x, long long lo,
                                                         long long per) {
    double t = 0.0;
    for (int i = 0; i < kNormBlocks; ++i) t += part[blockIdx.y * kNormBlocks + i];
    const double inv = 1.0 / (sqrt(t) + eps);
    const long long base = (long long)blockIdx.y * m * n;
    f16* y = x + blockIdx.y * per;
    const int lane = threadIdx.x & 63;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < m; r += gridDim.x * 4)
        for (int c = lane; c < np; c += 64) {
            float v = 0.f;
            if (c < n) {
                const long long i = base + (long long)r * n + c;
                v = dtype == DS_F32   ? static_cast<const float*>(g)[i]
                    : dtype == DS_F16 ? (float)static_cast<const f16*>(g)[i]
                                      : (float)static_cast<const bf16*>(g)[i];
            }
            f16 h, l;
            split16((float)(v * inv * kXs), h, l);   // scaled in double: a tiny or huge norm keeps its bits
            y[(long long)r * np + c] = h;
            y[(long long)r * np + c + lo] = l;
        }
}

// tile pair (i >= j) of a triangular index
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// One symmetric product of s x s: POLY false: A = X X^T (L = kK) or X^T X (L = kM);  true: B = a I + b A + c A A.
// Tiles with m0 >= n0; the element (m, n) is written at [n][m] (four consecutive m per lane) and, off the diagonal, at [m][n].
template <class S, Lay L, bool POLY>
__global__ __launch_bounds__(S::T) void ortho_sym_kernel(Operand X, long long per_x, int s, int k, f16* __restrict__ out, int ld,
                                                         long long lo, long long per_out, float ca, float cb, float cc,
                                                         float factor) {
    __shared__ __align__(16) char lds[S::kLds];
    int ti, tj;
    triangle(blockIdx.x, ti, tj);
    const int m0 = ti * S::BM, n0 = tj * S::BN;
    X.p = static_cast<const f16*>(X.p) + blockIdx.y * per_x;
    out += blockIdx.y * per_out;
    f32x4 acc[S::FM][S::FN];
    gemm_tile<f16, S, L, L, 3>(X, X, m0, n0, 0, k, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN;
    const f16* a = static_cast<const f16*>(X.p);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
        if (n >= s) continue;
#pragma unroll
        for (int i = 0; i < S::FM; ++i) {
            const int m = m0 + (wm * S::FM + i) * 16 + (lane >> 4) * 4;
            if (m >= ld) continue;
            float v[4];
            if (POLY) {
                const f16x4 h = *reinterpret_cast<const f16x4*>(a + (long long)n * X.ld + m);
                const f16x4 l = *reinterpret_cast<const f16x4*>(a + (long long)n * X.ld + m + X.lo);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = m + e < s ? fmaf(cc, acc[i][j][e], cb * ((float)h[e] + (float)l[e])) + (m + e == n ? ca : 0.f) : 0.f;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * factor;
            }
            put4<3>(out + (long long)n * ld + m, lo, v);
            if (ti != tj) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (m + e < s) {
                        f16 h, l;
                        split16(v[e], h, l);
                        out[(long long)(m + e) * ld + n] = h;
                        out[(long long)(m + e) * ld + n + lo] = l;
                    }
            }
        }
    }
}

// X' = B X (LA = kM on X, rows of B along n) or X B (LA = kK on B, rows of X along n): row r, columns along m.
// O = void: the next X (two planes); else the result in the caller's type, row pitch `cols`.
template <class S, Lay LA, class O>
__global__ __launch_bounds__(S::T) void ortho_apply_kernel(Operand A, Operand B, long long per_a, long long per_b, int rows,
                                                           int cols, int k, float factor, void* __restrict__ out, int ld,
                                                           long long lo, long long per_out) {
    __shared__ __align__(16) char lds[S::kLds];
    const int mt = cdiv(cols, S::BM);
    const int m0 = (int)(blockIdx.x % mt) * S::BM, n0 = (int)(blockIdx.x / mt) * S::BN;
    A.p = static_cast<const f16*>(A.p) + blockIdx.y * per_a;
    B.p = static_cast<const f16*>(B.p) + blockIdx.y * per_b;
    f32x4 acc[S::FM][S::FN];
    gemm_tile<f16, S, LA, kK, 3>(A, B, m0, n0, 0, k, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int r = n0 + (wn * S::FN + j) * 16 + (lane & 15);
        if (r >= rows) continue;
#pragma unroll
        for (int i = 0; i < S::FM; ++i) {
            const int c = m0 + (wm * S::FM + i) * 16 + (lane >> 4) * 4;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? acc[i][j][e] * factor : 0.f;
            if constexpr (std::is_same<O, void>::value) {
                if (c < ld) put4<3>(static_cast<f16*>(out) + blockIdx.y * per_out + (long long)r * ld + c, lo, v);
            } else {
                if (c < cols)
                    put_row4(static_cast<O*>(out) + blockIdx.y * per_out + (long long)r * cols, c, cols, v,
                             (cols & 3) == 0);
            }
        }
    }
}

template <class O>
__global__ __launch_bounds__(256) void ortho_only_scale_kernel(const void* __restrict__ g, double eps,
                                                               const double* __restrict__ part, long long mn,
                                                               void* __restrict__ out) {
    double t = 0.0;
    for (int i = 0; i < kNormBlocks; ++i) t += part[blockIdx.y * kNormBlocks + i];
    const double inv = 1.0 / (sqrt(t) + eps);
    const long long base = blockIdx.y * mn;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < mn; i += gridDim.x * 256ll)
        static_cast<O*>(out)[base + i] = (O)(float)((float)static_cast<const O*>(g)[base + i] * inv);
}

struct OrthoPlan {
    int s, l, sp, np;      // smaller and larger side; row pitch of A and of X
    size_t part, x0, x1, a, b, total;
};
OrthoPlan ortho_plan(int batch, int m, int n) {
    OrthoPlan p;
    p.s = m < n ? m : n;
    p.l = m < n ? n : m;
    p.sp = pad8(p.s);
    p.np = pad8(n);
    const size_t x = align256((size_t)batch * m * p.np * 4), a = align256((size_t)batch * p.s * p.sp * 4);
    size_t o = 0;
    p.part = o; o += align256((size_t)batch * kNormBlocks * 8);
    p.x0 = o; o += x;
    p.x1 = o; o += x;
    p.a = o; o += a;
    p.b = o; o += a;
    p.total = o;
    return p;
}

int check_ortho(int batch, int m, int n) {
    if (batch <= 0 || m <= 0 || n <= 0) return DS_ERR_INVALID_ARG;
    if (m > DS_ORTHO_MAX_SIDE || n > DS_ORTHO_MAX_SIDE || batch > 65535) return DS_ERR_UNSUPPORTED;
    if ((m < n ? m : n) > (1 << 15)) return DS_ERR_UNSUPPORTED;   // tiles of one launch
    return DS_OK;
}

template <class S, class O>
void ortho_steps(const OrthoPlan& p, int batch, int m, int n, int steps, const double* co, char* ws, void* out, hipStream_t q) {
    f16 *x = reinterpret_cast<f16*>(ws + p.x0), *y = reinterpret_cast<f16*>(ws + p.x1);
    f16 *a = reinterpret_cast<f16*>(ws + p.a), *b = reinterpret_cast<f16*>(ws + p.b);
    const long long px = 2ll * m * p.np, lox = (long long)m * p.np, pa = 2ll * p.s * p.sp, loa = (long long)p.s * p.sp;
    // stored B = 2^e B with |B| <= |a| + 2 |b| + 4 |c| below 2^15
    const double bound = fabs(co[0]) + 2 * fabs(co[1]) + 4 * fabs(co[2]);
    const float bs = (float)(bound > 0 ? exp2(floor(log2(32768.0 / bound))) : 1.0);
    const bool wide = m <= n;
    const int t = cdiv(p.s, S::BM), tiles = t * (t + 1) / 2;
    for (int i = 0; i < steps; ++i) {
        const Operand X{x, p.np, lox, m, p.np}, A{a, p.sp, loa, p.s, p.sp}, B{b, p.sp, loa, p.s, p.sp};
        const dim3 gs(tiles, batch);
        if (wide)
            ortho_sym_kernel<S, kK, false><<<gs, S::T, 0, q>>>(X, px, p.s, n, a, p.sp, loa, pa, 0, 0, 0, 1.f / kXs);
        else
            ortho_sym_kernel<S, kM, false><<<gs, S::T, 0, q>>>(X, px, p.s, m, a, p.sp, loa, pa, 0, 0, 0, 1.f / kXs);
        ortho_sym_kernel<S, kK, true><<<gs, S::T, 0, q>>>(A, pa, p.s, p.s, b, p.sp, loa, pa, (float)(co[0] * bs),
                                                          (float)(co[1] * bs / kXs), (float)(co[2] * bs / (kXs * kXs)), 0.f);
        const dim3 ga(cdiv(n, S::BM) * cdiv(m, S::BN), batch);
        const bool last = i + 1 == steps;
        const float f = last ? 1.f / (bs * kXs) : 1.f / bs;
        void* to = last ? out : y;
        const long long po = last ? (long long)m * n : px;
        if (wide) {
            if (last)
                ortho_apply_kernel<S, kM, O><<<ga, S::T, 0, q>>>(X, B, px, pa, m, n, p.s, f, to, p.np, lox, po);
            else
                ortho_apply_kernel<S, kM, void><<<ga, S::T, 0, q>>>(X, B, px, pa, m, n, p.s, f, to, p.np, lox, po);
        } else {
            if (last)
                ortho_apply_kernel<S, kK, O><<<ga, S::T, 0, q>>>(B, X, pa, px, m, n, p.s, f, to, p.np, lox, po);
            else
                ortho_apply_kernel<S, kK, void><<<ga, S::T, 0, q>>>(B, X, pa, px, m, n, p.s, f, to, p.np, lox, po);
        }
        f16* z = x;
        x = y;
        y = z;
    }
}

template <class O>
int ortho_any(const OrthoPlan& p, const void* g, int dtype, int batch, int m, int n, int steps, const double* co, double eps,
              void* out, char* ws, hipStream_t q) {
    double* part = reinterpret_cast<double*>(ws + p.part);
    const long long mn = (long long)m * n;
    ortho_norm_kernel<<<dim3(kNormBlocks, batch), 256, 0, q>>>(g, dtype, mn, part);
    if (steps == 0) {
        const int nb = cdiv(mn, 1024) < 4096 ? cdiv(mn, 1024) : 4096;
        ortho_only_scale_kernel<O><<<dim3(nb, batch), 256, 0, q>>>(g, eps, part, mn, out);
    } else {
        const int nb = cdiv(m, 4) < 2048 ? cdiv(m, 4) : 2048;
        ortho_load_kernel<<<dim3(nb, batch), 256, 0, q>>>(g, dtype, m, n, p.np, eps, part, reinterpret_cast<f16*>(ws + p.x0),
                                                          (long long)m * p.np, 2ll * m * p.np);
        // 64x64 tiles where 128x128 ones would leave most of the chip idle
        const int t = cdiv(p.s, 128);
        if ((long long)t * (t + 1) / 2 * batch < cu_count())
            ortho_steps<Shape<64, 64, 2, 2>, O>(p, batch, m, n, steps, co, ws, out, q);
        else
            ortho_steps<Shape<128, 128, 2, 2>, O>(p, batch, m, n, steps, co, ws, out, q);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DS_OK : (int)e;
}

}  // namespace
}  // namespace ds

extern "C" {

size_t ds_orthogonalize_workspace_bytes(int batch, int m, int n) {
    return ds::check_ortho(batch, m, n) ? 0 : ds::ortho_plan(batch, m, n).total;
}

int ds_orthogonalize(const void* update, int dtype, int batch, int m, int n, int steps, const double* coefficients, double eps,
                     void* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!update || !out || !coefficients || steps < 0 || !(eps >= 0)) return DS_ERR_INVALID_ARG;
    const int rc = ds::check_ortho(batch, m, n);
    if (rc) return rc;
    if (steps > DS_ORTHO_MAX_STEPS || (dtype != DS_F32 && dtype != DS_F16 && dtype != DS_BF16)) return DS_ERR_UNSUPPORTED;
    if (((uintptr_t)out & 15) != 0) return DS_ERR_INVALID_ARG;
    const ds::OrthoPlan p = ds::ortho_plan(batch, m, n);
    if (!workspace || workspace_bytes < p.total || ((uintptr_t)workspace & 15) != 0) return DS_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    hipStream_t q = static_cast<hipStream_t>(stream);
    if (dtype == DS_F32) return ds::ortho_any<float>(p, update, dtype, batch, m, n, steps, coefficients, eps, out, ws, q);
    if (dtype == DS_F16) return ds::ortho_any<ds::f16>(p, update, dtype, batch, m, n, steps, coefficients, eps, out, ws, q);
    return ds::ortho_any<ds::bf16>(p, update, dtype, batch, m, n, steps, coefficients, eps, out, ws, q);
}

}  // extern "C"
