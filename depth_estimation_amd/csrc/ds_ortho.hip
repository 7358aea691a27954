// ds_ortho.hip -- an update matrix orthogonalised by Newton-Schulz products (ds_orthogonalize).
//
//   X = G / (|G|_F + eps);   steps times:  A = X X^T,  B = a I + b A + c A A,  X = B X      (m <= n; else the mirror image)
//
// A step is three products.  The first two have symmetric results: only tiles on and below the diagonal are formed, their
// mirror images written along.  Small singular values grow by a factor a = 3.4 per step, and with them whatever the products
// lost: with X, A and B rounded to bf16 the result is off by 1e-2 .. 6e-2, to fp16 by up to 8e-3 (matrices with a spectrum of
// three decades; measured against 64 bits), so all three are kept as two fp16 planes (22 bits; 1e-6) under powers of two that
// follow from the coefficients alone: singular values begin in [0, 1], so how far each step can take them is known before it
// (steps_of), and entries are at most as large as the largest singular value.
//
// bf16 results of larger matrices after few steps need less, and take half the products (Light): A keeps one plane (11 bits) off
// the diagonal, where its entries are small, and its diagonal in fp32 beside it.  B keeps one plane; what its diagonal, which carries most of
// X, lost by that is made up for as a factor of the result's row: diag(d) X (1 + rounding) off the diagonal is the smaller part.
// X keeps two planes where it is multiplied by B.  What that costs after five steps is 4e-4 .. 9e-4 of the result's norm (sides
// of 256 and more; Gaussian, decaying and nearly low-rank matrices, written out in float64), under the 1.7e-3 that rounding the
// result to bf16 costs; without the factors 6e-4 .. 1.2e-3.  It grows with the steps (ten: 1.8e-3), and with how steep the
// polynomial is: small_errors() has the condition.
#include "ds_gemm.h"
#include "ds_internal.h"
#include "../../include/depthsynth.h"
#include <math.h>
#include <type_traits>

namespace ds {
namespace {

constexpr float kXs = 8192.f;    // stored X = 2^13 X where singular values are at most sqrt(2), stored A = 2^13 A

// Factors of one step's products, and of the result.  X is stored as 2^(13 - e) X and A as 2^(13 - 2e) A, where e, the step's
// own, is the least with |X| <= 2^e sqrt(2) (spectral norm; 0 for coefficients that keep it near one), so that A <= 2^14 as
// stored; B with its bound |a| + |b| A + |c| A^2 in (2^14, 2^15].
struct Step {
    float gram;          // accumulated X X^T -> stored A
    float ca, cb, cc;    // the identity, stored A and accumulated A A -> stored B
    float next;          // accumulated B X -> the next stored X, or after the last step X itself
};
struct Steps {
    Step s[DS_ORTHO_MAX_STEPS];
};
constexpr int kMostShift = 24;

// Whether one plane is enough for a bf16 result (Light): up to six steps of a polynomial p that lifts small singular values,
// keeps all of them positive and at most sqrt(2), and has slopes of -1.7 .. 4 where it meets any.  Over 130 such polynomials
// (written out in float64, 512 x 512 Gaussian, decaying and nearly low-rank) the result was off by 1.13e-3 of its norm at most;
// with slopes to -3 by 1.5e-2, after ten steps of the default polynomial by 1.8e-3 and after 32 by 3.2e-3.
bool small_errors(const double* co, int steps, double most /* the largest singular value before any step */) {
    const double m2 = most * most;
    auto value = [&](double t) { return co[0] + t * (co[1] + t * co[2]); };               // p(x) / x, t = x^2
    auto slope = [&](double t) { return co[0] + t * (3 * co[1] + t * 5 * co[2]); };
    auto steep = [&](double t) { return slope(t) > 4 || slope(t) < -1.7; };
    if (steps > 6 || m2 > 2 || co[0] < 1 || !(value(m2) > 0) || steep(0) || steep(m2)) return false;
    const double at = co[2] != 0 ? -co[1] / (2 * co[2]) : 0, turn = 0.6 * at;             // where the two have their extrema
    return !(at > 0 && at < m2 && !(value(at) > 0)) && !(turn > 0 && turn < m2 && steep(turn));
}

// the largest |x (a + b x^2 + c x^4)| for x in [0, m]
double reach_of(const double* co, double m) {
    auto at = [&](double t) { return fabs(sqrt(t) * (co[0] + t * (co[1] + t * co[2]))); };
    double most = at(m * m);
    // the derivative a + 3 b t + 5 c t^2, t = x^2, is zero
    const double p = 3 * co[1], q = 5 * co[2], d = p * p - 4 * q * co[0];
    if (d >= 0) {
        const double r = -0.5 * (p + (p >= 0 ? sqrt(d) : -sqrt(d))), roots[2] = {q != 0 ? r / q : -1, r != 0 ? co[0] / r : -1};
        for (double t : roots)
            if (t > 0 && t < m * m && at(t) > most) most = at(t);
    }
    return most;
}
// false: singular values would leave the range (2^kMostShift before the last step, 2^100 after it; NaN)
bool steps_of(const double* co, int steps, Steps& out, bool& light) {
    double m = 1, most = 1;
    auto shift = [](double x) {
        const double e = x > 0 ? ceil(log2(x / sqrt(2.0))) : -kMostShift;
        return e < -kMostShift ? -kMostShift : e;     // (smaller yet: bits are lost one by one, as below any type's range)
    };
    for (int i = 0; i < steps; ++i) {
        const double e = shift(m), xs = exp2(13 - e), as = exp2(13 - 2 * e), top = 2 * exp2(2 * e);
        const double bound = fabs(co[0]) + top * (fabs(co[1]) + top * fabs(co[2]));
        if (!(e <= kMostShift) || !(bound <= exp2(100))) return false;
        const double k = bound > 0 ? floor(log2(32768.0 / bound)) : 0, bs = exp2(k > 100 ? 100 : k);
        m = reach_of(co, m);
        const bool last = i + 1 == steps;
        if (!last && m > most) most = m;
        if (!(m <= exp2(last ? 100 : kMostShift))) return false;
        const double next = last ? 1 : exp2(13 - shift(m));
        out.s[i] = Step{(float)(as / (xs * xs)), (float)(co[0] * bs), (float)(co[1] * bs / as), (float)(co[2] * bs / (as * as)),
                        (float)(next / (bs * xs))};
    }
    light = small_errors(co, steps, most);
    return true;
}
// blocks that sum squares of one matrix: 4096 elements each, at most 512
__host__ __device__ inline int norm_blocks(long long mn) {
    const long long n = (mn + 4095) / 4096;
    return n < 512 ? (int)n : 512;
}
// sum over a workgroup of T threads, the same in every thread
template <int T>
__device__ __forceinline__ double sum_all(double a, double* s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o, 64);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = a;
    __syncthreads();
    a = 0.0;
    for (int i = 0; i < T / 64; ++i) a += s[i];
    __syncthreads();
    return a;
}

// 16 bytes a lane, four such loads under way; the elements behind the last whole vector by the first block
template <class O>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const O* __restrict__ g, long long mn, double* __restrict__ part) {
    constexpr int VEC = 16 / sizeof(O), U = 4;
    typedef O vec __attribute__((ext_vector_type(VEC)));
    typedef vec loose __attribute__((aligned(sizeof(O))));
    __shared__ double s[4];
    const O* x = g + blockIdx.y * mn;
    const long long nv = mn / VEC, step = gridDim.x * 256ll;
    double a = 0.0;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < nv; i += U * step) {
        vec v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = *reinterpret_cast<const loose*>(x + (i + u * step < nv ? i + u * step : i) * VEC);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * step < nv)
#pragma unroll
                for (int e = 0; e < VEC; ++e) a = fma((double)(float)v[u][e], (double)(float)v[u][e], a);
    }
    if (blockIdx.x == 0 && nv * VEC + threadIdx.x < mn) {
        const double y = (float)x[nv * VEC + threadIdx.x];
        a = fma(y, y, a);
    }
    a = sum_all<256>(a, s);
    if (threadIdx.x == 0) part[blockIdx.y * gridDim.x + blockIdx.x] = a;
}
template <int T>
__device__ __forceinline__ double inverse_norm(const double* part, int blocks, double eps, double* s) {
    double t = 0.0;
    for (int i = threadIdx.x; i < blocks; i += T) t += part[i];
    return 1.0 / (sqrt(sum_all<T>(t, s)) + eps);
}

// G / (|G| + eps) as two planes, rows padded with zeros to np.  Four elements a lane, four such loads under way (one at a time:
// 11 us at 512 x 4608 float32)
template <class O>
__global__ __launch_bounds__(256) void ortho_load_kernel(const O* __restrict__ g, int m, int n, int np, double eps,
                                                         const double* __restrict__ part, int blocks, f16* __restrict__ x,
                                                         long long lo, long long per) {
    constexpr int U = 4;
    typedef O o4 __attribute__((ext_vector_type(4)));
    typedef o4 loose __attribute__((aligned(sizeof(O))));
    __shared__ double s[4];
    const O* src = g + (long long)blockIdx.y * m * n;
    f16* y = x + blockIdx.y * per;
    const unsigned q = np / 4;
    const long long all = (long long)m * q, step = gridDim.x * 256ll;
    auto load = [&](long long i, o4& v) {
        const int r = all < (1ll << 31) ? (int)((unsigned)i / q) : (int)(i / q), c = (int)(i - (long long)r * q) * 4;
        const O* p = src + (long long)r * n + c;
        if (c + 4 <= n) {
            v = *reinterpret_cast<const loose*>(p);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = c + e < n ? p[e] : (O)0.f;
        }
    };
    const long long i0 = blockIdx.x * 256ll + threadIdx.x;
    o4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * step < all) load(i0 + u * step, v[u]);
    const double inv = inverse_norm<256>(part + (long long)blockIdx.y * blocks, blocks, eps, s) * kXs;
    for (long long i = i0; i < all; i += U * step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long at = i + u * step;
            if (at >= all) break;
            if (i != i0) load(at, v[u]);
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (float)((float)v[u][e] * inv);   // scaled in double: a tiny or huge norm keeps its bits
            put4<3>(y + at * 4, lo, w);
        }
    }
}

// tile pair (i >= j) of a triangular index
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
    i = (int)((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
}

// What becomes of a product's tile.  kGram: A = X X^T;  kPoly: B = a I + b A + c A A;  both symmetric: tiles with m0 >= n0, the
// element (m, n) written at [n][m] (four consecutive m per lane) and, off the diagonal, at [m][n].  kNext: the next X, row n,
// columns along m.  kLast: the result in the caller's type.
enum Use { kGram, kPoly, kNext, kLast };
template <Use U_, bool LIGHT_>
struct How {
    static constexpr Use U = U_;
    static constexpr bool LIGHT = LIGHT_;
};
struct UseArgs {
    int rows, cols;          // of the result; columns beyond `cols` up to ld are written as zeros
    void* out;
    int ld;
    long long lo, per_out;   // planes apart, matrices apart
    const f16* a;            // kPoly: A again
    long long per_a;
    float ca, cb, cc;        // kPoly: Step's; else ca: the factor
    float *da, *db;          // light: A's diagonal, scaled as A, and B's as it is over what its plane holds; `side` a matrix
    int side, wide;
};
// fragment rows i and i + 1 of a tile (of a shape with one: x)
template <class S, class H, class O>
__device__ __forceinline__ void use_rows(const f32x4 (&x)[S::FN], const f32x4 (&y)[S::FN], int i, int m0, int n0, int batch,
                                         const UseArgs& u) {
    constexpr Use U = H::U;
    constexpr int F = S::FM == 1 ? 1 : 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN;
    const int mi = m0 + (wm * S::FM + i) * 16;
    const float* da = H::LIGHT ? u.da + (long long)batch * u.side : nullptr;
    const float* db = H::LIGHT ? u.db + (long long)batch * u.side : nullptr;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
        if (n >= u.rows) continue;
        f32x4 v[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const f32x4 acc = f ? y[j] : x[j];
            const int m = mi + f * 16 + (lane >> 4) * 4;
            float old[4] = {0.f, 0.f, 0.f, 0.f};
            if (U == kPoly && m < u.ld) {      // A at the same place
                const f16* a = u.a + batch * u.per_a + (long long)n * u.ld + m;
                const f16x4 h = *reinterpret_cast<const f16x4*>(a);
#pragma unroll
                for (int e = 0; e < 4; ++e) old[e] = (float)h[e];
                if (!H::LIGHT) {
                    const f16x4 l = *reinterpret_cast<const f16x4*>(a + u.lo);
#pragma unroll
                    for (int e = 0; e < 4; ++e) old[e] += (float)l[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = m + e < u.cols, diagonal = m + e == n;
                if (U == kPoly && !H::LIGHT) {
                    v[f][e] = fmaf(u.cc, acc[e], u.cb * old[e]) + (diagonal ? u.ca : 0.f);
                } else if (U == kPoly) {
                    const float dn = da[n], dm = in ? da[m + e] : 0.f;
                    // (O + D)(O + D) = O O + O D + D O + D D
                    v[f][e] = diagonal ? fmaf(u.cc, fmaf(dn, dn, acc[e]), fmaf(u.cb, dn, u.ca))
                                       : fmaf(u.cc, fmaf(dn + dm, old[e], acc[e]), u.cb * old[e]);
                    if (diagonal) {      // (below fp16's normal numbers nothing is lost that matters beside B's other entries)
                        const float h = (float)(f16)v[f][e];
                        u.db[(long long)batch * u.side + n] = fabsf(h) >= 6.1035156e-5f ? v[f][e] / h : 1.f;
                    }
                } else if (H::LIGHT && U == kGram) {
                    v[f][e] = diagonal ? 0.f : acc[e] * u.ca;
                    if (diagonal) u.da[(long long)batch * u.side + n] = acc[e] * u.ca;
                } else if (H::LIGHT) {
                    v[f][e] = in ? acc[e] * (db[u.wide ? n : m + e] * u.ca) : 0.f;
                } else {
                    v[f][e] = acc[e] * u.ca;
                }
                if (!in) v[f][e] = 0.f;
            }
        }
        const float v0[4] = {v[0][0], v[0][1], v[0][2], v[0][3]};
        if (U == kLast) {
            O* row = static_cast<O*>(u.out) + batch * u.per_out + (long long)n * u.cols;
            if (F == 2)
                put_row8(row, mi, u.cols, lane, v[0], v[F - 1]);
            else
                put_row4(row, mi + (lane >> 4) * 4, u.cols, v0);
            continue;
        }
        constexpr bool kTwo = !H::LIGHT || U == kNext;      // planes of the result
        f16* out = static_cast<f16*>(u.out) + batch * u.per_out;
        if constexpr (F == 2) {
            const int m8 = mi + (lane >> 4) * 8;
            s16x8 hi, lo;
            eight_of(round4<f16>(v[0]), round4<f16>(v[1]), hi);
            if constexpr (kTwo) eight_of(rest4(v[0]), rest4(v[1]), lo);
            if (m8 < u.ld) {
                *reinterpret_cast<s16x8*>(out + (long long)n * u.ld + m8) = hi;
                if constexpr (kTwo) *reinterpret_cast<s16x8*>(out + (long long)n * u.ld + m8 + u.lo) = lo;
            }
        } else if (mi + (lane >> 4) * 4 < u.ld) {
            put4<kTwo ? 3 : 1>(out + (long long)n * u.ld + mi + (lane >> 4) * 4, u.lo, v0);
        }
        if ((U == kGram || U == kPoly) && m0 != n0) {
#pragma unroll
            for (int f = 0; f < F; ++f)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = mi + f * 16 + (lane >> 4) * 4 + e;
                    if (m < u.cols) {
                        f16 h, l;
                        split16(v[f][e], h, l);
                        out[(long long)m * u.ld + n] = h;
                        if (kTwo) out[(long long)m * u.ld + n + u.lo] = l;
                    }
                }
        }
    }
}
template <class S, class H, class O>
__device__ __forceinline__ void use_tile(const f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int batch, const UseArgs& u) {
#pragma unroll
    for (int i = 0; i < S::FM; i += 2) use_rows<S, H, O>(acc[i], acc[S::FM == 1 ? 0 : i + 1], i, m0, n0, batch, u);
}

// C = A B over k.  tri: only tiles with m0 >= n0.  Units: matrices x tiles x splits; part (may be NULL: no splits): the tiles'
// sums, a thread's fragments 16 bytes next to its neighbour's, for ortho_finish_kernel.
struct ProductArgs {
    Operand A, B;
    long long per_a, per_b;
    int mt, nt, tri, k, splits, batch;
    float* part;
};
// a tile's matrix and place; tiles: of a matrix
template <class S>
__device__ __forceinline__ void tile_of(const ProductArgs& p, int tile, int tiles, int& batch, int& m0, int& n0) {
    batch = tile / tiles;
    int m, n;
    if (p.tri)
        triangle(tile - batch * tiles, m, n);
    else
        Order(tiles, p.mt, p.nt).at(tile - batch * tiles, m, n);
    m0 = m * S::BM;
    n0 = n * S::BN;
}
// matrix by matrix, split by split: an XCD works on few ranges of k at a time
template <class S>
__device__ __forceinline__ void unit_of(const ProductArgs& p, int u, int units, int& batch, int& m0, int& n0, int& sp, int& tile) {
    const int v = Order(units, p.mt, p.nt).turn_of(u), per = units / p.batch, tiles = per / p.splits;
    batch = v / per;
    sp = (v - batch * per) / tiles;
    tile = v - sp * tiles - batch * (per - tiles);
    tile_of<S>(p, tile, tiles, batch, m0, n0);
}
template <class S>
__device__ __forceinline__ void keep_part(const f32x4 (&acc)[S::FM][S::FN], const ProductArgs& p, int tile, int sp) {
    f32x4* q = reinterpret_cast<f32x4*>(p.part) + ((long long)tile * p.splits + sp) * (S::BM * S::BN / 4) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) q[(i * S::FN + j) * S::T] = acc[i][j];
}
template <class S, Lay LA, Lay LB, int PA, int PB, class H, class O, bool PART>
__global__ __launch_bounds__(S::T) void ortho_product_kernel(ProductArgs p, UseArgs u, int units) {
    __shared__ __align__(16) char lds[std::is_same<S, Big>::value ? Big::kLds : lds_bytes<S, PA, PB>()];
    const int per = cdiv(cdiv(p.k, kBK), p.splits) * kBK;
    auto job = [&](int x) {
        int batch, m0, n0, sp, tile;
        unit_of<S>(p, x, units, batch, m0, n0, sp, tile);
        const int k0 = split_start(sp, per, p.k);
        Job j{p.A, p.B, m0, n0, k0, min(k0 + per, p.k)};
        j.A.p = static_cast<const f16*>(j.A.p) + batch * p.per_a;
        j.B.p = static_cast<const f16*>(j.B.p) + batch * p.per_b;
        return j;
    };
    auto done = [&](int x, const f32x4 (&acc)[S::FM][S::FN]) {
        int batch, m0, n0, sp, tile;
        unit_of<S>(p, x, units, batch, m0, n0, sp, tile);
        if (PART)
            keep_part<S>(acc, p, tile, sp);
        else
            use_tile<S, H, O>(acc, m0, n0, batch, u);
    };
    int t = blockIdx.x;
    f32x4 acc[S::FM][S::FN];
    if constexpr (std::is_same<S, Big>::value) {
        TileStream<f16, LA, LB, PA, PB> stream(lds, job(t));
        for (; t < units; t += gridDim.x) {
            stream.multiply(acc, [&](Job& j) {
                const int x = t + gridDim.x;
                if (x < units) j = job(x);
                return x < units;
            });
            done(t, acc);
        }
    } else {
        const Job j = job(t);
        gemm_tile<f16, S, LA, LB, PA, PB>(j.A, j.B, j.m0, j.n0, j.kbeg, j.kend, lds, acc);
        done(t, acc);
    }
}
// adds a tile's splits in order; a workgroup for every two fragment rows, because there are few tiles where there are splits
template <class S, class H, class O>
__global__ __launch_bounds__(S::T) void ortho_finish_kernel(ProductArgs p, UseArgs u) {
    int batch, m0, n0;
    const int tile = blockIdx.x, i = blockIdx.y * 2;
    tile_of<S>(p, tile, gridDim.x / p.batch, batch, m0, n0);
    const f32x4* q = reinterpret_cast<const f32x4*>(p.part) + (long long)tile * p.splits * (S::BM * S::BN / 4) + threadIdx.x +
                     i * S::FN * S::T;
    constexpr int F = S::FM == 1 ? 1 : 2;
    f32x4 acc[F][S::FN];
#pragma unroll
    for (int j = 0; j < F * S::FN; ++j) acc[j / S::FN][j % S::FN] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s)
#pragma unroll
        for (int j = 0; j < F * S::FN; ++j) acc[j / S::FN][j % S::FN] += q[(long long)s * (S::BM * S::BN / 4) + j * S::T];
    use_rows<S, H, O>(acc[0], acc[F - 1], i, m0, n0, batch, u);
}

// ---- small matrices: all steps in one workgroup ------------------------------------------------------------------------
//
// X (small side s first, so a tall matrix is held transposed) and A, later B in its place, stay in LDS as two planes each;
// rows are padded to a multiple of 32 with zeros and by 8 elements more, which spreads the fragment reads over the banks.
// A wave forms fragments (16 x 16) of the products in registers; a result replaces its operand behind a barrier.  What bounds
// it is the latency of the chain norm -> 3 products a step -> store: 64 x 147 in 5 steps 33 us (71 as 17 launches).
constexpr int kSmallT = 512;

struct SmallPlan {
    int sp, lp, px, pa;      // sides padded to 32; row pitches of X and A
    int bytes;
};
__host__ __device__ inline SmallPlan small_plan(int s, int l) {
    SmallPlan p;
    p.sp = (s + 31) & ~31;
    p.lp = (l + 31) & ~31;
    p.px = p.lp + 8;
    p.pa = p.sp + 8;
    p.bytes = 4 * p.sp * (p.px + p.pa);
    return p;
}
// Fits LDS, and every wave's fragments its registers, and a few matrices are not faster in slabs (32 x 600 61 us here, 46 there;
// 16 x 400 40 and 42, 40 x 256 48 and 54) or, with more than 96 rows, in separate launches (128 x 128 85 and 72, three of 100 x
// 120 81 and 73, 96 x 128 69 and 71).  A stack gains nothing there: 200 of 16 x 500 45 us here, 111 in slabs; 32 of 100 x 120
// 82 and 82, 200 of them 86 and 159.
inline bool small_fits(int batch, int s, int l) {
    if (s > 128 || l > 4096 || (batch < 32 && (s > 96 || l > 448))) return false;
    const SmallPlan p = small_plan(s, l);
    return p.bytes <= 152 * 1024 && cdiv(p.lp / 16, kSmallT / 64 / (p.sp / 16)) <= (s > 64 ? 8 : 10);
}

struct Planes {
    f16* hi;
    f16* lo;
    int pitch;
};
__device__ __forceinline__ s16x8 rows_frag(const f16* p, int pitch, int r0, int k0, int lane) {
    return *reinterpret_cast<const s16x8*>(p + (r0 + (lane & 15)) * pitch + k0 + (lane >> 4) * 8);
}
// the same fragment of the transposed matrix: 16 columns from c0, k along the rows
__device__ __forceinline__ s16x8 cols_frag(const f16* p, int pitch, int c0, int k0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* lp;
    const f16* q = p + (k0 + (lane >> 4) * 8 + ((lane >> 2) & 3)) * pitch + c0 + (lane & 3) * 4;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 4 * pitch));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
// A wave's fragments of a product: row block w % nr, column blocks w / nr, + G, .. (G waves share a row block; of nr = 6 row
// blocks two waves have none).  The result's row runs along the lanes (operand R), four columns per lane (operand C).  Blocks
// beyond the last repeat it, so that no branch keeps the loads of one k apart.
struct Share {
    int row, col, step, cols;    // this wave's row block, first column block and stride, column blocks there are
    bool has;
    __device__ __forceinline__ Share(int wave, int nr, int nc) {
        const int g = kSmallT / 64 / nr;
        row = wave % nr;
        col = wave / nr;
        step = g;
        cols = nc;
        has = col < g;
    }
    __device__ __forceinline__ int c0(int i) const {
        const int c = col + i * step;
        return (c < cols ? c : cols - 1) * 16;
    }
    __device__ __forceinline__ bool mine(int i) const { return has && col + i * step < cols; }
};
template <bool TRANS, int NF>
__device__ __forceinline__ void small_product(const Planes& R, const Planes& C, const Share& sh, int k, int lane,
                                              f32x4 (&acc)[NF]) {
#pragma unroll
    for (int i = 0; i < NF; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!sh.has) return;
    for (int k0 = 0; k0 < k; k0 += 32) {
        const s16x8 rh = rows_frag(R.hi, R.pitch, sh.row * 16, k0, lane), rl = rows_frag(R.lo, R.pitch, sh.row * 16, k0, lane);
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            s16x8 ch, cl;
            if (TRANS) {
                ch = cols_frag(C.hi, C.pitch, sh.c0(i), k0, lane);
                cl = cols_frag(C.lo, C.pitch, sh.c0(i), k0, lane);
            } else {
                ch = rows_frag(C.hi, C.pitch, sh.c0(i), k0, lane);
                cl = rows_frag(C.lo, C.pitch, sh.c0(i), k0, lane);
            }
            acc[i] = mfma(cl, rh, acc[i], f16());
            acc[i] = mfma(ch, rl, acc[i], f16());
            acc[i] = mfma(ch, rh, acc[i], f16());
        }
    }
}
struct SmallArgs {
    int m, n, steps;
    double eps;
};
// b: this wave's fragments of X X^T; leaves the polynomial B in A's place
template <int NA>
__device__ __forceinline__ void gram_to_poly(const Planes& A, const Share& sq, int s, int sp, int lane, const Step& a,
                                             f32x4 (&b)[NA]) {
    const int r = sq.row * 16 + (lane & 15), q = (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < NA; ++i)
        if (sq.mine(i)) {
            const float v[4] = {b[i][0] * a.gram, b[i][1] * a.gram, b[i][2] * a.gram, b[i][3] * a.gram};
            put4<3>(A.hi + r * A.pitch + sq.c0(i) + q, A.lo - A.hi, v);
        }
    __syncthreads();
    small_product<false, NA>(A, A, sq, sp, lane, b);
#pragma unroll
    for (int i = 0; i < NA; ++i)
        if (sq.mine(i)) {
            const int c = sq.c0(i) + q;
            const f16x4 h = *reinterpret_cast<const f16x4*>(A.hi + r * A.pitch + c);
            const f16x4 w = *reinterpret_cast<const f16x4*>(A.lo + r * A.pitch + c);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                b[i][e] = fmaf(a.cc, b[i][e], a.cb * ((float)h[e] + (float)w[e])) + (c + e == r && r < s ? a.ca : 0.f);
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NA; ++i)
        if (sq.mine(i)) {
            const float v[4] = {b[i][0], b[i][1], b[i][2], b[i][3]};
            put4<3>(A.hi + r * A.pitch + sq.c0(i) + q, A.lo - A.hi, v);
        }
    __syncthreads();
}

// NA, NX: fragments a wave holds of the square products and of X
template <class O, int NA, int NX>
__global__ __launch_bounds__(kSmallT) void ortho_small_kernel(const O* __restrict__ g, O* __restrict__ out, SmallArgs a, Steps steps) {
    extern __shared__ __align__(16) char lds[];
    __shared__ double red[kSmallT / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool wide = a.m <= a.n;
    const int s = wide ? a.m : a.n, l = wide ? a.n : a.m, mn = a.m * a.n;
    const SmallPlan p = small_plan(s, l);
    Planes X{reinterpret_cast<f16*>(lds), reinterpret_cast<f16*>(lds) + p.sp * p.px, p.px};
    Planes A{X.lo + p.sp * p.px, X.lo + p.sp * (p.px + p.pa), p.pa};
    const O* gm = g + (long long)blockIdx.x * mn;
    O* om = out + (long long)blockIdx.x * mn;
    for (int i = tid; i < p.sp * p.px / 2; i += kSmallT) reinterpret_cast<int*>(X.hi)[i] = reinterpret_cast<int*>(X.lo)[i] = 0;
    // eight loads under way at a time, in both passes over the matrix
    double t = 0.0;
    for (int i0 = tid; i0 < mn; i0 += 8 * kSmallT) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = i0 + u * kSmallT < mn ? (float)gm[i0 + u * kSmallT] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) t += (double)x[u] * x[u];
    }
    const double inv = 1.0 / (sqrt(sum_all<kSmallT>(t, red)) + a.eps) * kXs;
    const int dr = kSmallT / a.n, dc = kSmallT - dr * a.n;      // from one element of a thread to its next
    int r0 = tid / a.n, c0 = tid - r0 * a.n;
    for (int i0 = tid; i0 < mn; i0 += 8 * kSmallT) {
        float x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = i0 + u * kSmallT < mn ? (float)gm[i0 + u * kSmallT] : 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int at = wide ? r0 * p.px + c0 : c0 * p.px + r0;
            f16 h, w;
            split16((float)(x[u] * inv), h, w);
            if (i0 + u * kSmallT < mn) {
                X.hi[at] = h;
                X.lo[at] = w;
            }
            r0 += dr;
            c0 += dc;
            if (c0 >= a.n) {
                c0 -= a.n;
                ++r0;
            }
        }
    }
    __syncthreads();
    const int ns = p.sp / 16, nl = p.lp / 16;
    const Share sq(wave, ns, ns), sx(wave, ns, nl);
    const int r = sq.row * 16 + (lane & 15), q = (lane >> 4) * 4;
    for (int step = 0; step < a.steps; ++step) {
        f32x4 b[NA];
        small_product<false, NA>(X, X, sq, p.lp, lane, b);
        const Step st = steps.s[step];
        gram_to_poly<NA>(A, sq, s, p.sp, lane, st, b);
        f32x4 x[NX];
        small_product<true, NX>(A, X, sx, p.sp, lane, x);
        const bool last = step + 1 == a.steps;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NX; ++i)
            if (sx.mine(i)) {
                const int c = sx.c0(i) + q;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = x[i][e] * st.next;
                if (!last) {
                    put4<3>(X.hi + r * p.px + c, X.lo - X.hi, v);
                } else if (r < s) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (c + e < l) om[wide ? r * a.n + c + e : (c + e) * a.n + r] = (O)v[e];
                }
            }
        __syncthreads();
    }
}

// ---- a small side of up to 64 and a longer other one: a launch a step ---------------------------------------------------
//
// A workgroup owns a slab of X's columns.  A launch adds all slabs' parts of A = X X^T (every workgroup for itself: 16 KB a slab
// at s = 64), forms B from it, multiplies its slab and leaves the slab's part of the next A.  What bounds a step is its chain
// of latencies, 9 us, once instead of the 3 to 5 times of separate products: 64 x 576 in 5 steps 98 -> 56 us.
struct SlabArgs {
    SmallArgs a;
    Step step;                      // not the first launch's
    int w, slabs, first, last;      // columns of a slab, a multiple of 32
    const double* norm;
    int blocks;
    f16* x;                         // [matrix][slab][plane][sp][w]
    const f32x4* old;               // parts of A: [matrix][slab][fragment of a wave][thread]
    f32x4* part;
};
template <class O, int NA, int NX>
__global__ __launch_bounds__(kSmallT) void ortho_slab_kernel(const O* __restrict__ g, O* __restrict__ out, SlabArgs p) {
    extern __shared__ __align__(16) char lds[];
    __shared__ double red[kSmallT / 64];
    const SmallArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool wide = a.m <= a.n;
    const int s = wide ? a.m : a.n, l = wide ? a.n : a.m, sp = (s + 31) & ~31, px = p.w + 8, pa = sp + 8;
    const int c_beg = blockIdx.x * p.w, wc = min(p.w, l - c_beg), slab = blockIdx.y * p.slabs + blockIdx.x;
    Planes X{reinterpret_cast<f16*>(lds), reinterpret_cast<f16*>(lds) + sp * px, px};
    Planes A{X.lo + sp * px, X.lo + sp * (px + pa), pa};
    f16* keep = p.x + (long long)slab * 2 * sp * p.w;
    const O* gm = g + (long long)blockIdx.y * a.m * a.n;
    O* om = out + (long long)blockIdx.y * a.m * a.n;
    const int ns = sp / 16, nl = p.w / 16;
    const Share sq(wave, ns, ns), sx(wave, ns, nl);
    const int r = sq.row * 16 + (lane & 15), q = (lane >> 4) * 4;
    f32x4 b[NA];
    if (p.first) {
        for (int i = tid; i < sp * px / 2; i += kSmallT) reinterpret_cast<int*>(X.hi)[i] = reinterpret_cast<int*>(X.lo)[i] = 0;
        const double inv = inverse_norm<kSmallT>(p.norm + (long long)blockIdx.y * p.blocks, p.blocks, a.eps, red) * kXs;
        // the matrix's own rows along the lanes
        const int rows = wide ? s : wc, cols = wide ? wc : s;
        const O* src = gm + (wide ? (long long)c_beg : (long long)c_beg * a.n);
        for (int y = wave; y < rows; y += kSmallT / 64)
#pragma unroll 4
            for (int x = lane; x < cols; x += 64) {
                f16 h, w;
                split16((float)((float)src[(long long)y * a.n + x] * inv), h, w);
                const int at = wide ? y * px + x : x * px + y;
                X.hi[at] = h;
                X.lo[at] = w;
            }
    } else {
        for (int i = tid; i < sp * p.w / 4; i += kSmallT) {      // chunks of 8, both planes
            const int plane = i >= sp * p.w / 8, k = i - (plane ? sp * p.w / 8 : 0), y = k / (p.w / 8), x = k % (p.w / 8) * 8;
            *reinterpret_cast<i32x4*>((plane ? X.lo : X.hi) + y * px + x) =
                *reinterpret_cast<const i32x4*>(keep + (plane ? sp * p.w : 0) + y * p.w + x);
        }
#pragma unroll
        for (int i = 0; i < NA; ++i) b[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        const f32x4* old = p.old + (long long)blockIdx.y * p.slabs * NA * kSmallT + tid;
#pragma unroll 2
        for (int j = 0; j < p.slabs; ++j)
#pragma unroll
            for (int i = 0; i < NA; ++i) b[i] += old[(j * NA + i) * kSmallT];
        gram_to_poly<NA>(A, sq, s, sp, lane, p.step, b);
        f32x4 x[NX];
        small_product<true, NX>(A, X, sx, sp, lane, x);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NX; ++i)
            if (sx.mine(i)) {
                const int c = sx.c0(i) + q;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = x[i][e] * p.step.next;
                if (!p.last) {
                    put4<3>(X.hi + r * px + c, X.lo - X.hi, v);
                    put4<3>(keep + r * p.w + c, sp * p.w, v);
                } else if (r < s) {
                    if (wide) {
                        put_row4(om + (long long)r * a.n + c_beg, c, wc, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < wc) om[(long long)(c_beg + c + e) * a.n + r] = (O)v[e];
                    }
                }
            }
        if (p.last) return;
    }
    __syncthreads();
    if (p.first)
        for (int i = tid; i < sp * p.w / 4; i += kSmallT) {
            const int plane = i >= sp * p.w / 8, k = i - (plane ? sp * p.w / 8 : 0), y = k / (p.w / 8), x = k % (p.w / 8) * 8;
            *reinterpret_cast<i32x4*>(keep + (plane ? sp * p.w : 0) + y * p.w + x) =
                *reinterpret_cast<const i32x4*>((plane ? X.lo : X.hi) + y * px + x);
        }
    small_product<false, NA>(X, X, sq, p.w, lane, b);
    f32x4* to = p.part + (long long)slab * NA * kSmallT + tid;
#pragma unroll
    for (int i = 0; i < NA; ++i) to[i * kSmallT] = b[i];
}

template <class O>
__global__ __launch_bounds__(256) void ortho_only_scale_kernel(const void* __restrict__ g, double eps,
                                                               const double* __restrict__ part, int blocks, long long mn,
                                                               void* __restrict__ out) {
    __shared__ double s[4];
    const double inv = inverse_norm<256>(part + (long long)blockIdx.y * blocks, blocks, eps, s);
    const long long base = blockIdx.y * mn;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < mn; i += gridDim.x * 256ll)
        static_cast<O*>(out)[base + i] = (O)(float)((float)static_cast<const O*>(g)[base + i] * inv);
}

struct OrthoPlan {
    int s, l, sp, np, blocks;                 // smaller and larger side; row pitch of A and of X
    Cut gram, poly, apply;
    bool light, small;
    int slab, slabs;                          // columns of a slab (0: not that path), slabs
    size_t norm, x0, x1, a, b, da, part, total;
};
int tiles_of(ShapeId id, int M, int N, bool tri) {
    const int b = side_of(id), m = cdiv(M, b), n = cdiv(N, b);
    return tri ? m * (m + 1) / 2 : m * n;
}
size_t part_bytes(const Cut& c, int M, int N, bool tri, int batch) {
    const size_t b = side_of(c.shape);
    return c.splits > 1 ? (size_t)batch * tiles_of(c.shape, M, N, tri) * c.splits * b * b * 4 : 0;
}
OrthoPlan ortho_plan(int dtype, int batch, int m, int n, bool light) {      // light: where the sizes suit it
    OrthoPlan p;
    p.s = m < n ? m : n;
    p.l = m < n ? n : m;
    p.sp = pad8(p.s);
    p.np = pad8(n);
    p.blocks = norm_blocks((long long)m * n);
    // on smaller sides launches and latency are what a step takes, more than products (five steps of 256 x 1024: 116 us so, 105
    // with all planes; 128 x 4608 121 and 120, 300 x 1100 130 and 122, 384 x 4608 174 and 186; 512 x 512 119 and 126, 512 x 4608
    // 215 and 230, 1024 x 1024 205 and 252, 2048 x 2048 498 and 735)
    p.light = light && dtype == DS_BF16 && p.s >= 512;
    auto cut = [&](int M, int N, int K, int pairs, bool tri, bool strided) {
        return cut_of(
            [&](long long b) {
                const long long x = (M + b - 1) / b, y = (N + b - 1) / b;
                return batch * (tri ? x * (x + 1) / 2 : x * y);
            },
            (double)M * N * batch * (tri ? 0.5 : 1.0), K, pairs, true, strided, cu_count());
    };
    p.gram = cut(p.s, p.s, p.l, p.light ? 1 : 3, true, m > n);
    p.poly = cut(p.s, p.s, p.s, p.light ? 1 : 3, true, false);
    p.apply = cut(n, m, p.s, p.light ? 2 : 3, false, m <= n);
    const size_t x = align256((size_t)batch * m * p.np * 4), a = align256((size_t)batch * p.s * p.sp * 4);
    size_t part = part_bytes(p.gram, p.s, p.s, true, batch), q = part_bytes(p.poly, p.s, p.s, true, batch);
    if (q > part) part = q;
    q = part_bytes(p.apply, n, m, false, batch);
    if (q > part) part = q;
    p.small = small_fits(batch, p.s, p.l);
    const int s32 = (p.s + 31) & ~31;
    // (at s = 128 the parts are 64 KB a slab and the products of a slab 8 us: no gain over separate launches)
    p.slab = p.small || s32 > 64 ? 0 : p.l > 4096 ? 256 : 128;
    p.slabs = p.slab ? cdiv(p.l, p.slab) : 0;
    if ((size_t)p.slabs * s32 * s32 * 4 > (1u << 20)) p.slab = 0;       // parts that every workgroup reads
    size_t o = 0;
    p.norm = o; o += align256((size_t)batch * p.blocks * 8);
    if (p.small || p.slab) {
        p.x0 = o; o += align256((size_t)batch * p.slabs * s32 * p.slab * 4);
        const size_t parts = align256((size_t)batch * p.slabs * 2 * kSmallT * 16);
        p.a = o; o += parts;
        p.b = o; o += parts;
        p.x1 = p.da = p.part = p.total = o;
        return p;
    }
    p.x0 = o; o += x;
    p.x1 = o; o += x;
    p.a = o; o += a;
    p.b = o; o += a;
    p.da = o; o += align256((size_t)batch * p.s * 8);
    p.part = o; o += align256(part);
    p.total = o;
    return p;
}

int check_ortho(int batch, int m, int n) {
    if (batch <= 0 || m <= 0 || n <= 0) return DS_ERR_INVALID_ARG;
    if (m > DS_ORTHO_MAX_SIDE || n > DS_ORTHO_MAX_SIDE || batch > 65535) return DS_ERR_UNSUPPORTED;
    if ((m < n ? m : n) > (1 << 15)) return DS_ERR_UNSUPPORTED;   // tiles of one launch
    return DS_OK;
}

int check_call(int dtype, int batch, int m, int n, int steps, const double* co, double eps, Steps& st, bool& light) {
    if (!co || steps < 0 || !(eps >= 0)) return DS_ERR_INVALID_ARG;
    const int rc = check_ortho(batch, m, n);
    if (rc) return rc;
    if (steps > DS_ORTHO_MAX_STEPS || (dtype != DS_F32 && dtype != DS_F16 && dtype != DS_BF16)) return DS_ERR_UNSUPPORTED;
    if (!isfinite(co[0]) || !isfinite(co[1]) || !isfinite(co[2])) return DS_ERR_INVALID_ARG;
    return steps_of(co, steps, st, light) ? DS_OK : DS_ERR_UNSUPPORTED;
}

template <class S, Lay LA, Lay LB, int PA, int PB, class H, class O>
void product_shape(ProductArgs p, const UseArgs& u, int tiles, hipStream_t q) {
    const int units = tiles * p.splits;
    const int grid = std::is_same<S, Big>::value && units > cu_count() ? cu_count() : units;
    if (p.splits > 1) {
        ortho_product_kernel<S, LA, LB, PA, PB, How<kGram, false>, float, true><<<grid, S::T, 0, q>>>(p, u, units);
        ortho_finish_kernel<S, H, O><<<dim3(tiles, (S::FM + 1) / 2), S::T, 0, q>>>(p, u);
    } else {
        ortho_product_kernel<S, LA, LB, PA, PB, H, O, false><<<grid, S::T, 0, q>>>(p, u, units);
    }
}
template <Lay LA, Lay LB, int PA, int PB, class H, class O>
void product(const Cut& c, ProductArgs p, const UseArgs& u, int M, int N, hipStream_t q) {
    p.splits = c.splits;
    const int b = side_of(c.shape), tiles = tiles_of(c.shape, M, N, p.tri) * p.batch;
    p.mt = cdiv(M, b);
    p.nt = cdiv(N, b);
    if (c.shape == kBig)
        product_shape<Big, LA, LB, PA, PB, H, O>(p, u, tiles, q);
    else if (c.shape == kSq)
        product_shape<Sq, LA, LB, PA, PB, H, O>(p, u, tiles, q);
    else if (c.shape == kSmall)
        product_shape<Small, LA, LB, PA, PB, H, O>(p, u, tiles, q);
    else
        product_shape<Tiny, LA, LB, PA, PB, H, O>(p, u, tiles, q);
}

template <class O, bool LIGHT>
void ortho_steps(const OrthoPlan& p, int batch, int m, int n, int steps, const Steps& st, char* ws, void* out, hipStream_t q) {
    f16 *x = reinterpret_cast<f16*>(ws + p.x0), *y = reinterpret_cast<f16*>(ws + p.x1);
    f16 *a = reinterpret_cast<f16*>(ws + p.a), *b = reinterpret_cast<f16*>(ws + p.b);
    float *part = reinterpret_cast<float*>(ws + p.part), *da = reinterpret_cast<float*>(ws + p.da), *db = da + (long long)batch * p.s;
    const long long px = 2ll * m * p.np, lox = (long long)m * p.np, pa = 2ll * p.s * p.sp, loa = (long long)p.s * p.sp;
    const bool wide = m <= n;
    constexpr int P = LIGHT ? 1 : 2;      // planes of A, of B, and of X in A = X X^T
    for (int i = 0; i < steps; ++i) {
        const Operand X{x, p.np, lox, m, p.np}, A{a, p.sp, loa, p.s, p.sp}, B{b, p.sp, loa, p.s, p.sp};
        const Step& f = st.s[i];
        const ProductArgs pg{X, X, px, px, 0, 0, 1, p.l, 1, batch, part};
        const UseArgs ug{p.s, p.s, a, p.sp, loa, pa, nullptr, 0, f.gram, 0.f, 0.f, da, db, p.s, wide};
        if (wide)
            product<kK, kK, P, P, How<kGram, LIGHT>, float>(p.gram, pg, ug, p.s, p.s, q);
        else
            product<kM, kM, P, P, How<kGram, LIGHT>, float>(p.gram, pg, ug, p.s, p.s, q);
        const ProductArgs pp{A, A, pa, pa, 0, 0, 1, p.s, 1, batch, part};
        const UseArgs up{p.s, p.s, b, p.sp, loa, pa, a, pa, f.ca, f.cb, f.cc, da, db, p.s, wide};
        product<kK, kK, P, P, How<kPoly, LIGHT>, float>(p.poly, pp, up, p.s, p.s, q);
        const bool last = i + 1 == steps;
        const UseArgs ua{m, n, last ? out : y, p.np, lox, last ? (long long)m * n : px, nullptr, 0, f.next,
                         0.f, 0.f, da, db, p.s, wide};
        const ProductArgs pw{wide ? X : B, wide ? B : X, wide ? px : pa, wide ? pa : px, 0, 0, 0, p.s, 1, batch, part};
        if (wide) {
            if (last)
                product<kM, kK, 2, P, How<kLast, LIGHT>, O>(p.apply, pw, ua, n, m, q);
            else
                product<kM, kK, 2, P, How<kNext, LIGHT>, float>(p.apply, pw, ua, n, m, q);
        } else {
            if (last)
                product<kK, kK, P, 2, How<kLast, LIGHT>, O>(p.apply, pw, ua, n, m, q);
            else
                product<kK, kK, P, 2, How<kNext, LIGHT>, float>(p.apply, pw, ua, n, m, q);
        }
        f16* z = x;
        x = y;
        y = z;
    }
}

template <class O, int NA, int NX>
int small_launch(const void* g, void* out, int batch, const SmallArgs& a, const Steps& st, int bytes, hipStream_t q) {
    if (bytes > 64 * 1024) {   // what a kernel may ask for without saying so
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&ortho_small_kernel<O, NA, NX>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return (int)e;
    }
    ortho_small_kernel<O, NA, NX><<<batch, kSmallT, bytes, q>>>(static_cast<const O*>(g), static_cast<O*>(out), a, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DS_OK : (int)e;
}

template <class O, int NA, int NX>
int slab_launch(const OrthoPlan& p, const void* g, void* out, int batch, const SmallArgs& a, const Steps& st, char* ws,
                hipStream_t q) {
    const int s32 = (p.s + 31) & ~31, bytes = 4 * s32 * (p.slab + 8 + s32 + 8);
    if (bytes > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&ortho_slab_kernel<O, NA, NX>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != hipSuccess) return (int)e;
    }
    f32x4* parts[2] = {reinterpret_cast<f32x4*>(ws + p.a), reinterpret_cast<f32x4*>(ws + p.b)};
    double* norm = reinterpret_cast<double*>(ws + p.norm);
    ortho_norm_kernel<O><<<dim3(p.blocks, batch), 256, 0, q>>>(static_cast<const O*>(g), (long long)a.m * a.n, norm);
    for (int i = 0; i <= a.steps; ++i) {
        const SlabArgs b{a, st.s[i > 0 ? i - 1 : 0], p.slab, p.slabs, i == 0, i == a.steps, norm, p.blocks, reinterpret_cast<f16*>(ws + p.x0),
                         parts[(i + 1) & 1], parts[i & 1]};
        ortho_slab_kernel<O, NA, NX><<<dim3(p.slabs, batch), kSmallT, bytes, q>>>(static_cast<const O*>(g), static_cast<O*>(out), b);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DS_OK : (int)e;
}

template <class O>
int ortho_any(const OrthoPlan& p, const void* g, int dtype, int batch, int m, int n, int steps, const Steps& st, double eps,
              void* out, char* ws, hipStream_t q) {
    if (steps > 0 && (p.small || p.slab)) {
        const SmallArgs a{m, n, steps, eps};
        const SmallPlan sp = small_plan(p.s, p.l);
        if (p.slab) {
            const int nx = cdiv(p.slab / 16, kSmallT / 64 / (sp.sp / 16));
            return nx <= 2   ? slab_launch<O, 2, 2>(p, g, out, batch, a, st, ws, q)
                   : nx <= 5 ? slab_launch<O, 2, 5>(p, g, out, batch, a, st, ws, q)
                             : slab_launch<O, 2, 10>(p, g, out, batch, a, st, ws, q);
        }
        const int nx = cdiv(sp.lp / 16, kSmallT / 64 / (sp.sp / 16));      // fragments of X a wave holds
        if (sp.sp > 64) return small_launch<O, 8, 8>(g, out, batch, a, st, sp.bytes, q);
        return nx <= 2   ? small_launch<O, 2, 2>(g, out, batch, a, st, sp.bytes, q)
               : nx <= 5 ? small_launch<O, 2, 5>(g, out, batch, a, st, sp.bytes, q)
                         : small_launch<O, 2, 10>(g, out, batch, a, st, sp.bytes, q);
    }
    double* part = reinterpret_cast<double*>(ws + p.norm);
    const long long mn = (long long)m * n;
    ortho_norm_kernel<O><<<dim3(p.blocks, batch), 256, 0, q>>>(static_cast<const O*>(g), mn, part);
    if (steps == 0) {
        const int nb = cdiv(mn, 1024) < 4096 ? cdiv(mn, 1024) : 4096;
        ortho_only_scale_kernel<O><<<dim3(nb, batch), 256, 0, q>>>(g, eps, part, p.blocks, mn, out);
    } else {
        const int nb = cdiv((long long)m * p.np, 4096) < 2048 ? cdiv((long long)m * p.np, 4096) : 2048;
        ortho_load_kernel<O><<<dim3(nb, batch), 256, 0, q>>>(static_cast<const O*>(g), m, n, p.np, eps, part, p.blocks,
                                                          reinterpret_cast<f16*>(ws + p.x0), (long long)m * p.np,
                                                          2ll * m * p.np);
        if constexpr (std::is_same<O, bf16>::value) {
            if (p.light) ortho_steps<O, true>(p, batch, m, n, steps, st, ws, out, q);
        }
        if (!p.light) ortho_steps<O, false>(p, batch, m, n, steps, st, ws, out, q);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DS_OK : (int)e;
}

}  // namespace
}  // namespace ds

extern "C" {

size_t ds_orthogonalize_workspace_bytes(int dtype, int batch, int m, int n) {
    if (ds::check_ortho(batch, m, n)) return 0;
    const size_t a = ds::ortho_plan(dtype, batch, m, n, false).total, b = ds::ortho_plan(dtype, batch, m, n, true).total;
    return a > b ? a : b;
}

int ds_orthogonalize_check(int dtype, int batch, int m, int n, int steps, const double* coefficients, double eps) {
    ds::Steps st;
    bool light;
    return ds::check_call(dtype, batch, m, n, steps, coefficients, eps, st, light);
}

int ds_orthogonalize(const void* update, int dtype, int batch, int m, int n, int steps, const double* coefficients, double eps,
                     void* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!update || !out) return DS_ERR_INVALID_ARG;
    ds::Steps st;
    bool light;
    const int rc = ds::check_call(dtype, batch, m, n, steps, coefficients, eps, st, light);
    if (rc) return rc;
    if (((uintptr_t)out & 15) != 0) return DS_ERR_INVALID_ARG;
    const ds::OrthoPlan p = ds::ortho_plan(dtype, batch, m, n, light);
    if (!workspace || workspace_bytes < p.total || ((uintptr_t)workspace & 15) != 0) return DS_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    hipStream_t q = static_cast<hipStream_t>(stream);
    if (dtype == DS_F32) return ds::ortho_any<float>(p, update, dtype, batch, m, n, steps, st, eps, out, ws, q);
    if (dtype == DS_F16) return ds::ortho_any<ds::f16>(p, update, dtype, batch, m, n, steps, st, eps, out, ws, q);
    return ds::ortho_any<ds::bf16>(p, update, dtype, batch, m, n, steps, st, eps, out, ws, q);
}

}  // extern "C"
