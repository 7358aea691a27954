// ds_head.hip -- a linear classification head over V classes (depth bins, a large vocabulary), without keeping its logits:
// softmax cross entropy with its gradient (ds_linear_ce_*) and the expected bin centre under the softmax with its gradient
// (ds_bin_expect_*).
//
//   l = H W^T (rows x classes)        lse_r = log sum_v exp l_rv
//   cross entropy   loss_r = lse_r - l[r,t_r]      dl_rv = g_r (p_rv - [v = t_r])
//   expectation     E_r = sum_v p_rv c_v           dl_rv = g_r p_rv (c_v - E_r)
//   dH = dl W,  dW = dl^T H
//
// Forward: a workgroup forms a tile of l in registers and leaves three numbers per row and class tile (maximum, sum of
// exponentials, sum of exponentials times centres); a second launch joins the tiles of a row.  Backward: per piece of the
// classes, the tile is formed again, turned into dl with the saved maximum and sum and written once in 16 bits (two planes for fp32
// inputs and for smaller 16-bit heads); the two products read it in place, one as kK, one as kM operand.
//
// Rows whose target is ignore_index take no part: the kept rows are listed first (in order, so results do not depend on
// scheduling), everything after works on that list, and how long it is stays on the device.
#include "ds_gemm.h"
#include "ds_internal.h"
#include "../../include/depthsynth.h"
#include <algorithm>
#include <type_traits>

namespace ds {
namespace {

// planes of an operand; SPLIT: products a step, 1 (16-bit inputs) or 3 (fp32), or 2 (16-bit inputs, but dl in two planes)
template <int SPLIT>
constexpr int kP = SPLIT == 3 ? 2 : 1;
template <int SPLIT>
constexpr int kPdl = SPLIT > 1 ? 2 : 1;

enum Mode { kCE = 0, kExpect = 1 };
constexpr int kNone = -(1 << 30);   // no exponent

// What the forward leaves for the backward besides the softmax statistics: opaque to the caller.
constexpr int kReach = 16;          // places where workgroups meet, each in a cache line of its own
struct HeadState {
    int count;                      // rows kept
    unsigned amax_w;                // bits of max |weight|: the scale of its fp16 planes (fp32 inputs)
    int pad[30];
    struct {
        int most, pad[31];          // max over staged rows of the exponent above their largest feature (cross entropy)
    } reach[kReach];
};
struct Centers {
    unsigned most;       // bits of max |centre|
    int signs;           // 1: some are positive, 2: some are negative
};
struct BackState {
    int most;            // the largest exponent that a kept row takes part in dW with (kNone: no row does)
    Centers centers;
    int pad[13];
};


__device__ __forceinline__ float from_bits(unsigned u) { return __builtin_bit_cast(float, u); }

// max over finite magnitudes: an infinity or a NaN in one place must not take the scale from all others
__device__ __forceinline__ float finite_abs(float x) { return __builtin_isfinite(x) ? fabsf(x) : 0.f; }

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// ------------------------------------------------------------------------------------------------ kept rows, in order
constexpr int kListT = 1024, kListPer = 16, kListBlock = kListT * kListPer;

__global__ void head_init_kernel(HeadState* st, int rows) {
    st->count = rows;
    st->amax_w = 0;
}

// Up to four workgroups count what comes before them themselves: a launch (3 us of the host's time) less, and no slower (61440
// rows: 15 us, against 7.3 and 7.7 in two launches; every further workgroup waits for 2 us more).
constexpr int kListAlone = 4;

// rows kept per 16384 (only launched for more workgroups than that)
__global__ __launch_bounds__(kListT) void count_rows_kernel(const long long* __restrict__ target, int n, long long ignore,
                                                            int* __restrict__ counts) {
    __shared__ int s[kListT / 64];
    int c = 0;
    long long t[kListPer];
#pragma unroll
    for (int i = 0; i < kListPer; ++i) {
        const long long r = (long long)blockIdx.x * kListBlock + i * kListT + threadIdx.x;
        t[i] = r < n ? target[r] : ignore;
    }
#pragma unroll
    for (int i = 0; i < kListPer; ++i) c += __popcll(__ballot(t[i] != ignore));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = c;
    __syncthreads();
    if (threadIdx.x == 0) {
        int t = 0;
        for (int i = 0; i < kListT / 64; ++i) t += s[i];
        counts[blockIdx.x] = t;
    }
}

// rows[j] = j-th kept row, tgt[j] = its class (-1 where it is none of 0..V-1: its loss is NaN); each_loss (may be NULL) of
// the others is 0
__global__ __launch_bounds__(kListT) void list_rows_kernel(const long long* __restrict__ target, int n, int V, long long ignore,
                                                           const int* __restrict__ counts, HeadState* __restrict__ st,
                                                           int* __restrict__ rows, int* __restrict__ tgt,
                                                           float* __restrict__ each_loss) {
    constexpr int kW = kListT / 64;
    __shared__ int s[kListPer * kW + 1];
    __shared__ int before;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) before = 0;
    __syncthreads();
    long long t[kListPer];
    if (blockIdx.x > 0) {   // integer sums: any order gives the same
        int c = 0;
        if (counts) {
            for (int i = threadIdx.x; i < (int)blockIdx.x; i += kListT) c += counts[i];
        } else {
            for (int b = 0; b < (int)blockIdx.x; ++b) {      // whole blocks of rows
#pragma unroll
                for (int i = 0; i < kListPer; ++i) t[i] = target[b * kListBlock + i * kListT + threadIdx.x];
#pragma unroll
                for (int i = 0; i < kListPer; ++i) c += __popcll(__ballot(t[i] != ignore));
            }
            if (lane != 0) c = 0;
        }
        if (c) atomicAdd(&before, c);
    }
    const long long base = (long long)blockIdx.x * kListBlock;
    unsigned long long m[kListPer];
#pragma unroll
    for (int i = 0; i < kListPer; ++i) {
        const long long r = base + i * kListT + threadIdx.x;
        t[i] = r < n ? target[r] : ignore;
        m[i] = __ballot(t[i] != ignore);
        if (lane == 0) s[i * kW + wave] = __popcll(m[i]);
    }
    __syncthreads();
    if (wave == 0) {   // exclusive prefix over the 256 counts, four a lane
        int v[4], sum = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = s[lane * 4 + e];
            sum += v[e];
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(inc, o, 64);
            if (lane >= o) inc += u;
        }
        int ex = inc - sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[lane * 4 + e] = ex;
            ex += v[e];
        }
        if (lane == 63) s[kListPer * kW] = ex;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kListPer; ++i) {
        const long long r = base + i * kListT + threadIdx.x;
        if (t[i] != ignore) {
            const int j = before + s[i * kW + wave] + __popcll(m[i] & ((1ull << lane) - 1));
            rows[j] = (int)r;
            tgt[j] = t[i] >= 0 && t[i] < V ? (int)t[i] : -1;
        } else if (r < n && each_loss) {
            each_loss[r] = 0.f;
        }
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
        st->count = before + s[kListPer * kW];
        st->amax_w = 0;
    }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x < kReach) st->reach[threadIdx.x].most = kNone;
}
static_assert(kListPer * kListT / 64 == 256, "the prefix handles four counts a lane");

// --------------------------------------------------------------------------------------------------- staged operands
// Row-wise passes over a matrix: a wave takes 64 / L rows at once, L lanes a row, VEC elements (16 bytes) a lane; L is the power
// of two that a row of D elements needs, at most 64.
inline int lanes_for(int vectors) {
    int l = 1;
    while (l < vectors && l < 64) l <<= 1;
    return l;
}
template <class IT, int VEC>
struct Vec {
    typedef IT type __attribute__((ext_vector_type(VEC)));
};
// VEC elements of a row from element d on, zero behind its last; rows need only their type's alignment (gfx950 loads 16 bytes
// from any address)
template <class IT, int VEC>
__device__ __forceinline__ void load_vec(const IT* row, int d, int D, IT (&x)[VEC]) {
    typedef typename Vec<IT, VEC>::type loose __attribute__((aligned(sizeof(IT))));
    if (d + VEC <= D) {
        const loose v = *reinterpret_cast<const loose*>(row + d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = d + e < D ? row[d + e] : (IT)0.f;
    }
}

// max |weight|; order-independent, so repeatable.  One workgroup writes what it finds, and the row count if set_count gives it;
// where there are more, *st was cleared before.
template <class IT, int VEC>
__global__ __launch_bounds__(256) void amax_kernel(const IT* __restrict__ w, HeadState* __restrict__ st, int V, int D, int L,
                                                   int set_count) {
    const bool alone = gridDim.x == 1;
    const int lane = threadIdx.x & 63, sub = lane & (L - 1), R = 64 / L;
    float m = 0.f;
    constexpr int U = 4;        // rows under way at a time
    const int hop = gridDim.x * 4 * R;
    for (int r0 = ((int)blockIdx.x * 4 + (threadIdx.x >> 6)) * R + lane / L; r0 < V; r0 += hop * U)
        for (int d = sub * VEC; d < D; d += L * VEC) {
            IT v[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) load_vec<IT, VEC>(w + (long long)min(r0 + u * hop, V - 1) * D, d, D, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) m = fmaxf(m, finite_abs((float)v[u][e]));
        }
    m = wave_max(m);
    __shared__ float s[4];
    if (lane == 0) s[threadIdx.x >> 6] = m;
    __syncthreads();
    // one atomic a workgroup: they all meet in one place, 20 ns each
    if (threadIdx.x == 0) {
        m = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        if (alone) st->amax_w = __builtin_bit_cast(unsigned, m);
        if (alone && set_count) st->count = set_count;
        if (!alone && m > 0.f) atomicMax(&st->amax_w, __builtin_bit_cast(unsigned, m));
    }
}

// Rows of one or two matrices (one launch) packed with a row pitch of Dp elements, zero behind D; fp32 as two scaled fp16
// planes: the weight under one scale (dH sums over its rows), every row of the features under its own, so that a row's result
// does not depend on what else is in the batch.  Workgroups [first, first + blocks) take a source.
struct Source {
    const void* x;
    long long ld;
    const int* rows;           // listed rows (NULL: in order)
    const int* cnt;            // how many, on the device (NULL: n)
    int n;
    const unsigned* amax;      // scale of all rows (fp32), or
    int* shifts;               // every row's own, left here: 2^shift brings its largest element into [2^14, 2^15)
    HeadState* reach;          // NULL: not asked for
    void* y;
    long long lo;
    int first, blocks;         // blocks 0: not there
};
constexpr int kReachTop = 15;      // a row with that shift has features below 2^15 as stored
constexpr int kZeroShift = 163;    // of a row without finite elements but zeros: it reaches nowhere
// Own: rows find their own shifts; kept: and one load brings a whole row
enum StageHow { kSame, kOwn, kOwnKept };
template <class IT, class T, int SPLIT, int VEC, StageHow HOW>
__device__ __forceinline__ int stage_rows(const Source& s, int D, int Dp, int L) {
    const IT* x = static_cast<const IT*>(s.x);
    const int c = s.cnt ? *s.cnt : s.n;
    const int lane = threadIdx.x & 63, sub = lane & (L - 1), R = 64 / L;
    constexpr int U = 4;
    int shift[U], reach = kNone;
    const int same = SPLIT == 3 && HOW == kSame ? shift_for(from_bits(*s.amax)) : 0;
    const int hop = s.blocks * 4 * R;
    for (int r0 = (((int)blockIdx.x - s.first) * 4 + (threadIdx.x >> 6)) * R + lane / L; r0 < c; r0 += hop * U) {
        auto load = [&](int d, IT (&v)[U][VEC]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(r0 + u * hop, c - 1);
                load_vec<IT, VEC>(x + (s.rows ? s.rows[r] : r) * s.ld, d, D, v[u]);
            }
        };
        auto store = [&](int d, const IT (&v)[U][VEC]) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * hop;
                if (r >= c) continue;
                T* q = static_cast<T*>(s.y) + (long long)r * Dp + d;
                typename Vec<T, VEC>::type h, l;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if constexpr (SPLIT == 3) {
                        f16 a, b;
                        split16(ldexpf((float)v[u][e], HOW == kSame ? same : shift[u]), a, b);
                        h[e] = a;
                        l[e] = b;
                    } else {
                        h[e] = v[u][e];
                    }
                }
                *reinterpret_cast<typename Vec<T, VEC>::type*>(q) = h;
                if (SPLIT == 3) *reinterpret_cast<typename Vec<T, VEC>::type*>(q + s.lo) = l;
            }
        };
        float m[U] = {};
        auto largest = [&](const IT (&v)[U][VEC]) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < VEC; ++e) m[u] = fmaxf(m[u], finite_abs((float)v[u][e]));
        };
        auto settle = [&] {
            // (all lanes of a row are here: L divides 64 and r0 is the row's)
            for (int o = 1; o < L; o <<= 1)
#pragma unroll
                for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor(m[u], o, 64));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                shift[u] = m[u] > 0.f ? shift_for(m[u]) : kZeroShift;
                if (sub == 0 && r0 + u * hop < c) {
                    s.shifts[r0 + u * hop] = shift[u];
                    reach = max(reach, kReachTop - shift[u]);
                }
            }
        };
        const int d0 = sub * VEC;
        if constexpr (HOW == kOwnKept) {
            IT v[U][VEC] = {};
            if (d0 < Dp) load(d0, v);
            largest(v);
            settle();
            if (d0 < Dp) store(d0, v);
        } else {
            if (HOW == kOwn) {
                for (int d = d0; d < Dp; d += L * VEC) {
                    IT v[U][VEC];
                    load(d, v);
                    largest(v);
                }
                settle();
            }
            for (int d = d0; d < Dp; d += L * VEC) {
                IT v[U][VEC];
                load(d, v);
                store(d, v);
            }
        }
    }
    return reach;
}
template <class IT, class T, int SPLIT, int VEC>
__global__ __launch_bounds__(256) void stage_kernel(Source s0, Source s1, int D, int Dp, int L) {
    const bool second = s1.blocks > 0 && (int)blockIdx.x >= s1.first;
    const Source s = second ? s1 : s0;
    // (bf16 rows need no shifts; fp16 rows are left as they are, but dW wants to know)
    if (std::is_same<T, bf16>::value || !s.shifts) {
        stage_rows<IT, T, SPLIT, VEC, kSame>(s, D, Dp, L);
        return;
    }
    int reach = Dp <= L * VEC ? stage_rows<IT, T, SPLIT, VEC, kOwnKept>(s, D, Dp, L)
                              : stage_rows<IT, T, SPLIT, VEC, kOwn>(s, D, Dp, L);
    if (SPLIT == 3 && s.reach) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) reach = max(reach, __shfl_xor(reach, o, 64));
        __shared__ int top[4];
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = reach;
        __syncthreads();
        reach = max(max(top[0], top[1]), max(top[2], top[3]));
        if (threadIdx.x == 0 && reach > kNone) atomicMax(&s.reach->reach[blockIdx.x % kReach].most, reach);
    }
}

// exponent of the weight's planes
__device__ __forceinline__ int weight_shift(const HeadState* st) { return shift_for(from_bits(st->amax_w)); }

// ------------------------------------------------------------------------------------------------------------ forward
// Statistics of one tile of l^T: classes along m, rows along n, so that a lane holds 4 FM classes of FN rows and most of the
// softmax stays inside it.  part: three planes [class tile][row].  red: [WM][BN][3] floats in LDS; behind a barrier on entry
// and on return.
struct StatsArgs {
    int V;
    const int* shifts;   // exponents of the rows' planes
    const int* tgt;
    const float* centers;
    float* tlogit;
    float* part;
    long long plane;
    int ld_part;
    int set_count;       // not 0: so many rows, and *st gets to know it here
};
__device__ __forceinline__ int rows_of(const StatsArgs& a, HeadState* st) {
    if (a.set_count && blockIdx.x == 0 && threadIdx.x == 0) st->count = a.set_count;
    return a.set_count ? a.set_count : st->count;
}
template <class S, int SPLIT, int MODE>
__device__ __forceinline__ void stats_of_tile(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int cnt, const HeadState* st,
                                              const StatsArgs& a, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, v0 = m0 + wm * S::FM * 16 + (lane >> 4) * 4;
    const int ws = SPLIT == 3 ? weight_shift(st) : 0;
    const bool edge = m0 + S::BM > a.V;      // only the last class tile has classes that do not exist
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int nl = (wn * S::FN + j) * 16 + (lane & 15), n = n0 + nl;
        if (SPLIT == 3) {
            const int shift = -ws - (n < cnt ? a.shifts[n] : 0);
#pragma unroll
            for (int i = 0; i < S::FM; ++i) acc[i][j] = scaled(acc[i][j], shift);
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v0 + i * 16 + e >= a.V) acc[i][j][e] = -INFINITY;
        }
        if (MODE == kCE) {
            const int t = n < cnt ? a.tgt[n] - v0 : -1;     // the row's class, counted from this lane's first one
            if (t >= 0 && t < S::FM * 16 && (t & 15) < 4) {
                float l = 0.f;
#pragma unroll
                for (int i = 0; i < S::FM; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (t == i * 16 + e) l = acc[i][j][e];
                a.tlogit[n] = l;
            }
        }
        float mx = -INFINITY, s = 0.f, sc = 0.f;
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx = fmaxf(mx, acc[i][j][e]);     // passes over NaN, which reaches the sum below
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = exp_of(acc[i][j][e] - ref);
                s += x;
                if (MODE == kExpect) sc = fmaf(x, edge && v0 + i * 16 + e >= a.V ? 0.f : a.centers[v0 + i * 16 + e], sc);
            }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        sc += __shfl_xor(sc, 16, 64);
        sc += __shfl_xor(sc, 32, 64);
        if (lane < 16) {
            float* q = red + (wm * S::BN + nl) * 3;
            q[0] = mx;
            q[1] = s;
            q[2] = sc;
        }
    }
    __syncthreads();
    for (int nl = threadIdx.x; nl < S::BN; nl += S::T) {
        if (n0 + nl >= cnt) break;
        float mx = -INFINITY, s = 0.f, sc = 0.f;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) mx = fmaxf(mx, red[(w * S::BN + nl) * 3]);
        const float ref = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) {
            const float* q = red + (w * S::BN + nl) * 3;
            const float f = exp_of(q[0] - ref);
            s += q[1] * f;
            sc += q[2] * f;
        }
        float* q = a.part + (long long)(m0 / S::BM) * a.ld_part + n0 + nl;
        q[0] = mx;
        q[a.plane] = s;
        if (MODE == kExpect) q[2 * a.plane] = sc;
    }
    __syncthreads();
}

template <class T, class S, int SPLIT, int MODE>
__global__ __launch_bounds__(S::T) void head_stats_kernel(Operand W, Operand H, HeadState* __restrict__ st, int D,
                                                          StatsArgs a) {
    __shared__ __align__(16) char lds[lds_bytes<S, kP<SPLIT>, kP<SPLIT>>()];
    const int vt = cdiv(a.V, S::BM);
    const int m0 = (int)(blockIdx.x % vt) * S::BM, n0 = (int)(blockIdx.x / vt) * S::BN;
    const int cnt = rows_of(a, st);
    if (n0 >= cnt) return;
    H.outer = cnt;
    f32x4 acc[S::FM][S::FN];
    gemm_tile<T, S, kK, kK, kP<SPLIT>, kP<SPLIT>>(W, H, m0, n0, 0, D, lds, acc);
    stats_of_tile<S, SPLIT, MODE>(acc, m0, n0, cnt, st, a, reinterpret_cast<float*>(lds));
}

// the same in tiles of 256 x 256, a workgroup going through several
template <class T, int SPLIT, int MODE>
__global__ __launch_bounds__(Big::T) void head_stats_big_kernel(Operand W, Operand H, HeadState* __restrict__ st, int D,
                                                                StatsArgs a) {
    __shared__ __align__(16) char lds[Big::kLds];
    __shared__ float red[Big::WM * Big::BN * 3];
    const int cnt = rows_of(a, st), mt = cdiv(a.V, Big::BM), nt = cdiv(cnt, Big::BN), tiles = mt * nt;
    int t = blockIdx.x;
    if (t >= tiles) return;
    H.outer = cnt;
    const Order order(tiles, mt, nt);
    auto job = [&](int u) {
        int m, n;
        order(u, m, n);
        return Job{W, H, m * Big::BM, n * Big::BN, 0, D};
    };
    TileStream<T, kK, kK, kP<SPLIT>, kP<SPLIT>> stream(lds, job(t));
    for (; t < tiles; t += gridDim.x) {
        const int m0 = stream.job.m0, n0 = stream.job.n0;
        f32x4 acc[Big::FM][Big::FN];
        stream.multiply(acc, [&](Job& j) {
            const int u = t + gridDim.x;
            if (u < tiles) j = job(u);
            return u < tiles;
        });
        stats_of_tile<Big, SPLIT, MODE>(acc, m0, n0, cnt, st, a, red);
    }
}

// joins the class tiles of a row: 32 rows x 8 lanes over the tiles
__global__ __launch_bounds__(256) void head_join_kernel(const float* __restrict__ part, long long plane, int ld_part, int tiles,
                                                        const HeadState* __restrict__ st, int mode,
                                                        const int* __restrict__ rows, const int* __restrict__ tgt,
                                                        const float* __restrict__ tlogit, float* __restrict__ top,
                                                        float* __restrict__ inv_sum, float* __restrict__ mean,
                                                        float* __restrict__ out, double* __restrict__ sums) {
    __shared__ float red[8][32][3];
    __shared__ double tot[32];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5, n = blockIdx.x * 32 + x;
    const int cnt = st->count;
    float mx = -INFINITY, s = 0.f, sc = 0.f;
    constexpr int U = 8;        // tiles under way at a time
    if (n < cnt)
        for (int t0 = y; t0 < tiles; t0 += 8 * U) {
            float m[U], a[U], c[U], nm = mx;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = t0 + u * 8 < tiles;
                const float* q = part + (long long)(t0 + u * 8) * ld_part + n;
                m[u] = in ? q[0] : -INFINITY;
                a[u] = in ? q[plane] : 0.f;
                c[u] = in && mode == kExpect ? q[2 * plane] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) nm = fmaxf(nm, m[u]);
            const float ref = nm == -INFINITY ? 0.f : nm, f0 = exp_of(mx - ref);
            s *= f0;
            sc *= f0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float f = exp_of(m[u] - ref);
                s = fmaf(a[u], f, s);
                sc = fmaf(c[u], f, sc);
            }
            mx = nm;
        }
    red[y][x][0] = mx;
    red[y][x][1] = s;
    red[y][x][2] = sc;
    __syncthreads();
    if (y == 0) {
        double loss = 0.0;
        if (n < cnt) {
            mx = red[0][x][0];
            for (int i = 1; i < 8; ++i) mx = fmaxf(mx, red[i][x][0]);
            const float ref = mx == -INFINITY ? 0.f : mx;
            s = sc = 0.f;
            for (int i = 0; i < 8; ++i) {
                const float f = exp_of(red[i][x][0] - ref);
                s += red[i][x][1] * f;
                sc += red[i][x][2] * f;
            }
            top[n] = ref;
            inv_sum[n] = 1.f / s;
            if (mode == kExpect) {
                out[n] = mean[n] = sc / s;
            } else {
                const float each = tgt[n] < 0 ? __builtin_nanf("") : (ref - tlogit[n]) + logf(s);
                if (sums)
                    loss = each;
                else
                    out[rows[n]] = each;
            }
        }
        tot[x] = loss;
    }
    if (!sums) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0.0;
        for (int i = 0; i < 32; ++i) a += tot[i];
        sums[blockIdx.x] = a;
    }
}

// the sum (mean) of the rows' losses, in a fixed order
__global__ __launch_bounds__(256) void loss_total_kernel(const double* __restrict__ sums, const HeadState* __restrict__ st,
                                                         int mean, int entries, float* __restrict__ out) {
    __shared__ double s[256];
    const int cnt = st->count, nb = entries > 0 ? entries : (cnt + 31) / 32;
    double a = 0.0;
    for (int i = threadIdx.x; i < nb; i += 256) a += sums[i];
    s[threadIdx.x] = a;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[0] = (float)(mean ? s[0] / cnt : s[0]);
}

// ----------------------------------------------------------------------------------------------------------- backward
// How dl is scaled: fp16 storage wants values of a fixed size, so a row of dl is kept as 2^14 dl / 2^e, where 2^e is above the
// row's upstream value, times the row's p |c - E| for the expectation; dH's rows are scaled back one by one, so that a row keeps
// its digits whatever the others' upstream is.  dW adds rows up, weighted with 2^e, and what is lost there is 2^-39 of the largest
// row's part.  bf16 has fp32's range and takes dl as it is.  All powers of two are exponents, for ldexpf: upstreams of 1e38 or
// 1e-38 are in range.
constexpr int kDlTop = 14;

// the least e with |x| < 2^e; 0 where there is none
__device__ __forceinline__ int exp_above(float x) { return x > 0.f && __builtin_isfinite(x) ? ilogbf(x) + 1 : 0; }
struct Upstream {
    const float* g;      // one value, or one per row of the caller
    int each, mean;
    const int* rows;     // caller's row of a kept row (NULL: the same)
    const float* expect; // E of a kept row (NULL: cross entropy)
};
__device__ __forceinline__ float upstream(const Upstream& u, int n, int cnt) {
    if (u.each) return u.g[u.rows ? u.rows[n] : n];
    return u.mean ? u.g[0] / cnt : u.g[0];
}
// p |c - E| < 2^e.  Centres of one sign: it is at most |E|, however far the largest centre is (a bin of 1e9 for "no depth" takes no
// digits from rows that are sure of another); else twice the largest.  As a factor 2^-e of the centres in float32's normal range,
// which leaves them below 2^100.
__device__ __forceinline__ int center_exp(const Centers& c, float E) {
    const int top = exp_above(from_bits(c.most)) + 1, own = c.signs == 3 ? top : max(exp_above(fabsf(E)) + 1, top - 100);
    return own < -125 ? -125 : (own > 126 ? 126 : own);
}
__device__ __forceinline__ int row_exp_of(const Upstream& u, const Centers& c, int n, float g) {
    return exp_above(fabsf(g)) + (u.expect ? center_exp(c, u.expect[n]) : 0);
}
// exponent e of a row: its upstream value's (g) and its centres', 0 where T needs none
template <class T>
__device__ __forceinline__ int row_exp(const Upstream& u, const BackState* bs, int n, float g) {
    return std::is_same<T, bf16>::value ? 0 : row_exp_of(u, u.expect ? bs->centers : Centers{0, 0}, n, g);
}
// exponent of a row of stored dl -> dl: this and the row's
template <class T>
constexpr int kDlExp = std::is_same<T, bf16>::value ? 0 : -kDlTop;
// What a row weighs in dW.  A product there is dl_r h_r; dl is stored under the row's exponent e, features of fp32
// under the row's own shift, so that a row takes part with 2^(e + 15 - shift), and that is brought to 2^most by the weight, at
// most 1 (most: the largest of the sums e + 15 - shift, or of e where features have one size for all, `reach` 0).  Rows
// without a gradient are left as they are.
__device__ __forceinline__ int weight_exp(float g, int e, int reach, int most) {
    return g != 0.f && __builtin_isfinite(g) && most > kNone ? e + reach - most : 0;
}
// the largest exponent that a row takes part with.  SPLIT 3: always with its features' reach
template <class T, int SPLIT>
__device__ __forceinline__ int most_of(const HeadState* st, const BackState* bs, const Upstream& u, int cnt) {
    if (std::is_same<T, bf16>::value) return 0;
    if (u.each) return bs->most;
    int r = SPLIT == 3 ? kNone : 0;
    if (SPLIT == 3)
        for (int i = 0; i < kReach; ++i) r = max(r, st->reach[i].most);
    return r == kNone ? kNone : r + exp_above(fabsf(upstream(u, 0, cnt)));
}
// exponent of sums over rows -> dW
template <class T, int SPLIT>
__device__ __forceinline__ int dw_exp(const HeadState* st, const BackState* bs, const Upstream& u, int cnt, bool reach) {
    if (std::is_same<T, bf16>::value) return 0;
    const int most = most_of<T, SPLIT>(st, bs, u, cnt);
    return kDlExp<T> + (most == kNone ? 0 : most) - (reach ? kReachTop : 0);
}

// bs->most (with the rows' shifts, or of float16 rows that lie as the caller left them the features themselves, where rows weigh
// with their reach) and the centres' size and signs, which every workgroup finds for itself; for upstreams that differ.  *bs is
// set by back_init_kernel before, unless one workgroup does it all (a launch less).
constexpr int kScaleT = 512, kScaleAlone = 16 * kScaleT;
__global__ void back_init_kernel(BackState* bs) { bs->most = kNone; }
struct Features {
    const int* shifts;   // of staged rows
    const f16* h;        // both NULL: not asked for
    long long ld;
    const int* rows;     // listed rows (NULL: in order)
    int D, L;
};
__global__ __launch_bounds__(kScaleT) void back_scale_kernel(Upstream u, const HeadState* __restrict__ st,
                                                             const float* __restrict__ centers, int V, Features f,
                                                             BackState* __restrict__ bs) {
    __shared__ float red[kScaleT / 64];
    __shared__ int top[kScaleT / 64], sign[kScaleT / 64];
    const int cnt = st->count, step = gridDim.x * kScaleT, i0 = blockIdx.x * kScaleT + threadIdx.x;
    const int lane = threadIdx.x & 63;
    Centers all{0, 0};
    if (centers) {
        float c = 0.f;
        int signs = 0;
#pragma unroll 4
        for (int v = threadIdx.x; v < V; v += kScaleT) {
            const float x = centers[v];
            c = fmaxf(c, finite_abs(x));
            signs |= x > 0.f ? 1 : x < 0.f ? 2 : 0;
        }
        c = wave_max(c);
        signs = (__ballot(signs & 1) ? 1 : 0) | (__ballot(signs & 2) ? 2 : 0);
        if (lane == 0) {
            red[threadIdx.x >> 6] = c;
            sign[threadIdx.x >> 6] = signs;
        }
        __syncthreads();
        for (int i = 0; i < kScaleT / 64; ++i) {
            c = fmaxf(c, red[i]);
            signs |= sign[i];
        }
        all = Centers{__builtin_bit_cast(unsigned, c), signs};
        if (blockIdx.x == 0 && threadIdx.x == 0) bs->centers = all;
    }
    int most = kNone;
    auto take = [&](int n, int more) {
        const float g = upstream(u, n, cnt);
        if (g != 0.f && __builtin_isfinite(g)) most = max(most, row_exp_of(u, all, n, g) + more);
    };
    if (f.h) {
        const int sub = lane & (f.L - 1), R = 64 / f.L;
        for (int n = i0 / 64 * R + lane / f.L; n < cnt; n += step / 64 * R) {
            const f16* row = f.h + (f.rows ? f.rows[n] : n) * f.ld;
            float m = 0.f;
            for (int d = sub * 8; d < f.D; d += f.L * 8) {
                f16 x[8];
                load_vec<f16, 8>(row, d, f.D, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs((float)x[e]));
            }
            for (int o = 1; o < f.L; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            if (m > 0.f) take(n, exp_above(m));
        }
    } else {
#pragma unroll 4
        for (int n = i0; n < cnt; n += step) take(n, f.shifts ? kReachTop - f.shifts[n] : 0);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
    if (lane == 0) top[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < kScaleT / 64; ++i) most = max(most, top[i]);
    if (gridDim.x == 1)
        bs->most = most;
    else if (most > kNone)
        atomicMax(&bs->most, most);
}

// The features of kept rows times 2^weight_exp, for dW, whose other operand holds every row of dl at full size (float16: from
// their own size to that of fp32's planes).  Eight elements a thread.
template <int SPLIT>
__global__ __launch_bounds__(256) void fold_rows_kernel(Operand H, const int* __restrict__ shifts,
                                                        const HeadState* __restrict__ st, Upstream u,
                                                        const BackState* __restrict__ bs, f16* __restrict__ y, int Dp,
                                                        long long lo) {
    const int cnt = st->count, q = Dp / 8, most = most_of<f16, SPLIT>(st, bs, u, cnt);
    const long long all = (long long)cnt * q;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
        const int n = (int)(i / q), d = (int)(i - (long long)n * q) * 8;
        const float g = upstream(u, n, cnt);
        const int e = weight_exp(g, row_exp<f16>(u, bs, n, g), kReachTop - (SPLIT == 3 ? shifts[n] : 0), most);
#pragma unroll
        for (int p = 0; p < (SPLIT == 3 ? 2 : 1); ++p) {
            f16x8 x = *reinterpret_cast<const f16x8*>(static_cast<const f16*>(H.p) + n * H.ld + d + p * H.lo);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = (f16)ldexpf((float)x[k], e);
            *reinterpret_cast<f16x8*>(y + n * (long long)Dp + d + p * lo) = x;
        }
    }
}

// dl of classes [v0, v0 + cols) in 16 bits: [row][class - v0], pitch ld (cols rounded up to 8; zeros behind the last class).
// p - 1 and c - E are formed in fp32, and what is dropped is 2^-22 of dl in two planes of fp16, 2^-16 of bf16, or half a step of
// the gradients' own type where 16-bit inputs take one plane: Plan::dl_planes.
struct DlArgs {
    int v0, cols;
    const int* shifts;
    const int* tgt;
    const float* centers;
    const float* top;
    const float* inv_sum;
    const float* mean;
    Upstream up;
    void* dl;
    int ld;
    long long lo;
};
template <class T, class S, int SPLIT, int MODE>
__device__ __forceinline__ void dl_of_tile(f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int cnt, const HeadState* st,
                                           const BackState* bs, const DlArgs& a) {
    const int ws = SPLIT == 3 ? weight_shift(st) : 0;
    constexpr bool kScaled = !std::is_same<T, bf16>::value;
    const Centers all = MODE == kExpect && kScaled ? bs->centers : Centers{0, 0};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, c0 = m0 + wm * S::FM * 16 + (lane >> 4) * 4;
    T* dl = static_cast<T*>(a.dl);
    const bool edge = m0 + S::BM > a.cols;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
        if (n >= cnt) continue;
        const float tp = a.top[n], rs = a.inv_sum[n];
        const int shift = SPLIT == 3 ? -ws - a.shifts[n] : 0;
        float g = upstream(a.up, n, cnt);
        if (kScaled) g = ldexpf(g, kDlTop - exp_above(fabsf(g)));
        if (MODE == kCE) {
            const int t = a.tgt[n] - a.v0 - c0;
            if (a.tgt[n] < 0) g = __builtin_nanf("");
            const float gr = g * rs;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float l = SPLIT == 3 ? ldexpf(acc[i][j][e], shift) : acc[i][j][e];
                    const float x = exp_of(l - tp);
                    acc[i][j][e] = fmaf(x, gr, t == i * 16 + e ? -g : 0.f);
                }
        } else {
            const float cs = kScaled ? ldexpf(1.f, -center_exp(all, a.mean[n])) : 1.f;      // (a power of two: exact)
            const float e0 = a.mean[n] * cs, gr = g * rs;
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int c = c0 + i * 16 + e;
                    const float l = SPLIT == 3 ? ldexpf(acc[i][j][e], shift) : acc[i][j][e];
                    acc[i][j][e] = exp_of(l - tp) * gr * fmaf(edge && c >= a.cols ? 0.f : a.centers[a.v0 + c], cs, -e0);
                }
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < S::FM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c0 + i * 16 + e >= a.cols) acc[i][j][e] = 0.f;
        }
        if constexpr (S::FM == 1) {
            const float d[4] = {acc[0][j][0], acc[0][j][1], acc[0][j][2], acc[0][j][3]};
            if (!(edge && c0 >= a.ld)) put4<SPLIT == 1 ? 1 : 3>(dl + (long long)n * a.ld + c0, a.lo, d);
            continue;
        }
        const int c8 = m0 + wm * S::FM * 16 + (lane >> 4) * 8;
#pragma unroll
        for (int i = 0; i + 1 < S::FM; i += 2) {
            const int c = c8 + i * 16;
            s16x8 hi, lo;
            eight_of(round4<T>(acc[i][j]), round4<T>(acc[i + 1][j]), hi);
            if constexpr (SPLIT > 1) eight_of(rest4<T>(acc[i][j]), rest4<T>(acc[i + 1][j]), lo);
            if (edge && c >= a.ld) continue;
            T* q = dl + (long long)n * a.ld + c;
            *reinterpret_cast<s16x8*>(q) = hi;
            if constexpr (SPLIT > 1) *reinterpret_cast<s16x8*>(q + a.lo) = lo;
        }
    }
}
template <class T, class S, int SPLIT, int MODE>
__global__ __launch_bounds__(S::T) void head_dl_kernel(Operand W, Operand H, const HeadState* __restrict__ st,
                                                       const BackState* __restrict__ bs, int D, DlArgs a) {
    __shared__ __align__(16) char lds[lds_bytes<S, kP<SPLIT>, kP<SPLIT>>()];
    const int vt = cdiv(a.cols, S::BM);
    const int m0 = (int)(blockIdx.x % vt) * S::BM, n0 = (int)(blockIdx.x / vt) * S::BN;
    const int cnt = st->count;
    if (n0 >= cnt) return;
    H.outer = cnt;
    f32x4 acc[S::FM][S::FN];
    gemm_tile<T, S, kK, kK, kP<SPLIT>, kP<SPLIT>>(W, H, m0, n0, 0, D, lds, acc);
    dl_of_tile<T, S, SPLIT, MODE>(acc, m0, n0, cnt, st, bs, a);
}
template <class T, int SPLIT, int MODE>
__global__ __launch_bounds__(Big::T) void head_dl_big_kernel(Operand W, Operand H, const HeadState* __restrict__ st,
                                                             const BackState* __restrict__ bs, int D, DlArgs a) {
    __shared__ __align__(16) char lds[Big::kLds];
    const int cnt = st->count, mt = cdiv(a.cols, Big::BM), nt = cdiv(cnt, Big::BN), tiles = mt * nt;
    int t = blockIdx.x;
    if (t >= tiles) return;
    H.outer = cnt;
    const Order order(tiles, mt, nt);
    auto job = [&](int u) {
        int m, n;
        order(u, m, n);
        return Job{W, H, m * Big::BM, n * Big::BN, 0, D};
    };
    TileStream<T, kK, kK, kP<SPLIT>, kP<SPLIT>> stream(lds, job(t));
    for (; t < tiles; t += gridDim.x) {
        const int m0 = stream.job.m0, n0 = stream.job.n0;
        f32x4 acc[Big::FM][Big::FN];
        stream.multiply(acc, [&](Job& j) {
            const int u = t + gridDim.x;
            if (u < tiles) j = job(u);
            return u < tiles;
        });
        dl_of_tile<T, Big, SPLIT, MODE>(acc, m0, n0, cnt, st, bs, a);
    }
}

// dH = dl W: features along m (W as kM operand, classes are k), rows along n.  ACC: fp32 partials [split][row][Dp4], added to
// what earlier pieces of the classes left; otherwise straight into the caller's rows.
// dW of one piece = dl^T H: features along m, classes along n, k = rows (both kM operands).
struct GradArgs {
    int D, k, splits;            // k: classes of the piece (dH); cols: classes of the piece (dW, whose k is the row count)
    int cols, first;
    const int* rows;
    void* out;
    float* part;
    long long part_split;
    Upstream up;
    bool reach;                  // dW: rows weigh with their reach
};
// which: 0 = dH, 1 = dW.  Writes the tile of row / class n and features m.
template <class T, class S, int SPLIT, class O, bool ACC, int WHICH>
__device__ __forceinline__ void grad_of_tile(const f32x4 (&acc)[S::FM][S::FN], int m0, int n0, int sp, int bound,
                                             const HeadState* st, const BackState* bs, const GradArgs& a) {
    const int cnt = st->count;
    const int all = WHICH == 0 ? kDlExp<T> - (SPLIT == 3 ? weight_shift(st) : 0) : dw_exp<T, SPLIT>(st, bs, a.up, cnt, a.reach);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, Dp = (a.D + 3) & ~3;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
        const int n = n0 + (wn * S::FN + j) * 16 + (lane & 15);
        if (n >= bound) continue;
        const long long row = !ACC && WHICH == 0 && a.rows ? a.rows[n] : n;
        const int back = !ACC && WHICH == 0 ? all + row_exp<T>(a.up, bs, n, upstream(a.up, n, cnt)) : all;
        if (ACC) {
#pragma unroll
            for (int i = 0; i < S::FM; ++i) {
                const int d = m0 + (wm * S::FM + i) * 16 + (lane >> 4) * 4;
                if (d >= a.D) continue;
                f32x4* q = reinterpret_cast<f32x4*>(a.part + sp * a.part_split + row * Dp + d);
                f32x4 v = acc[i][j];
                if (WHICH == 0 && !a.first) v += *q;
                *q = v;
            }
        } else if (S::FM == 1) {
            const f32x4 v = scaled(acc[0][j], back);
            const float w[4] = {v[0], v[1], v[2], v[3]};
            put_row4(static_cast<O*>(a.out) + row * a.D, m0 + wm * 16 + (lane >> 4) * 4, a.D, w);
        } else {
#pragma unroll
            for (int i = 0; i + 1 < S::FM; i += 2)
                put_row8(static_cast<O*>(a.out) + row * a.D, m0 + (wm * S::FM + i) * 16, a.D, lane, scaled(acc[i][j], back),
                         scaled(acc[i + 1][j], back));
        }
    }
}
// A: W (dH) or H (dW), B: dl.  Workgroups: tiles x splits in Order.
template <class T, class S, int SPLIT, class O, bool ACC, int WHICH>
__global__ __launch_bounds__(S::T) void head_grad_kernel(Operand A, Operand B, const HeadState* __restrict__ st,
                                                         const BackState* __restrict__ bs, GradArgs a) {
    __shared__ __align__(16) char lds[std::is_same<S, Big>::value ? Big::kLds : lds_bytes<S, kP<SPLIT>, kPdl<SPLIT>>()];
    const int cnt = st->count, mt = cdiv(a.D, S::BM), bound = WHICH == 0 ? cnt : a.cols;
    const int k = WHICH == 0 ? a.k : cnt, per = cdiv(cdiv(k, kBK), a.splits) * kBK;
    B.outer = cnt;
    if (WHICH == 1) A.outer = cnt;
    constexpr Lay LB = WHICH == 0 ? kK : kM;
    const int nt = cdiv(bound, S::BN), units = mt * nt * a.splits;
    int t = blockIdx.x;
    if (t >= units) return;
    const Order order(units, mt * a.splits, nt);
    auto job = [&](int u, int& sp) {
        int x, n;
        order(u, x, n);
        sp = x / mt;
        const int k0 = split_start(sp, per, k);
        return Job{A, B, (x - sp * mt) * S::BM, n * S::BN, k0, min(k0 + per, k)};
    };
    int sp;
    if constexpr (std::is_same<S, Big>::value) {
        int next_sp = 0;
        TileStream<T, kM, LB, kP<SPLIT>, kPdl<SPLIT>> stream(lds, job(t, sp));
        for (; t < units; t += gridDim.x) {
            const int m0 = stream.job.m0, n0 = stream.job.n0;
            f32x4 acc[S::FM][S::FN];
            stream.multiply(acc, [&](Job& j) {
                const int u = t + gridDim.x;
                if (u < units) j = job(u, next_sp);
                return u < units;
            });
            grad_of_tile<T, S, SPLIT, O, ACC, WHICH>(acc, m0, n0, sp, bound, st, bs, a);
            sp = next_sp;
        }
    } else {
        const Job j = job(t, sp);
        f32x4 acc[S::FM][S::FN];
        gemm_tile<T, S, kM, LB, kP<SPLIT>, kPdl<SPLIT>>(A, B, j.m0, j.n0, j.kbeg, j.kend, lds, acc);
        grad_of_tile<T, S, SPLIT, O, ACC, WHICH>(acc, j.m0, j.n0, sp, bound, st, bs, a);
    }
}

// sums the splits of a product in order, scales, and writes rows of the caller.  which: 0 = dH, 1 = dW.  PAR lanes share the
// splits of an output (each a contiguous share, joined in order), for products of few outputs and many splits.
// (16 of them: 80 x 64 outputs of 100000 rows 66 us a step against 84, 256 x 128 of 20000 57 against 60, 600 x 256 199 against
// 198.)
constexpr long long kShareOuts = 1 << 17;
template <class T, int SPLIT, class O, int PAR>
__global__ __launch_bounds__(256) void head_sum_kernel(const float* __restrict__ part, long long part_split, int splits,
                                                       const HeadState* __restrict__ st, const BackState* __restrict__ bs, int n,
                                                       int D, int which, Upstream up, bool reach,
                                                       const int* __restrict__ rows, O* __restrict__ out) {
    constexpr int kOuts = 256 / PAR;
    __shared__ f32x4 red[PAR][kOuts + 1];
    const int cnt = which == 0 ? st->count : n, Dp = (D + 3) & ~3, q = Dp / 4;
    const int same = which == 0 ? kDlExp<T> - (SPLIT == 3 ? weight_shift(st) : 0) : dw_exp<T, SPLIT>(st, bs, up, st->count, reach);
    const long long all = (long long)cnt * q;
    const int x = threadIdx.x % kOuts, y = threadIdx.x / kOuts, per = (splits + PAR - 1) / PAR;
    for (long long i0 = (long long)blockIdx.x * kOuts; i0 < all; i0 += (long long)gridDim.x * kOuts) {
        const long long i = i0 + x;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
        if (i < all) {
            const float* p = part + i * 4;
            const int s1 = min(splits, (y + 1) * per);
#pragma unroll 4
            for (int s = y * per; s < s1; ++s) a += *reinterpret_cast<const f32x4*>(p + s * part_split);
        }
        if (PAR > 1) {
            red[y][x] = a;
            __syncthreads();
            a = f32x4{0.f, 0.f, 0.f, 0.f};
            if (y == 0)
                for (int s = 0; s < PAR; ++s) a += red[s][x];
            __syncthreads();
        }
        if (i < all && y == 0) {
            const long long r = i / q;
            const int d = (int)(i - r * q) * 4;
            a = scaled(a, which == 0 ? same + row_exp<T>(up, bs, (int)r, upstream(up, (int)r, cnt)) : same);
            const float v[4] = {a[0], a[1], a[2], a[3]};
            put_row4(out + (rows && which == 0 ? (long long)rows[r] : r) * D, d, D, v);
        }
    }
}

// Rows that were left out have no gradient.  Waves w, w + waves, .. of a launch.
struct Ignored {
    const long long* target;     // NULL: nothing to do
    int n, L, vec;
    long long ignore;
};
template <class O>
__device__ __forceinline__ void zero_ignored(const Ignored& g, int D, const HeadState* st, O* out, int w, int waves) {
    if (!g.target || st->count == g.n) return;
    constexpr int VEC = 16 / sizeof(O), U = 4;
    const int lane = threadIdx.x & 63, sub = lane & (g.L - 1), R = 64 / g.L, hop = waves * R;
    for (int r0 = w * R + lane / g.L; r0 < g.n; r0 += hop * U) {
        long long t[U];
#pragma unroll
        for (int u = 0; u < U; ++u) t[u] = g.target[min(r0 + u * hop, g.n - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r0 + u * hop < g.n && t[u] == g.ignore) {
                O* q = out + (long long)(r0 + u * hop) * D;
                if (g.vec) {
                    typename Vec<O, VEC>::type z;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z[e] = (O)0.f;
                    for (int d = sub * VEC; d < D; d += g.L * VEC) *reinterpret_cast<typename Vec<O, VEC>::type*>(q + d) = z;
                } else {
                    for (int d = sub; d < D; d += g.L) q[d] = (O)0.f;
                }
            }
    }
}
template <class O>
__global__ __launch_bounds__(256) void zero_ignored_kernel(Ignored g, int D, const HeadState* __restrict__ st,
                                                           O* __restrict__ out) {
    zero_ignored(g, D, st, out, blockIdx.x * 4 + (threadIdx.x >> 6), gridDim.x * 4);
}

// ------------------------------------------------------------------------------------------------------ small heads
//
// A head whose weight fits LDS (depth bins) is bound by the features' bytes, not by its products: a wave takes 16 rows, keeps
// their features in registers, meets all classes in LDS and has the whole softmax of its rows to itself -- no partial
// statistics, no barrier.  Backward the same: dl of 32 classes, as the matrix instruction leaves it, is the operand of
// dH = dl W as it stands (its lanes hold rows, its registers classes, taken as k in the order 4 q + e of two fragments; the
// transposing LDS reads of W follow that order), so dH needs no second pass; dl itself is written once for dW.  dH takes two
// planes of dl, straight from registers, whatever the inputs' type.
//   12 x 96 x 320 rows, 64 features, 80 bins, bf16, forward 18 us (47 MB of features; the tiles above: 48).  By its counters the
//   vector instructions are what it takes: 88 % of a busy CU's time, LDS 24 %, matrix instructions 12 %.
constexpr int kSlimT = 512;
struct SlimArgs {
    const void* h;             // features: the caller's rows, or staged ones
    long long ldh, lo_h;
    const int* gather;         // where the features of a kept row are (NULL: in order)
    const int* rows;           // the caller's row of a kept row (NULL: the same)
    HeadState* st;             // count of kept rows and scales; set_count: n rows, and st->count is written
    int set_count;
    int n, D, V, Vp;           // Vp: V rounded up to 32
    Operand W;
    const int* shifts;         // exponents of the rows' planes
    const int* tgt;
    const float* centers;
    float *top, *inv_sum, *mean;
};
struct SlimFwd {
    float* out;                // CE: per caller's row (NULL: only sums), expectation: per row
    double* sums;              // CE: a workgroup's sum of losses (NULL: none)
};
struct SlimBwd {
    const BackState* bs;
    Upstream up;
    void* g_hidden;            // NULL: not wanted
    void* dl;                  // NULL: dW not wanted
    int ld, planes;
    long long lo;
    Ignored ignored;           // the caller's rows that were left out (with g_hidden)
    void* packed;              // kept rows' features written densely for dW (NULL: they lie so already), pitch Dp
    int Dp;
};

// W to LDS: per plane, blocks of 64 columns, each [Vp][64] in lds_chunk's order
template <int P, int ND>
__device__ __forceinline__ void slim_load_w(const SlimArgs& a, char* lds) {
    constexpr int kChunks = ND * 4, U = 4;       // chunks of a row; loads under way at a time
    for (int i0 = threadIdx.x; i0 < a.Vp * kChunks; i0 += U * kSlimT) {
        i32x4 x[U][P];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kSlimT, v = i / kChunks, c = i % kChunks;
            const bool in = v < a.V && c * 8 < a.W.inner;
            const char* src = static_cast<const char*>(a.W.p) + 2 * ((long long)v * a.W.ld + c * 8);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                x[u][p] = i32x4{0, 0, 0, 0};
                if (in) x[u][p] = *reinterpret_cast<const i32x4*>(src + 2 * p * a.W.lo);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kSlimT, v = i / kChunks, c = i % kChunks;
            if (v >= a.Vp) break;
#pragma unroll
            for (int p = 0; p < P; ++p)
                *reinterpret_cast<i32x4*>(lds + p * a.Vp * ND * 64 + (c >> 3) * a.Vp * 128 + lds_chunk<kK, 16>(v, c & 7)) = x[u][p];
        }
    }
    if (a.centers) {      // behind the weight; zero where there is no class
        float* c = reinterpret_cast<float*>(lds + P * a.Vp * ND * 64);
        for (int v = threadIdx.x; v < a.Vp; v += kSlimT) c[v] = v < a.V ? a.centers[v] : 0.f;
    }
    __syncthreads();
}
template <int P, int ND>
struct SlimRows {
    s16x8 h[P][ND];
    __device__ __forceinline__ void load(const SlimArgs& a, int n, int cnt, int lane) {
        const int m = n < cnt ? n : cnt - 1;
        const long long row = a.gather ? a.gather[m] : m;
        const char* p = static_cast<const char*>(a.h) + 2 * (row * a.ldh + (lane >> 4) * 8);
#pragma unroll
        for (int k = 0; k < ND; ++k)
#pragma unroll
            for (int q = 0; q < P; ++q) {
                s16x8 x = {0, 0, 0, 0, 0, 0, 0, 0};
                if (k * 32 + (lane >> 4) * 8 < a.D) x = *reinterpret_cast<const s16x8*>(p + 2 * (k * 32 + q * a.lo_h));
                h[q][k] = x;
            }
    }
};
// logits of the 16 classes of fragment f for the wave's rows: lane holds row lane % 16, classes 16 f + 4 (lane / 16) + e
template <class T, int P, int ND>
__device__ __forceinline__ f32x4 slim_logits(const SlimRows<P, ND>& r, const char* lds, int base, int f, int Vp, int shift) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < ND; ++k) {
        const char* p = lds + (k >> 1) * Vp * 128 + f * 16 * 128 + (base ^ ((k & 1) << 6));
        const s16x8 w = *reinterpret_cast<const s16x8*>(p);
        if (P == 2) {
            const s16x8 wl = *reinterpret_cast<const s16x8*>(p + Vp * ND * 64);
            acc = mfma(wl, r.h[0][k], acc, T());
            acc = mfma(w, r.h[P - 1][k], acc, T());
        }
        acc = mfma(w, r.h[0][k], acc, T());
    }
    return P == 2 ? scaled(acc, shift) : acc;
}
__device__ __forceinline__ void join_softmax(float& mx, float& s, float& sc, float m2, float s2, float c2) {
    const float nm = fmaxf(mx, m2), ref = nm == -INFINITY ? 0.f : nm;
    const float f1 = exp_of(mx - ref), f2 = exp_of(m2 - ref);
    s = s * f1 + s2 * f2;
    sc = sc * f1 + c2 * f2;
    mx = nm;
}

template <class T, int P, int ND, int MODE>
__global__ __launch_bounds__(kSlimT) void slim_fwd_kernel(SlimArgs a, SlimFwd o) {
    extern __shared__ __align__(16) char lds[];
    __shared__ double wsum[kSlimT / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cnt = a.set_count ? a.n : a.st->count, blocks = (cnt + 15) / 16, step = gridDim.x * (kSlimT / 64);
    int b = blockIdx.x * (kSlimT / 64) + wave;
    if (a.set_count && blockIdx.x == 0 && threadIdx.x == 0) a.st->count = a.n;
    SlimRows<P, ND> next;
    if (b < blocks) next.load(a, b * 16 + (lane & 15), cnt, lane);
    slim_load_w<P, ND>(a, lds);
    const int ws = P == 2 ? weight_shift(a.st) : 0;
    const int base = lds_chunk<kK, 16>(lane & 15, lane >> 4), frags = a.Vp / 16, q4 = (lane >> 4) * 4;
    const float* centers = reinterpret_cast<const float*>(lds + P * a.Vp * ND * 64);
    double total = 0.0;
    for (; b < blocks; b += step) {
        const SlimRows<P, ND> r = next;
        const int n = b * 16 + (lane & 15);
        if (b + step < blocks) next.load(a, (b + step) * 16 + (lane & 15), cnt, lane);
        const int target = MODE == kCE ? a.tgt[n < cnt ? n : cnt - 1] : -1, t = target - q4;      // t: from the lane's first class
        const int shift = P == 2 ? -ws - a.shifts[n < cnt ? n : cnt - 1] : 0;
        float mx = -INFINITY, s = 0.f, sc = 0.f, tl = 0.f;
        for (int f = 0; f < frags; f += 2) {
            f32x4 l[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) l[u] = slim_logits<T, P, ND>(r, lds, base, f + u, a.Vp, shift);
            if (f * 16 + 32 > a.V) {       // classes that do not exist
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((f + u) * 16 + q4 + e >= a.V) l[u][e] = -INFINITY;
            }
            float m = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (MODE == kCE && (f + u) * 16 + e == t) tl = l[u][e];
                    m = fmaxf(m, l[u][e]);      // passes over NaN, which reaches the sum
                }
            // the running maximum moves only where it must: its factor is exp(0) = 1 otherwise
            const float nm = fmaxf(mx, m), ref = nm == -INFINITY ? 0.f : nm, f1 = exp_of(mx - ref);
            s *= f1;
            sc *= f1;
            mx = nm;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                f32x4 c = {0.f, 0.f, 0.f, 0.f};
                if (MODE == kExpect) c = *reinterpret_cast<const f32x4*>(centers + (f + u) * 16 + q4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = exp_of(l[u][e] - ref);
                    s += x;
                    if (MODE == kExpect) sc = fmaf(x, c[e], sc);
                }
            }
        }
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) {
            join_softmax(mx, s, sc, __shfl_xor(mx, d, 64), __shfl_xor(s, d, 64), __shfl_xor(sc, d, 64));
            if (MODE == kCE) tl += __shfl_xor(tl, d, 64);     // three of the four are zero
        }
        if (lane < 16 && n < cnt) {
            const float ref = mx == -INFINITY ? 0.f : mx;
            a.top[n] = ref;
            a.inv_sum[n] = 1.f / s;
            if (MODE == kExpect) {
                o.out[n] = a.mean[n] = sc / s;
            } else {
                const float each = target < 0 ? __builtin_nanf("") : (ref - tl) + logf(s);
                if (o.out) o.out[a.rows ? a.rows[n] : n] = each;
                total += each;
            }
        }
    }
    if (MODE == kCE && o.sums) {
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) total += __shfl_xor(total, d, 64);
        if (lane == 0) wsum[wave] = total;
        __syncthreads();
        if (threadIdx.x == 0) {
            double x = 0.0;
            for (int i = 0; i < kSlimT / 64; ++i) x += wsum[i];
            o.sums[blockIdx.x] = x;
        }
    }
}

template <class T, int P, int ND, int MODE, class O>
__global__ __launch_bounds__(kSlimT) void slim_bwd_kernel(SlimArgs a, SlimBwd o) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cnt = a.st->count, blocks = (cnt + 15) / 16, step = gridDim.x * (kSlimT / 64);
    int b = blockIdx.x * (kSlimT / 64) + wave;
    SlimRows<P, ND> next;
    if (b < blocks) next.load(a, b * 16 + (lane & 15), cnt, lane);
    slim_load_w<P, ND>(a, lds);
    const int ws = P == 2 ? weight_shift(a.st) : 0, same = kDlExp<T> - ws;
    const int most = most_of<T, P == 2 ? 3 : 1>(a.st, o.bs, o.up, cnt);
    constexpr bool kScaled = !std::is_same<T, bf16>::value;
    const Centers all = MODE == kExpect && kScaled ? o.bs->centers : Centers{0, 0};
    const int base = lds_chunk<kK, 16>(lane & 15, lane >> 4), frags = a.Vp / 16, q4 = (lane >> 4) * 4;
    const float* centers = reinterpret_cast<const float*>(lds + P * a.Vp * ND * 64);
    // transposing reads: lane i of a 16-lane group q starts at class 4 q + i / 4, feature 4 (i % 4)
    const int tr = (lane >> 4) * 4 + ((lane >> 2) & 3);
    const int tbase = lds_chunk<kK, 16>(tr, (lane >> 1) & 1) + (lane & 1) * 8;
    typedef __attribute__((address_space(3))) s16x4* lp;
    T* dl = static_cast<T*>(o.dl);
    for (; b < blocks; b += step) {
        const SlimRows<P, ND> r = next;
        const int n = b * 16 + (lane & 15), m = n < cnt ? n : cnt - 1;
        if (b + step < blocks) next.load(a, (b + step) * 16 + (lane & 15), cnt, lane);
        const float tp = a.top[m], rs = a.inv_sum[m], mean = MODE == kExpect ? a.mean[m] : 0.f;
        const int ce = MODE == kExpect && kScaled ? center_exp(all, mean) : 0;
        const float cs = ldexpf(1.f, -ce), e0 = mean * cs;
        const int target = MODE == kCE ? a.tgt[m] : -1, t = target - q4;
        float g = upstream(o.up, m, cnt);
        const int own = P == 2 ? a.shifts[m] : 0, shift = -ws - own;
        const int ge = kScaled ? exp_above(fabsf(g)) : 0, re = ge + ce;
        const int we = kScaled ? weight_exp(g, re, P == 2 ? kReachTop - own : 0, most) : 0;
        if (kScaled) g = ldexpf(g, kDlTop - ge);
        if (MODE == kCE && target < 0) g = __builtin_nanf("");
        const float gr = g * rs;
        f32x4 acc[2 * ND];
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int f = 0; f < frags; f += 2) {
            f32x4 d[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const f32x4 l = slim_logits<T, P, ND>(r, lds, base, f + u, a.Vp, shift);
                const int v = (f + u) * 16 + q4;
                f32x4 c = {0.f, 0.f, 0.f, 0.f};
                if (MODE == kExpect) c = *reinterpret_cast<const f32x4*>(centers + v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = exp_of(l[e] - tp);
                    if (MODE == kExpect)
                        d[u][e] = x * gr * fmaf(c[e], cs, -e0);
                    else
                        d[u][e] = fmaf(x, gr, (f + u) * 16 + e == t ? -g : 0.f);
                }
                if (f * 16 + 32 > a.V) {      // classes that do not exist
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (v + e >= a.V) d[u][e] = 0.f;
                }
                if (dl && n < cnt && v < o.ld) {
                    const f32x4 w = std::is_same<T, bf16>::value ? d[u] : scaled(d[u], we);      // weighted for dW
                    const float y[4] = {w[0], w[1], w[2], w[3]};
                    if (P == 2 || o.planes == 2)
                        put4<3>(dl + (long long)n * o.ld + v, o.lo, y);
                    else
                        put4<1>(dl + (long long)n * o.ld + v, o.lo, y);
                }
            }
            if (o.g_hidden) {
                typedef T t8 __attribute__((ext_vector_type(8)));
                t8 hi, lw;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    T p, q;
                    split16(d[e >> 2][e & 3], p, q);
                    hi[e] = p;
                    lw[e] = q;
                }
                const s16x8 bh = __builtin_bit_cast(s16x8, hi);
#pragma unroll
                for (int i = 0; i < 2 * ND; ++i) {
                    const char* p = lds + (i >> 2) * a.Vp * 128 + f * 16 * 128 + (tbase ^ ((i & 3) << 5));
                    auto get = [&](const char* q) {
                        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q));
                        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 16 * 128));
                        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                    };
                    const s16x8 w = get(p);
                    if constexpr (P == 2) acc[i] = mfma(get(p + a.Vp * ND * 64), bh, acc[i], T());
                    acc[i] = mfma(w, __builtin_bit_cast(s16x8, lw), acc[i], T());
                    acc[i] = mfma(w, bh, acc[i], T());
                }
            }
        }
        if (n < cnt) {
            if (o.g_hidden) {
                O* row = static_cast<O*>(o.g_hidden) + (long long)(a.rows ? a.rows[n] : n) * a.D;
#pragma unroll
                for (int i = 0; i < 2 * ND; ++i) {
                    const int c = i * 16 + (lane >> 4) * 4;
                    const f32x4 x = scaled(acc[i], same + re);
                    const float y[4] = {x[0], x[1], x[2], x[3]};
                    if (c < a.D) put_row4(row, c, a.D, y);
                }
            }
            if (o.packed) {
#pragma unroll
                for (int k = 0; k < ND; ++k) {
                    const int c = k * 32 + (lane >> 4) * 8;
                    if (c < o.Dp) *reinterpret_cast<s16x8*>(static_cast<T*>(o.packed) + (long long)n * o.Dp + c) = r.h[0][k];
                }
            }
        }
    }
    if (o.g_hidden)
        zero_ignored(o.ignored, a.D, a.st, static_cast<O*>(o.g_hidden), blockIdx.x * (kSlimT / 64) + wave, gridDim.x * (kSlimT / 64));
}

// ----------------------------------------------------------------------------------------------------------- few rows
//
// Up to four rows (a single position answered) read the weight once and are bound by that: every class row goes straight from
// memory to registers, as it is (fp32 too: no planes), and meets the rows' features out of LDS in fp32.  L lanes share a
// class, four classes a group are under way at a time.
constexpr int kFewT = 512, kFewMax = 4;
struct FewArgs {
    const int* rows;
    HeadState* st;
    int set_count, n, D, V, L;
    const int* tgt;
    const float* centers;
    float* part;               // [workgroup][row][4]: maximum, sum, sum of centres, logit of the target
};
template <class IT, int VEC, int NR>
__global__ __launch_bounds__(kFewT) void few_kernel(const IT* __restrict__ h, long long ldh, const IT* __restrict__ w, FewArgs a) {
    extern __shared__ __align__(16) char lds_[];
    float* hs = reinterpret_cast<float*>(lds_);            // [NR][Dq]
    __shared__ float red[kFewT / 64][NR][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, Dq = (a.D + 7) & ~7;
    if (a.set_count && blockIdx.x == 0 && threadIdx.x == 0) {
        a.st->count = a.n;
        a.st->amax_w = 0;
    }
    const int cnt = a.set_count ? a.n : a.st->count;
    for (int r = 0; r < NR; ++r)
        for (int d = threadIdx.x; d < Dq; d += kFewT)
            hs[r * Dq + d] = r < cnt && d < a.D ? (float)h[(a.rows ? a.rows[r] : r) * ldh + d] : 0.f;
    __syncthreads();
    const int L = a.L, sub = lane & (L - 1), G = 64 / L;
    const int groups = gridDim.x * (kFewT / 64) * G, g = (blockIdx.x * (kFewT / 64) + wave) * G + lane / L;
    constexpr int U = 4;
    float mx[NR], s[NR], sc[NR], tl[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        mx[r] = -INFINITY;
        s[r] = sc[r] = tl[r] = 0.f;
    }
    for (int v0 = g; v0 < a.V; v0 += groups * U) {
        float acc[U][NR];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[u][r] = 0.f;
        for (int d = sub * VEC; d < a.D; d += L * VEC) {
            IT x[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = min(v0 + u * groups, a.V - 1);
                load_vec<IT, VEC>(w + (long long)v * a.D, d, a.D, x[u]);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float y = hs[r * Dq + d + e];
#pragma unroll
                    for (int u = 0; u < U; ++u) acc[u][r] = fmaf((float)x[u][e], y, acc[u][r]);
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = v0 + u * groups;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                float l = acc[u][r];
                for (int o = 1; o < L; o <<= 1) l += __shfl_xor(l, o, 64);
                if (v < a.V) {
                    if (a.tgt && v == a.tgt[r < cnt ? r : 0]) tl[r] = l;
                    join_softmax(mx[r], s[r], sc[r], l, 1.f, a.centers ? a.centers[v] : 0.f);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        for (int o = L; o < 64; o <<= 1) {
            join_softmax(mx[r], s[r], sc[r], __shfl_xor(mx[r], o, 64), __shfl_xor(s[r], o, 64), __shfl_xor(sc[r], o, 64));
            tl[r] += __shfl_xor(tl[r], o, 64);          // one group met the target
        }
        if (lane == 0) {
            red[wave][r][0] = mx[r];
            red[wave][r][1] = s[r];
            red[wave][r][2] = sc[r];
            red[wave][r][3] = tl[r];
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < NR) {
        const int r = threadIdx.x;
        float m = -INFINITY, t = 0.f, c = 0.f, l = 0.f;
        for (int i = 0; i < kFewT / 64; ++i) {
            join_softmax(m, t, c, red[i][r][0], red[i][r][1], red[i][r][2]);
            l += red[i][r][3];
        }
        float* q = a.part + ((long long)blockIdx.x * NR + r) * 4;
        q[0] = m;
        q[1] = t;
        q[2] = c;
        q[3] = l;
    }
}
// joins the workgroups of few_kernel (or the class tiles of the thin shape): one workgroup, a wave per row at a time
struct JoinArgs {
    const float *mx, *s, *sc, *tl;      // entry i of row r at [i * step + r * pitch]; tl: per row where tl_step is 0
    long long step, pitch, tl_step;
    int entries, mode;
    const HeadState* st;
    const int* rows;
    const int* tgt;
    float *top, *inv_sum, *mean, *out;
    int total;                          // CE: 0 each row, 1 sum, 2 mean
};
__global__ __launch_bounds__(1024) void join_few_kernel(JoinArgs a) {
    __shared__ float each[32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cnt = a.st->count;
    for (int r = wave; r < cnt; r += 16) {
        float mx = -INFINITY, s = 0.f, sc = 0.f, tl = 0.f;
        for (int i = lane; i < a.entries; i += 64) {
            const long long at = i * a.step + r * a.pitch;
            join_softmax(mx, s, sc, a.mx[at], a.s[at], a.mode == kExpect ? a.sc[at] : 0.f);
            if (a.mode == kCE && a.tl_step) tl += a.tl[at];
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            join_softmax(mx, s, sc, __shfl_xor(mx, o, 64), __shfl_xor(s, o, 64), __shfl_xor(sc, o, 64));
            tl += __shfl_xor(tl, o, 64);
        }
        if (lane == 0) {
            const float ref = mx == -INFINITY ? 0.f : mx;
            a.top[r] = ref;
            a.inv_sum[r] = 1.f / s;
            if (a.mode == kExpect) {
                a.out[r] = a.mean[r] = sc / s;
            } else {
                if (!a.tl_step) tl = a.tl[r];
                each[r] = a.tgt[r] < 0 ? __builtin_nanf("") : (ref - tl) + logf(s);
                if (!a.total) a.out[a.rows[r]] = each[r];
            }
        }
    }
    if (a.mode == kExpect || !a.total) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int r = 0; r < cnt; ++r) t += each[r];
        a.out[0] = (float)(a.total == DS_REDUCE_MEAN ? t / cnt : t);
    }
}

// ------------------------------------------------------------------------------------------------------------- host
// Shapes: 256x256 outputs a workgroup (TileStream) for large products; 128x128, 64x64 and 32x32 below that.  Up to 32 rows of many
// classes have a shape of their own: long tiles read the weight in long runs (training steps of 16 rows, 65536 classes of 1024
// features, bf16, 137 us against 152 in the others; of 32 rows, 65536 of 256, float32, 141 / 183, 16000 of 64, bf16, 43 / 50, but
// 4000 of 256 43 / 40 and 1000 of 256, float32, 54 / 47).
typedef Shape<128, 32, 4, 1> Thin;    // 32 along n
Cut cut_of(long long M, long long N, long long K, int pairs, bool grad) {      // grad: operands kM, sums may be split
    return ds::cut_of([&](long long b) { return ((M + b - 1) / b) * ((N + b - 1) / b); }, (double)M * N, K, pairs, grad, grad,
                      cu_count());
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

struct Saved {
    HeadState* st;
    float* top;        // a kept row's largest logit and 1 / sum exp(l - top): more exact than their join lse, whose last
    float* inv_sum;    // bit is worth |lse| 2^-24 in every probability of the row
    float* mean;
    int* rows;
    int* tgt;
    int* shifts;       // exponents of staged rows (fp32, fp16)
};
size_t saved_bytes(long long N) { return align256(sizeof(HeadState)) + 6 * align256((size_t)N * 4); }
Saved saved_of(void* p, long long N) {
    char* c = static_cast<char*>(p);
    Saved s;
    s.st = reinterpret_cast<HeadState*>(c);
    c += align256(sizeof(HeadState));
    const size_t a = align256((size_t)N * 4);
    s.top = reinterpret_cast<float*>(c);
    s.inv_sum = reinterpret_cast<float*>(c + a);
    s.mean = reinterpret_cast<float*>(c + 2 * a);
    s.rows = reinterpret_cast<int*>(c + 3 * a);
    s.tgt = reinterpret_cast<int*>(c + 4 * a);
    s.shifts = reinterpret_cast<int*>(c + 5 * a);
    return s;
}

struct Plan {
    int planes, dl_planes, Dp, vt_fwd, piece, piece_ld, dh_splits, dw_splits;
    bool stage_w, stage_h, dh_part;
    ShapeId fwd, dl_shape, dh, dw;
    int few, few_grid;                 // forward of few rows: rows a workgroup holds (0: not that path)
    int slim, slim_bytes, slim_grid;   // small head: k steps of 32 a row (0: not that path); backward: slim_back
    bool slim_back, pack;
    size_t sh, sw, saved_total;                                            // staged operands behind Saved (not of few rows)
    size_t counts, tlogit, part, sums, alone, fwd_total;                   // offsets of the forward's workspace
    size_t bh, bs, hw, dl, dhp, dwp, bwd_total;                            // offsets of the backward's
};

int splits_for(long long tiles, long long steps) {
    // enough workgroups for two a CU, no split shorter than four steps of 64
    const long long want = cdiv(2ll * cu_count(), tiles > 0 ? tiles : 1), most = steps / 4;
    long long s = want < most ? want : most;
    return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}

// alone: a forward that no backward follows
Plan plan_of(int mode, int dtype, long long N, int D, int V, long long ldh, bool alone = false) {
    Plan p;
    p.planes = dtype == DS_F32 ? 2 : 1;
    p.Dp = pad8(D);
    p.stage_w = dtype == DS_F32 || D % 8 != 0;
    const size_t el = 2 * p.planes;
    const bool thin = N <= 32 && V >= 16000;
    // Few rows of a weight that would have to be packed first (20000 classes of 256 features, float32, 1 / 2 / 4 rows: 18 / 22 / 31
    // us here, 40 packed and multiplied; a 16-bit weight is read as it is by the matrix instructions as well: 65536 of 1024, bf16,
    // 39 / 49 / 70 us here, 36 there).  Not where a backward follows: it needs the packed weight, and logits with the forward's
    // bits, which these are not (the training step 92 us here with its statistics formed again, 77 all packed).  Their features
    // have to fit LDS in fp32 beside three more workgroups.
    p.few = !alone || N > kFewMax || !p.stage_w ? 0 : N <= 1 ? 1 : N <= 2 ? 2 : 4;
    if (p.few && (size_t)p.few * pad8(D) * 4 > 40 * 1024) p.few = 0;
    const int vec = dtype == DS_F32 ? 4 : 8, lanes = lanes_for(cdiv(D, vec));
    p.few_grid = cdiv(V, kFewT / lanes * 4) < 2 * cu_count() ? cdiv(V, kFewT / lanes * 4) : 2 * cu_count();
    // small head: the weight in LDS, two workgroups a CU (training steps of 100000 rows, here / in tiles: 80 classes of 64
    // features, bf16, 65 / 101 us; 576 of 64 141 / 188; 256 of 128 120 / 135; 128 of 250 144 / 141, forward 48 / 52; 288 of 64,
    // float32, 150 / 219).  Every workgroup brings the whole weight, which does not pay for a few rows of a large one (576 of 64,
    // bf16: 300 rows 49 / 39, 3000 57 / 51, 8000 67 / 68, 20000 72 / 85; 288 of 64, float32: 1000 51 / 47, 8000 64 / 74; but 80 of 64,
    // bf16: 300 30 / 35)
    const int Vp = (V + 31) & ~31;
    p.slim = D <= 64 ? 2 : D <= 128 ? 4 : D <= 256 ? 8 : 0;
    const long long bytes = (long long)Vp * p.slim * 64 * p.planes;
    if (bytes + Vp * 4 > 78 * 1024 || (bytes > 40 * 1024 && N < 6144)) p.slim = 0;
    p.slim_bytes = (int)bytes + Vp * 4;
    p.slim_grid = cdiv(N, 16 * (kSlimT / 64)) < 2 * cu_count() ? cdiv(N, 16 * (kSlimT / 64)) : 2 * cu_count();
    p.slim_back = p.slim && (long long)N * pad8(V) * (long long)el <= (1ll << 30);
    // 16-bit inputs: one plane of dl makes the gradients' error against 64 bits 1.2 .. 1.5 times that of rounding them, and up to 2.2
    // times for a few rows or classes (a row of 56, 3784 classes, bf16, 1.8; 483 rows of 56, 19229 classes, fp16, a twentieth kept,
    // 1.5); two planes make it 1.0.  They are taken where the products are not the bound: up to 2^31 products of numbers (a second
    // plane of 8192 x 65536 x 1024 would take six products for four, 5.8 ms for 4.0).  On chip dl is stored for dW alone, whose sums
    // over 64 rows a class and more average its rounding out (1.0 .. 1.15; 368640 x 64, 512 classes, bf16 403 us, 626 with two).
    p.dl_planes = p.planes == 2 ? 2 : (p.slim_back ? N < 64ll * V : (double)N * V * D <= 2147483648.0) ? 2 : 1;
    const size_t el_dl = 2 * p.dl_planes;
    // rows of the caller's can be read as they are (a tile's byte offsets have 31 bits: 256 rows)
    const bool whole = D % 8 == 0 && ldh % 8 == 0 && dtype != DS_F32 && ldh <= (1 << 21);
    p.stage_h = !whole || (mode == kCE && !p.slim_back);
    p.pack = whole && mode == kCE && p.slim_back;
    const size_t h = align256((size_t)N * p.Dp * el), w = p.stage_w ? align256((size_t)V * p.Dp * el) : 0;
    // what the forward stages is kept for the backward (staging 50021 classes of 771 features once more: 35 of 490 us)
    const int pairs = p.planes == 2 ? 3 : 1;
    p.fwd = thin ? kThin : cut_of(V, N, D, pairs, false).shape;
    p.vt_fwd = cdiv(V, side_of(p.fwd));
    size_t o = saved_bytes(N);
    p.sh = o; o += p.stage_h && !p.few ? h : 0;
    p.sw = o; o += p.few ? 0 : w;
    p.saved_total = o;
    o = 0;
    p.counts = o; o += align256((size_t)cdiv(N, kListBlock) * 4);
    p.tlogit = o; o += align256((size_t)N * 4);
    p.part = o; o += p.few ? align256((size_t)p.few_grid * p.few * 16) : p.slim ? 0 : 3 * align256((size_t)p.vt_fwd * N * 4);
    p.sums = o; o += align256((size_t)(cdiv(N, 32) > p.slim_grid ? cdiv(N, 32) : p.slim_grid) * 8);
    p.alone = o; o += alone ? p.saved_total : 0;        // what would be saved
    p.fwd_total = o;
    // a piece of the classes: about 256 MB of dl (64 MB: 16 % slower at 8192 x 65536 x 1024, 128 MB: 4 %, 512 MB: the same), at
    // least 1024 classes; pieces of one size, up to half larger where that saves one (6872 x 19619 x 496, bf16, in pieces of
    // 19456 and 163 classes 959 us, in two of 9856 761, in one 749)
    const long long room = (256ll << 20) / ((long long)el_dl * N), fit = room < 1024 ? 1024 : room;
    const long long pieces = p.slim_back || V <= fit ? 1 : (V + fit / 2) / fit;
    p.piece = pieces == 1 ? V : (cdiv((long long)V, pieces) + 63) / 64 * 64;
    p.piece_ld = pad8(p.piece);
    p.dl_shape = thin ? kThin : cut_of(p.piece, N, D, pairs, false).shape;
    // The backward's logits must have the forward's bits: probabilities are exp(l - top), and where logits are large their
    // rounding is too.  All shapes add up in the same order, but the large one takes planes pair by pair.
    if (p.planes == 2 && (p.slim || (p.fwd == kBig) != (p.dl_shape == kBig)))
        p.dl_shape = !p.slim ? p.fwd : p.dl_shape == kBig ? kSq : p.dl_shape;
    const int gp = p.planes + p.dl_planes - 1;
    const Cut dh = cut_of(D, N, p.piece, gp, true), dw = cut_of(D, p.piece, N, gp, true);
    p.dh = thin ? kThin : dh.shape;
    p.dh_splits = thin ? splits_for(cdiv(D, 128), cdiv(p.piece, kBK)) : dh.splits;
    p.dw = dw.shape;
    p.dw_splits = dw.splits;
    p.dh_part = p.dh_splits > 1 || p.piece < V;
    const size_t D4 = (D + 3) & ~3;
    o = 0;
    p.bh = o; o += p.pack ? h : 0;
    p.bs = o; o += 256;
    p.hw = o; o += dtype == DS_BF16 || p.slim_back ? 0 : h;      // weighted rows for dW
    p.dl = o; o += align256((size_t)N * p.piece_ld * el_dl);
    p.dhp = o; o += p.dh_part ? align256((size_t)p.dh_splits * N * D4 * 4) : 0;
    p.dwp = o; o += p.dw_splits > 1 ? align256((size_t)p.dw_splits * p.piece * D4 * 4) : 0;
    p.bwd_total = o;
    return p;
}

int check_sizes(int dtype, long long N, int D, int V, long long ldh) {
    if (N <= 0 || D <= 0 || V <= 0 || ldh < D) return DS_ERR_INVALID_ARG;
    if (dtype != DS_F32 && dtype != DS_F16 && dtype != DS_BF16) return DS_ERR_UNSUPPORTED;
    if ((long long)cdiv(V, 128) * cdiv(N, 32) > (1ll << 30)) return DS_ERR_UNSUPPORTED;   // workgroups of one launch
    if (N > DS_HEAD_MAX_ROWS || D > DS_HEAD_MAX_FEATURES || V > DS_HEAD_MAX_CLASSES) return DS_ERR_UNSUPPORTED;
    return DS_OK;
}

int launched() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? DS_OK : (int)e;
}

// the scale of an fp32 weight; `clear`: *st is not set yet, all N rows
template <class IT>
void scale_weight(const IT* weight, long long N, int D, int V, HeadState* st, bool clear, hipStream_t q) {
    constexpr int VEC = 16 / sizeof(IT);
    const int L = lanes_for(cdiv(D, VEC)), per = 4 * 64 / L * 4, b = cdiv(V, per);
    const int blocks = b <= 4 ? 1 : b < 512 ? b : 512;       // four passes of loads take less than a launch
    if (clear && blocks > 1) head_init_kernel<<<1, 1, 0, q>>>(st, (int)N);
    amax_kernel<IT, VEC><<<blocks, 256, 0, q>>>(weight, st, V, D, L, clear ? (int)N : 0);
}
// inputs as matrix operands: in place, or staged at wh and ww (stage: now; clear: *s.st is not set yet)
template <class IT, class T, int SPLIT>
void operands(const Plan& p, int mode, const IT* hidden, long long ldh, const IT* weight, long long N, int D, int V, const Saved& s,
              const int* rows, bool stage, bool clear, char* wh, char* ww, Operand& H, Operand& W, hipStream_t q) {
    if constexpr (SPLIT == 3)
        if (stage) scale_weight(weight, N, D, V, s.st, clear, q);
    H = Operand{hidden, ldh, 0, (int)N, D};
    W = Operand{weight, D, 0, V, D};
    constexpr int VEC = 16 / sizeof(IT);
    const int L = lanes_for(cdiv(p.Dp, VEC));
    auto blocks = [&](long long n) {
        const int b = cdiv(n, 4 * 64 / L * 2);
        return b < 4096 ? b : 4096;
    };
    Source a{}, b{};
    if (p.stage_h) {
        const long long lo = N * p.Dp;
        a = Source{hidden, ldh, rows, &s.st->count, (int)N, nullptr, s.shifts, mode == kCE ? s.st : nullptr, wh, lo, 0, blocks(N)};
        H = Operand{wh, p.Dp, lo, (int)N, p.Dp};
    }
    if (p.stage_w) {
        const long long lo = (long long)V * p.Dp;
        b = Source{weight, D, nullptr, nullptr, V, &s.st->amax_w, nullptr, nullptr, ww, lo, a.blocks, blocks(V)};
        W = Operand{ww, p.Dp, lo, V, p.Dp};
    }
    if (stage && a.blocks + b.blocks > 0)
        stage_kernel<IT, T, SPLIT, VEC><<<a.blocks + b.blocks, 256, 0, q>>>(a.blocks ? a : b, a.blocks ? b : Source{}, D, p.Dp, L);
}

template <class K>
int with_lds(K kernel, int bytes) {    // what a kernel may use beyond 64 KB it has to ask for
    return bytes <= 64 * 1024 ? 0
                              : (int)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
SlimArgs slim_args(const Plan& p, const Operand& H, const Operand& W, const Saved& s, const int* rows, long long N, int D, int V,
                   const float* centers) {
    return SlimArgs{H.p, H.ld, H.lo, p.stage_h ? nullptr : rows, rows, s.st, 0, (int)N, D, V, (V + 31) & ~31, W,
                    s.shifts, s.tgt, centers, s.top, s.inv_sum, s.mean};
}
template <class T, int P, int ND, int MODE>
int slim_fwd_launch(const Plan& p, const SlimArgs& a, const SlimFwd& o, hipStream_t q) {
    const int rc = with_lds(&slim_fwd_kernel<T, P, ND, MODE>, p.slim_bytes);
    if (rc) return rc;
    slim_fwd_kernel<T, P, ND, MODE><<<p.slim_grid, kSlimT, p.slim_bytes, q>>>(a, o);
    return 0;
}
template <class T, int P, int ND, int MODE, class O>
int slim_bwd_launch(const Plan& p, const SlimArgs& a, const SlimBwd& o, hipStream_t q) {
    const int rc = with_lds(&slim_bwd_kernel<T, P, ND, MODE, O>, p.slim_bytes);
    if (rc) return rc;
    slim_bwd_kernel<T, P, ND, MODE, O><<<p.slim_grid, kSlimT, p.slim_bytes, q>>>(a, o);
    return 0;
}
template <class T, int P, int MODE>
int slim_fwd(const Plan& p, const SlimArgs& a, const SlimFwd& o, hipStream_t q) {
    return p.slim == 2   ? slim_fwd_launch<T, P, 2, MODE>(p, a, o, q)
           : p.slim == 4 ? slim_fwd_launch<T, P, 4, MODE>(p, a, o, q)
                         : slim_fwd_launch<T, P, 8, MODE>(p, a, o, q);
}
template <class T, int P, int MODE, class O>
int slim_bwd(const Plan& p, const SlimArgs& a, const SlimBwd& o, hipStream_t q) {
    return p.slim == 2   ? slim_bwd_launch<T, P, 2, MODE, O>(p, a, o, q)
           : p.slim == 4 ? slim_bwd_launch<T, P, 4, MODE, O>(p, a, o, q)
                         : slim_bwd_launch<T, P, 8, MODE, O>(p, a, o, q);
}

template <class IT, int NR>
void few_launch(const Plan& p, const IT* h, long long ldh, const IT* w, FewArgs a, hipStream_t q) {
    constexpr int VEC = 16 / sizeof(IT);
    a.L = lanes_for(cdiv(a.D, VEC));
    few_kernel<IT, VEC, NR><<<p.few_grid, kFewT, NR * pad8(a.D) * 4, q>>>(h, ldh, w, a);
}

template <class T, int SPLIT, int MODE>
void stats_launch(const Plan& p, const Operand& W, const Operand& H, const Saved& s, long long N, int D, const StatsArgs& a,
                  hipStream_t q) {
    const int tiles = p.vt_fwd * cdiv(N, p.fwd == kThin ? Thin::BN : side_of(p.fwd));
    if (p.fwd == kThin)
        head_stats_kernel<T, Thin, SPLIT, MODE><<<tiles, Thin::T, 0, q>>>(W, H, s.st, D, a);
    else if (p.fwd == kBig)
        head_stats_big_kernel<T, SPLIT, MODE><<<tiles < cu_count() ? tiles : cu_count(), Big::T, 0, q>>>(W, H, s.st, D, a);
    else if (p.fwd == kSmall)
        head_stats_kernel<T, Small, SPLIT, MODE><<<tiles, Small::T, 0, q>>>(W, H, s.st, D, a);
    else if (p.fwd == kTiny)
        head_stats_kernel<T, Tiny, SPLIT, MODE><<<tiles, Tiny::T, 0, q>>>(W, H, s.st, D, a);
    else
        head_stats_kernel<T, Sq, SPLIT, MODE><<<tiles, Sq::T, 0, q>>>(W, H, s.st, D, a);
}

// of stats_launch, up to 32 rows
JoinArgs join_tiles(const Plan& p, int mode, const Saved& s, const StatsArgs& a, long long N, float* out, int total) {
    return JoinArgs{a.part, a.part + a.plane, a.part + 2 * a.plane, a.tlogit, N, 1, 0, p.vt_fwd, mode, s.st, s.rows, s.tgt,
                    s.top, s.inv_sum, s.mean, out, total};
}

template <class IT, class T, int SPLIT>
int head_fwd(const Plan& p, int mode, const IT* hidden, long long ldh, const IT* weight, const long long* target, const float* centers,
             long long N, int D, int V, long long ignore, int reduction, float* out, void* saved, char* ws, hipStream_t q) {
    const Saved s = saved_of(saved, N);
    const int* rows = nullptr;
    if (mode == kCE) {
        const int nb = cdiv(N, kListBlock);
        int* counts = nb > kListAlone ? reinterpret_cast<int*>(ws + p.counts) : nullptr;
        if (counts) count_rows_kernel<<<nb, kListT, 0, q>>>(target, (int)N, ignore, counts);
        list_rows_kernel<<<nb, kListT, 0, q>>>(target, (int)N, V, ignore, counts, s.st, s.rows, s.tgt,
                                               reduction == DS_REDUCE_NONE ? out : nullptr);
        rows = s.rows;
    }
    // expectation: all rows; the count is written by the first kernel that runs
    const bool set_count = mode == kExpect && (p.few || !p.stage_h);
    const bool clear = mode == kExpect && !set_count;
    if (clear && SPLIT != 3) head_init_kernel<<<1, 1, 0, q>>>(s.st, (int)N);
    float* part = reinterpret_cast<float*>(ws + p.part);
    float* tlogit = reinterpret_cast<float*>(ws + p.tlogit);
    if (p.few) {
        const FewArgs fa{rows, s.st, set_count, (int)N, D, V, 0, mode == kCE ? s.tgt : nullptr, centers, part};
        p.few == 1   ? few_launch<IT, 1>(p, hidden, ldh, weight, fa, q)
        : p.few == 2 ? few_launch<IT, 2>(p, hidden, ldh, weight, fa, q)
                     : few_launch<IT, 4>(p, hidden, ldh, weight, fa, q);
        const int step = p.few * 4;
        join_few_kernel<<<1, 1024, 0, q>>>(JoinArgs{part, part + 1, part + 2, part + 3, step, 4, step, p.few_grid, mode, s.st, s.rows,
                                                    s.tgt, s.top, s.inv_sum, s.mean, out, mode == kCE ? reduction : DS_REDUCE_NONE});
        return launched();
    }
    Operand H, W;
    char* keep = static_cast<char*>(saved);
    operands<IT, T, SPLIT>(p, mode, hidden, ldh, weight, N, D, V, s, rows, true, clear, keep + p.sh, keep + p.sw, H, W, q);
    double* sums = mode == kCE && reduction != DS_REDUCE_NONE ? reinterpret_cast<double*>(ws + p.sums) : nullptr;
    if (p.slim) {
        SlimArgs a = slim_args(p, H, W, s, rows, N, D, V, centers);
        a.set_count = set_count;
        const SlimFwd o{sums ? nullptr : out, sums};
        const int rc = mode == kCE ? slim_fwd<T, SPLIT == 3 ? 2 : 1, kCE>(p, a, o, q) : slim_fwd<T, SPLIT == 3 ? 2 : 1, kExpect>(p, a, o, q);
        if (rc) return rc;
        if (sums) loss_total_kernel<<<1, 256, 0, q>>>(sums, s.st, reduction == DS_REDUCE_MEAN, p.slim_grid, out);
        return launched();
    }
    const StatsArgs sa{V, s.shifts, s.tgt, centers, tlogit, part, (long long)(align256((size_t)p.vt_fwd * N * 4) / 4), (int)N,
                       set_count ? (int)N : 0};
    if (mode == kCE)
        stats_launch<T, SPLIT, kCE>(p, W, H, s, N, D, sa, q);
    else
        stats_launch<T, SPLIT, kExpect>(p, W, H, s, N, D, sa, q);
    if (N <= 32) {
        join_few_kernel<<<1, 1024, 0, q>>>(join_tiles(p, mode, s, sa, N, out, mode == kCE ? reduction : DS_REDUCE_NONE));
        return launched();
    }
    head_join_kernel<<<cdiv(N, 32), 256, 0, q>>>(part, sa.plane, (int)N, p.vt_fwd, s.st, mode, s.rows, s.tgt, tlogit, s.top,
                                                 s.inv_sum, s.mean, out, sums);
    if (sums) loss_total_kernel<<<1, 256, 0, q>>>(sums, s.st, reduction == DS_REDUCE_MEAN, 0, out);
    return launched();
}

template <class T, int SPLIT, int MODE>
void dl_launch(const Plan& p, const Operand& W, const Operand& H, const Saved& s, const BackState* bs, long long N, int D,
               const DlArgs& a, hipStream_t q) {
    const int tiles = cdiv(a.cols, side_of(p.dl_shape)) * cdiv(N, p.dl_shape == kThin ? Thin::BN : side_of(p.dl_shape));
    if (p.dl_shape == kThin)
        head_dl_kernel<T, Thin, SPLIT, MODE><<<tiles, Thin::T, 0, q>>>(W, H, s.st, bs, D, a);
    else if (p.dl_shape == kBig)
        head_dl_big_kernel<T, SPLIT, MODE><<<tiles < cu_count() ? tiles : cu_count(), Big::T, 0, q>>>(W, H, s.st, bs, D, a);
    else if (p.dl_shape == kSmall)
        head_dl_kernel<T, Small, SPLIT, MODE><<<tiles, Small::T, 0, q>>>(W, H, s.st, bs, D, a);
    else if (p.dl_shape == kTiny)
        head_dl_kernel<T, Tiny, SPLIT, MODE><<<tiles, Tiny::T, 0, q>>>(W, H, s.st, bs, D, a);
    else
        head_dl_kernel<T, Sq, SPLIT, MODE><<<tiles, Sq::T, 0, q>>>(W, H, s.st, bs, D, a);
}
template <class IT, class T, class S, int SPLIT, int WHICH>
void grad_shape(bool acc, const Operand& A, const Operand& B, const Saved& s, const BackState* bs, long long n,
                const GradArgs& a, hipStream_t q) {
    int grid = cdiv(a.D, S::BM) * cdiv(n, S::BN) * a.splits;
    if (std::is_same<S, Big>::value && grid > cu_count()) grid = cu_count();
    if (acc)
        head_grad_kernel<T, S, SPLIT, IT, true, WHICH><<<grid, S::T, 0, q>>>(A, B, s.st, bs, a);
    else
        head_grad_kernel<T, S, SPLIT, IT, false, WHICH><<<grid, S::T, 0, q>>>(A, B, s.st, bs, a);
}
template <class IT, class T, int SPLIT, int WHICH>
void grad_launch(ShapeId shape, bool acc, const Operand& A, const Operand& B, const Saved& s, const BackState* bs, long long n,
                 const GradArgs& a, hipStream_t q) {
    if (WHICH == 0 && shape == kThin)
        grad_shape<IT, T, Thin, SPLIT, 0>(acc, A, B, s, bs, n, a, q);
    else if (shape == kBig)
        grad_shape<IT, T, Big, SPLIT, WHICH>(acc, A, B, s, bs, n, a, q);
    else if (shape == kSmall)
        grad_shape<IT, T, Small, SPLIT, WHICH>(acc, A, B, s, bs, n, a, q);
    else if (shape == kTiny)
        grad_shape<IT, T, Tiny, SPLIT, WHICH>(acc, A, B, s, bs, n, a, q);
    else
        grad_shape<IT, T, Sq, SPLIT, WHICH>(acc, A, B, s, bs, n, a, q);
}

template <class IT, class T, int SPLIT>
int head_bwd(const Plan& p, int mode, const IT* hidden, long long ldh, const IT* weight, const long long* target, const float* centers,
             const float* g, long long N, int D, int V, long long ignore, int reduction, void* saved, IT* g_hidden,
             IT* g_weight, char* ws, hipStream_t q) {
    const Saved s = saved_of(saved, N);
    const int* rows = mode == kCE ? s.rows : nullptr;
    BackState* bs = reinterpret_cast<BackState*>(ws + p.bs);
    Upstream up{g, reduction == DS_REDUCE_NONE, reduction == DS_REDUCE_MEAN, rows, mode == kExpect ? s.mean : nullptr};
    Operand H, W;
    char* keep = static_cast<char*>(saved);
    operands<IT, T, SPLIT>(p, mode, hidden, ldh, weight, N, D, V, s, rows, false, false, keep + p.sh, keep + p.sw, H, W, q);
    // dW weighs rows where their upstream differs, and fp32's always; heads on chip weigh dl as they store it
    const bool fold = std::is_same<T, f16>::value && (up.each || SPLIT == 3) && g_weight && !p.slim_back;
    const bool reach = SPLIT == 3 || fold;
    if (!std::is_same<T, bf16>::value && up.each) {
        Features f{};
        if (reach && p.stage_h) f.shifts = s.shifts;
        if constexpr (std::is_same<IT, f16>::value)
            if (fold && !p.stage_h) f = Features{nullptr, hidden, ldh, rows, D, lanes_for(cdiv(D, 8))};
        const long long most = std::max<long long>(centers ? V : 0, f.h ? N * f.L : N);      // threads
        const int blocks = most <= kScaleAlone ? 1 : cdiv(most, 4 * kScaleT) < 256 ? cdiv(most, 4 * kScaleT) : 256;
        if (blocks > 1) back_init_kernel<<<1, 1, 0, q>>>(bs);
        back_scale_kernel<<<blocks, kScaleT, 0, q>>>(up, s.st, centers, V, f, bs);
    }
    Ignored ignored{};
    if (mode == kCE && g_hidden) {
        constexpr int VEC = 16 / sizeof(IT);
        ignored = Ignored{target, (int)N, lanes_for(D % VEC == 0 ? D / VEC : D), D % VEC == 0, ignore};
        if (!p.slim_back) {
            const int blocks = cdiv(N, 4 * 64 / ignored.L * 4);
            zero_ignored_kernel<IT><<<blocks < 4096 ? blocks : 4096, 256, 0, q>>>(ignored, D, s.st, g_hidden);
        }
    }
    Operand Hw = H;      // dW's features
    if constexpr (std::is_same<T, f16>::value)
        if (fold) {
            Hw = Operand{ws + p.hw, p.Dp, N * p.Dp, (int)N, p.Dp};
            const int blocks = cdiv(N * p.Dp, 8 * 256 * 2);
            fold_rows_kernel<SPLIT><<<blocks < 4096 ? blocks : 4096, 256, 0, q>>>(H, s.shifts, s.st, up, bs,
                                                                                  reinterpret_cast<f16*>(ws + p.hw), p.Dp, N * p.Dp);
        }
    T* dl = reinterpret_cast<T*>(ws + p.dl);
    float* dhp = reinterpret_cast<float*>(ws + p.dhp);
    float* dwp = reinterpret_cast<float*>(ws + p.dwp);
    const long long lo = N * p.piece_ld;
    constexpr int kTwo = SPLIT == 1 ? 2 : SPLIT;
    const bool two = SPLIT == 1 && p.dl_planes == 2;
    const int D4 = (D + 3) & ~3;
    for (int v0 = 0; v0 < V; v0 += p.piece) {
        const int cols = V - v0 < p.piece ? V - v0 : p.piece, ld = pad8(cols);
        Operand Wp = W;   // classes [v0, v0 + cols)
        Wp.p = static_cast<const T*>(W.p) + (long long)v0 * W.ld;
        Wp.outer = cols;
        if (p.slim_back) {
            const SlimArgs a = slim_args(p, H, W, s, rows, N, D, V, centers);
            const SlimBwd o{bs, up, g_hidden, g_weight ? dl : nullptr, ld, p.dl_planes, lo, ignored,
                            g_weight && p.pack ? ws + p.bh : nullptr, p.Dp};
            const int rc = mode == kCE ? slim_bwd<T, SPLIT == 3 ? 2 : 1, kCE, IT>(p, a, o, q)
                                       : slim_bwd<T, SPLIT == 3 ? 2 : 1, kExpect, IT>(p, a, o, q);
            if (rc) return rc;
            if (p.pack) Hw = Operand{ws + p.bh, p.Dp, 0, (int)N, p.Dp};
        } else {
            const DlArgs da{v0, cols, s.shifts, s.tgt, centers, s.top, s.inv_sum, s.mean, up, dl, ld, lo};
            if (two)
                mode == kCE ? dl_launch<T, kTwo, kCE>(p, Wp, H, s, bs, N, D, da, q)
                            : dl_launch<T, kTwo, kExpect>(p, Wp, H, s, bs, N, D, da, q);
            else
                mode == kCE ? dl_launch<T, SPLIT, kCE>(p, Wp, H, s, bs, N, D, da, q)
                            : dl_launch<T, SPLIT, kExpect>(p, Wp, H, s, bs, N, D, da, q);
        }
        const Operand G{dl, ld, lo, (int)N, ld};
        if (g_hidden && !p.slim_back) {
            const GradArgs ga{D, cols, p.dh_splits, cols, v0 == 0, rows, g_hidden, dhp, N * D4, up, false};
            if (two)
                grad_launch<IT, T, kTwo, 0>(p.dh, p.dh_part, Wp, G, s, bs, N, ga, q);
            else
                grad_launch<IT, T, SPLIT, 0>(p.dh, p.dh_part, Wp, G, s, bs, N, ga, q);
        }
        if (g_weight) {
            IT* gw = g_weight + (long long)v0 * D;
            const GradArgs ga{D, cols, p.dw_splits, cols, 1, nullptr, gw, dwp, (long long)p.piece * D4, up, reach};
            if (two)
                grad_launch<IT, T, kTwo, 1>(p.dw, p.dw_splits > 1, Hw, G, s, bs, cols, ga, q);
            else
                grad_launch<IT, T, SPLIT, 1>(p.dw, p.dw_splits > 1, Hw, G, s, bs, cols, ga, q);
            if (p.dw_splits > 8 && (long long)cols * D4 <= kShareOuts)
                head_sum_kernel<T, SPLIT, IT, 16><<<cdiv((long long)cols * D4 / 4, 16), 256, 0, q>>>(
                    dwp, (long long)p.piece * D4, p.dw_splits, s.st, bs, cols, D, 1, up, reach, nullptr, gw);
            else if (p.dw_splits > 1)
                head_sum_kernel<T, SPLIT, IT, 1><<<cdiv((long long)cols * D4 / 4, 256), 256, 0, q>>>(
                    dwp, (long long)p.piece * D4, p.dw_splits, s.st, bs, cols, D, 1, up, reach, nullptr, gw);
        }
    }
    if (g_hidden && p.dh_part && !p.slim_back) {
        const bool many = p.dh_splits > 8 && N * D4 <= kShareOuts;
        const int blocks = cdiv(N * (D4 / 4), many ? 16 : 256), grid = blocks < 16384 ? blocks : 16384;
        if (many)
            head_sum_kernel<T, SPLIT, IT, 16><<<grid, 256, 0, q>>>(dhp, N * D4, p.dh_splits, s.st, bs, (int)N, D, 0, up, false, rows,
                                                                   g_hidden);
        else
            head_sum_kernel<T, SPLIT, IT, 1><<<grid, 256, 0, q>>>(dhp, N * D4, p.dh_splits, s.st, bs, (int)N, D, 0, up, false, rows,
                                                                  g_hidden);
    }
    return launched();
}

template <class F32, class F16, class BF16>
int by_type(int dtype, F32 f32, F16 h, BF16 b) {
    return dtype == DS_F32 ? f32() : dtype == DS_F16 ? h() : b();
}

// saved NULL: no backward follows
int fwd_any(int mode, const void* hidden, long long ldh, const void* weight, const long long* target, const float* centers,
            int dtype, long long N, int D, int V, long long ignore, int reduction, float* out, void* saved, void* ws,
            size_t bytes, void* stream) {
    if (!hidden || !weight || !out) return DS_ERR_INVALID_ARG;
    const int rc = check_sizes(dtype, N, D, V, ldh);
    if (rc) return rc;
    const Plan p = plan_of(mode, dtype, N, D, V, ldh, !saved);
    if (!ws || bytes < p.fwd_total || misaligned(ws) || misaligned(saved)) return DS_ERR_WORKSPACE;
    if ((!p.stage_w && misaligned(weight)) || (!p.stage_h && misaligned(hidden))) return DS_ERR_INVALID_ARG;
    char* w = static_cast<char*>(ws);
    if (!saved) saved = w + p.alone;
    hipStream_t q = static_cast<hipStream_t>(stream);
#define DS_GO(IT, T, SP)                                                                                                     \
    [&] {                                                                                                                    \
        return head_fwd<IT, T, SP>(p, mode, static_cast<const IT*>(hidden), ldh, static_cast<const IT*>(weight), target, centers, \
                                   N, D, V, ignore, reduction, out, saved, w, q);                                            \
    }
    return by_type(dtype, DS_GO(float, f16, 3), DS_GO(f16, f16, 1), DS_GO(bf16, bf16, 1));
#undef DS_GO
}

int bwd_any(int mode, const void* hidden, long long ldh, const void* weight, const long long* target, const float* centers,
            const float* g, int dtype, long long N, int D, int V, long long ignore, int reduction, void* saved, void* g_hidden,
            void* g_weight, void* ws, size_t bytes, void* stream) {
    if (!hidden || !weight || !saved || !g || (!g_hidden && !g_weight)) return DS_ERR_INVALID_ARG;
    const int rc = check_sizes(dtype, N, D, V, ldh);
    if (rc) return rc;
    const Plan p = plan_of(mode, dtype, N, D, V, ldh);
    if (!ws || bytes < p.bwd_total || misaligned(ws) || misaligned(saved)) return DS_ERR_WORKSPACE;
    if ((!p.stage_w && misaligned(weight)) || (!p.stage_h && misaligned(hidden)) || misaligned(g_hidden) || misaligned(g_weight))
        return DS_ERR_INVALID_ARG;
    char* w = static_cast<char*>(ws);
    hipStream_t q = static_cast<hipStream_t>(stream);
#define DS_GO(IT, T, SP)                                                                                                       \
    [&] {                                                                                                                      \
        return head_bwd<IT, T, SP>(p, mode, static_cast<const IT*>(hidden), ldh, static_cast<const IT*>(weight), target, centers, \
                                   g, N, D, V, ignore, reduction, saved, static_cast<IT*>(g_hidden),                           \
                                   static_cast<IT*>(g_weight), w, q);                                                          \
    }
    return by_type(dtype, DS_GO(float, f16, 3), DS_GO(f16, f16, 1), DS_GO(bf16, bf16, 1));
#undef DS_GO
}

}  // namespace
}  // namespace ds

extern "C" {

size_t ds_linear_ce_saved_bytes(int dtype, long long N, int D, int V, long long ldh) {
    return ds::check_sizes(dtype, N, D, V, ldh) ? 0 : ds::plan_of(ds::kCE, dtype, N, D, V, ldh).saved_total;
}
size_t ds_linear_ce_workspace_bytes(int dtype, long long N, int D, int V, long long ldh, int backward) {
    if (ds::check_sizes(dtype, N, D, V, ldh)) return 0;
    const ds::Plan p = ds::plan_of(ds::kCE, dtype, N, D, V, ldh);
    return backward ? p.bwd_total : p.fwd_total;
}
int ds_linear_ce_fwd(const void* hidden, long long ldh, const void* weight, const long long* target, int dtype, long long N,
                     int D, int V, long long ignore_index, int reduction, float* loss, void* saved, void* workspace,
                     size_t workspace_bytes, void* stream) {
    if (!target || !saved || reduction < DS_REDUCE_NONE || reduction > DS_REDUCE_MEAN) return DS_ERR_INVALID_ARG;
    return ds::fwd_any(ds::kCE, hidden, ldh, weight, target, nullptr, dtype, N, D, V, ignore_index, reduction, loss, saved,
                       workspace, workspace_bytes, stream);
}
size_t ds_linear_ce_eval_workspace_bytes(int dtype, long long N, int D, int V, long long ldh) {
    return ds::check_sizes(dtype, N, D, V, ldh) ? 0 : ds::plan_of(ds::kCE, dtype, N, D, V, ldh, true).fwd_total;
}
int ds_linear_ce_eval(const void* hidden, long long ldh, const void* weight, const long long* target, int dtype, long long N,
                      int D, int V, long long ignore_index, int reduction, float* loss, void* workspace, size_t workspace_bytes,
                      void* stream) {
    if (!target || reduction < DS_REDUCE_NONE || reduction > DS_REDUCE_MEAN) return DS_ERR_INVALID_ARG;
    return ds::fwd_any(ds::kCE, hidden, ldh, weight, target, nullptr, dtype, N, D, V, ignore_index, reduction, loss, nullptr,
                       workspace, workspace_bytes, stream);
}
int ds_linear_ce_bwd(const void* hidden, long long ldh, const void* weight, const long long* target, const float* g_loss,
                     int dtype, long long N, int D, int V, long long ignore_index, int reduction, const void* saved,
                     void* g_hidden, void* g_weight, void* workspace, size_t workspace_bytes, void* stream) {
    if (!target || reduction < DS_REDUCE_NONE || reduction > DS_REDUCE_MEAN) return DS_ERR_INVALID_ARG;
    return ds::bwd_any(ds::kCE, hidden, ldh, weight, target, nullptr, g_loss, dtype, N, D, V, ignore_index, reduction,
                       const_cast<void*>(saved), g_hidden, g_weight, workspace, workspace_bytes, stream);
}

size_t ds_bin_expect_saved_bytes(int dtype, long long N, int D, int V, long long ldh) {
    return ds::check_sizes(dtype, N, D, V, ldh) ? 0 : ds::plan_of(ds::kExpect, dtype, N, D, V, ldh).saved_total;
}
size_t ds_bin_expect_workspace_bytes(int dtype, long long N, int D, int V, long long ldh, int backward) {
    if (ds::check_sizes(dtype, N, D, V, ldh)) return 0;
    const ds::Plan p = ds::plan_of(ds::kExpect, dtype, N, D, V, ldh);
    return backward ? p.bwd_total : p.fwd_total;
}
int ds_bin_expect_fwd(const void* hidden, long long ldh, const void* weight, const float* centers, int dtype, long long N, int D,
                      int V, float* out, void* saved, void* workspace, size_t workspace_bytes, void* stream) {
    if (!centers || !saved) return DS_ERR_INVALID_ARG;
    return ds::fwd_any(ds::kExpect, hidden, ldh, weight, nullptr, centers, dtype, N, D, V, 0, DS_REDUCE_NONE, out, saved,
                       workspace, workspace_bytes, stream);
}
size_t ds_bin_expect_eval_workspace_bytes(int dtype, long long N, int D, int V, long long ldh) {
    return ds::check_sizes(dtype, N, D, V, ldh) ? 0 : ds::plan_of(ds::kExpect, dtype, N, D, V, ldh, true).fwd_total;
}
int ds_bin_expect_eval(const void* hidden, long long ldh, const void* weight, const float* centers, int dtype, long long N, int D,
                       int V, float* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!centers) return DS_ERR_INVALID_ARG;
    return ds::fwd_any(ds::kExpect, hidden, ldh, weight, nullptr, centers, dtype, N, D, V, 0, DS_REDUCE_NONE, out, nullptr,
                       workspace, workspace_bytes, stream);
}
int ds_bin_expect_bwd(const void* hidden, long long ldh, const void* weight, const float* centers, const float* g_out, int dtype,
                      long long N, int D, int V, const void* saved, void* g_hidden, void* g_weight, void* workspace,
                      size_t workspace_bytes, void* stream) {
    if (!centers) return DS_ERR_INVALID_ARG;
    return ds::bwd_any(ds::kExpect, hidden, ldh, weight, nullptr, centers, g_out, dtype, N, D, V, 0, DS_REDUCE_NONE,
                       const_cast<void*>(saved), g_hidden, g_weight, workspace, workspace_bytes, stream);
}

}  // extern "C"
