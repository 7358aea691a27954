// ds_gemm.h -- the matrix core shared by the classification head (ds_head.hip) and the matrix update (ds_ortho.hip).
//
// One workgroup forms a BM x BN tile of C[m][n] = sum_k A(m,k) B(n,k) with v_mfma_f32_16x16x32.  Either operand may be
// stored with k contiguous (kK: row m of A holds its k values) or with m contiguous (kM: row k holds all m, i.e. the
// transposed matrix), so that none of the products here needs a transposed copy: W serves logits = H W^T as kK and
// dH = dL W as kM.  A kM tile lies in LDS as it lies in memory, and ds_read_b64_tr_b16 hands every lane the four k values of
// its m (measured layout: lane 4r+c of a 16-lane group reads four values of row r, lane i receives rows 0..3 of column i).
//
// Numbers wider than 16 bits go through as two fp16 planes x = hi + lo (22 bits, after an exact power-of-two scale that the
// caller keeps): lo*hi + hi*lo + hi*hi go into the same fp32 accumulators.  What is dropped, lo*lo, is 2^-22 of the product.
// PA and PB say how many planes A and B have.  Three 16-bit products cost a third of the 16-bit rate, still above the rate of
// fp32 matrix instructions (1/16 of it).
//
// Rows and columns beyond an operand's bounds read as zero (buffer loads whose offset is out of range), so every size works
// without padded copies; only the contiguous extent must be a multiple of 8 elements and 16-byte aligned.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "ds_common.h"

namespace ds {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

__host__ __device__ constexpr int cdiv(int a, int b) { return (int)(((unsigned)a + (unsigned)b - 1) / (unsigned)b); }
inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }
inline int cdiv(long long a, int b) { return cdiv(a, (long long)b); }
inline int pad8(int x) { return (x + 7) & ~7; }
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

enum Lay { kK = 0, kM = 1 };   // which index of the operand is contiguous

struct Operand {
    const void* p;      // 16-bit elements, 16-byte aligned
    long long ld;       // elements between stored rows, a multiple of 8
    long long lo;       // elements from the hi plane to the lo plane (two planes)
    int outer;          // stored rows that exist
    int inner;          // elements of a row that may be read, a multiple of 8 (what lies beyond the matrix must be zero)
};

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, f16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

constexpr int kBK = 64;                 // k per step: 128 bytes of a kK row = 8 chunks of 16 bytes
constexpr unsigned kOut = 0xfffffff0u;  // an offset beyond every descriptor: the load returns zero

// a workgroup's shape: BM x BN outputs, WM x WN waves
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, T = 64 * WM_ * WN_;
    static constexpr int FM = BM_ / WM_ / 16, FN = BN_ / WN_ / 16;   // 16x16 fragments of a wave
    static constexpr int kLds = 2 * (BM_ + BN_) * kBK * 2;           // two steps of one plane
};

// byte offset of 16-byte chunk c of row r in an LDS tile.  kK: the eight chunks of a row trade places by the row's low bits,
// so that the 16 rows of a ds_read_b128 spread over all banks.  kM: 32-byte granules trade places by those bits of k in which
// the rows of one transposing read differ.
template <Lay L, int R>
__device__ __forceinline__ int lds_chunk(int r, int c) {
    if (L == kK) return r * (kBK * 2) + ((c ^ (r & 7)) << 4);
    const int swz = ((r & 3) | ((r >> 1) & 4)) & (R / 16 - 1);
    return r * (R * 2) + (((((c >> 1) ^ swz) << 1) | (c & 1)) << 4);
}

// One operand's tile on its way from memory to LDS: R x 64 elements, N16 16-byte chunks per thread, staged in registers.
template <Lay L, int R, int T>
struct Stager {
    static constexpr int N16 = R * kBK * 2 / 16 / T;
    static constexpr int CPR = (L == kK ? kBK : R) / 8;              // chunks per stored row
    i32x4 v[N16];

    __device__ __forceinline__ void load(const Operand& o, int r0, int k0, bool lo, int tid) {
        // descriptor at the tile's corner: 32-bit offsets stay small however large the matrix is
        const long long corner = L == kK ? (long long)r0 * o.ld + k0 : (long long)k0 * o.ld + r0;
        const rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(o.p) + 2 * (corner + (lo ? o.lo : 0))), 0, 0x7fffffff, 0x00020000);
        const int outer0 = L == kK ? r0 : k0, inner0 = L == kK ? k0 : r0;
#pragma unroll
        for (int i = 0; i < N16; ++i) {
            const int c = tid + i * T, r = c / CPR, cc = c % CPR;
            const bool in = outer0 + r < o.outer && inner0 + cc * 8 < o.inner;
            const unsigned off = in ? (unsigned)(r * (int)o.ld + cc * 8) * 2u : kOut;
            v[i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
        }
    }
    __device__ __forceinline__ void store(char* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < N16; ++i) {
            const int c = tid + i * T;
            *reinterpret_cast<i32x4*>(lds + lds_chunk<L, R>(c / CPR, c % CPR)) = v[i];
        }
    }
};

// Fragments of 16 rows and 32 k out of an LDS tile: lane l holds row l % 16, k = 8 (l / 16) .. + 7.  Fragment i of a wave whose
// rows begin at m0 (a multiple of 16 times the power of two above i), sub-step kk of the tile's two: what depends on the lane
// is one number, the rest constants and exclusive-ors of constants.
template <Lay L, int R>
struct Fragments {
    int base;
    __device__ __forceinline__ Fragments(int m0, int lane) {
        if (L == kK)
            base = lds_chunk<L, R>(m0 + (lane & 15), lane >> 4);
        else
            base = lds_chunk<L, R>((lane >> 4) * 8 + ((lane >> 2) & 3), m0 / 8 + ((lane >> 1) & 1)) + (lane & 1) * 8;
    }
    __device__ __forceinline__ s16x8 get(const char* tile, int i, int kk) const {
        if (L == kK) return *reinterpret_cast<const s16x8*>(tile + (base ^ (kk << 6)) + i * 16 * (kBK * 2));
        typedef __attribute__((address_space(3))) s16x4* lp;
        const char* p = tile + (base ^ (i << 5)) + kk * 32 * (R * 2);
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p + 4 * (R * 2)));
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// acc[i][j][e]: C at m = m0 + wave's row + 16 i + 4 (lane / 16) + e, n = n0 + wave's column + 16 j + lane % 16, over k in
// [kbeg, kend) (kbeg a multiple of 64).  `lds`: lds_bytes<S, PA, PB>() bytes.  Ends behind a barrier: the caller may reuse
// `lds`.  A step brings all planes of both operands and adds its products from them, so that each plane is moved once and a
// step's latency is covered by up to three products.  128 x 128 tiles then keep one step in LDS (the next one
// waits in registers), which leaves room for two workgroups a CU.  Eight waves a 128 x 128 tile, two a SIMD, so that one's
// LDS reads run beside the other's products: 512 x 4608 x 512 of two planes, within an update, 18.6 us, 21.2 with four waves;
// two buffers or loads two steps ahead gained nothing.
template <class S, int PA, int PB>
constexpr int lds_buffers() { return PA + PB > 2 && S::BM * S::BN > 64 * 128 ? 1 : 2; }
template <class S, int PA, int PB>
constexpr int lds_bytes() { return lds_buffers<S, PA, PB>() * (PA * S::BM + PB * S::BN) * kBK * 2; }

template <class T, class S, Lay LA, Lay LB, int PA, int PB>
__device__ __forceinline__ void gemm_tile(const Operand& A, const Operand& B, int m0, int n0, int kbeg, int kend, char* lds,
                                          f32x4 (&acc)[S::FM][S::FN]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave / S::WN) * S::FM * 16, wn = (wave % S::WN) * S::FN * 16;
    constexpr int kA = S::BM * kBK * 2, kB = S::BN * kBK * 2, kBuf = PA * kA + PB * kB;
    constexpr int NB = lds_buffers<S, PA, PB>();
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int j = 0; j < S::FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const Fragments<LA, S::BM> fa(wm, lane);
    const Fragments<LB, S::BN> fb(wn, lane);
    Stager<LA, S::BM, S::T> sa[PA];
    Stager<LB, S::BN, S::T> sb[PB];
    const int steps = (kend - kbeg + kBK - 1) / kBK;
    auto load = [&](int s) {
#pragma unroll
        for (int p = 0; p < PA; ++p) sa[p].load(A, m0, kbeg + s * kBK, p == 1, tid);
#pragma unroll
        for (int p = 0; p < PB; ++p) sb[p].load(B, n0, kbeg + s * kBK, p == 1, tid);
    };
    auto store = [&](char* buf) {
#pragma unroll
        for (int p = 0; p < PA; ++p) sa[p].store(buf + p * kA, tid);
#pragma unroll
        for (int p = 0; p < PB; ++p) sb[p].store(buf + PA * kA + p * kB, tid);
    };
    if (steps > 0) {
        load(0);
        store(lds);
    }
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const char* buf = lds + (NB == 2 ? (s & 1) * kBuf : 0);
        const bool more = s + 1 < steps;
        if (more) load(s + 1);
#pragma unroll
        for (int kk = 0; kk < kBK / 32; ++kk) {
            s16x8 a[PA][S::FM], b[PB][S::FN];
#pragma unroll
            for (int p = 0; p < PA; ++p)
#pragma unroll
                for (int i = 0; i < S::FM; ++i) a[p][i] = fa.get(buf + p * kA, i, kk);
#pragma unroll
            for (int p = 0; p < PB; ++p)
#pragma unroll
                for (int j = 0; j < S::FN; ++j) b[p][j] = fb.get(buf + PA * kA + p * kB, j, kk);
#pragma unroll
            for (int pair = PA + PB - 2; pair >= 0; --pair) {      // (lo, hi) and (hi, lo), as far as there are any, then (hi, hi)
                const int p = pair > 0 && PA == 2 && pair == PA + PB - 2 ? 1 : 0, q = pair > 0 && !p ? 1 : 0;
#pragma unroll
                for (int i = 0; i < S::FM; ++i)
#pragma unroll
                    for (int j = 0; j < S::FN; ++j) acc[i][j] = mfma(a[PA == 2 ? p : 0][i], b[PB == 2 ? q : 0][j], acc[i][j], T());
            }
        }
        if (NB == 1) __syncthreads();
        if (more) store(lds + (NB == 2 ? ((s + 1) & 1) * kBuf : 0));
        __syncthreads();
    }
}

// ---- the large shape: 256 x 256, eight waves in two groups that take turns ---------------------------------------------
//
// At this size a step (64 k) is 2048 cycles of matrix instructions and 1536 cycles of LDS reads, which only run side by side
// if different waves do them: every SIMD holds one wave of each group, and while one group multiplies, the other fetches its
// operands of the next 32 k; an s_barrier ends each turn.  Tiles come to LDS by DMA (buffer_load ... lds: no registers, no
// LDS store instructions), the next step's under way during the whole current one, and the next tile's first step during the
// last one of the tile before, so that a workgroup that goes through several tiles waits for memory once.
//   4096 x 4096 x 4096 bf16: 103 us = 1337 TFLOP/s, 109 us with one operand kM (register-staged 128 x 128 tiles: 166 us; the
//   same 256 x 256 tile with all waves in step: 142 us); a library product of that size reaches 1436 TFLOP/s here.

// 16 bytes per lane from a buffer to LDS at `lds` + 16 * lane; out-of-range lanes write zeros.  In assembly because the
// compiler, which cannot tell the two buffers apart, would wait for every such load before the next LDS read; wait_dma()
// before a barrier is the wait.  The instruction has no destination register.  (m0 holds the LDS address; the compiler warns
// that it reserves the register for itself, and sets it anew before each use of its own.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(unsigned lds, unsigned off, rsrc_t r) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(off), "s"(r)
                 : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void turn() {   // end of a turn; nothing moves across it
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// a wave's share of one operand's tile: N16 DMA instructions, offsets kept per lane
template <Lay L, int R, int T>
struct Mover {
    static constexpr int N16 = R * kBK * 2 / 16 / T;
    static constexpr int CPR = (L == kK ? kBK : R) / 8;
    unsigned off[N16];
    // LDS slot p holds row r = p / CPR and, of that row, the chunk c that lds_chunk() puts there (its permutations are
    // their own inverse)
    static __device__ __forceinline__ void at(int i, int tid, int& r, int& c) {
        const int p = i * T + tid, x = p % CPR;
        r = p / CPR;
        if (L == kK) {
            c = x ^ (r & 7);
        } else {
            const int swz = ((r & 3) | ((r >> 1) & 4)) & (R / 16 - 1);
            c = (((x >> 1) ^ swz) << 1) | (x & 1);
        }
    }
    __device__ __forceinline__ void init(const Operand& o, int r0, int tid) {
#pragma unroll
        for (int i = 0; i < N16; ++i) {
            int r, c;
            at(i, tid, r, c);
            const bool in = L == kK ? r0 + r < o.outer : r0 + c * 8 < o.inner;
            off[i] = in ? (unsigned)(r * (int)o.ld + c * 8) * 2u : kOut;
        }
    }
    __device__ __forceinline__ void move(const Operand& o, int r0, int k0, bool lo, unsigned lds, int tid) const {
        const long long corner = L == kK ? (long long)r0 * o.ld + k0 : (long long)k0 * o.ld + r0;
        const rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(static_cast<const char*>(o.p) + 2 * (corner + (lo ? o.lo : 0))), 0, 0x7fffffff, 0x00020000);
        const unsigned base = __builtin_amdgcn_readfirstlane(lds + (tid >> 6) * 1024);
        const int left = (L == kK ? o.inner : o.outer) - k0;
        if (left >= kBK) {
#pragma unroll
            for (int i = 0; i < N16; ++i) dma16(base + i * T * 16, off[i], rs);
        } else {
#pragma unroll
            for (int i = 0; i < N16; ++i) {
                int r, c;
                at(i, tid, r, c);
                dma16(base + i * T * 16, (L == kK ? c * 8 : r) < left ? off[i] : kOut, rs);
            }
        }
    }
};

typedef Shape<256, 256, 2, 4> Big;

// Where split sp of a sum over k begins, `per` (a multiple of 64) each.  A split behind the last step begins at the next multiple
// of 64, where every operand ends: from k itself a row's padding would run into the row after it.
__device__ __forceinline__ int split_start(int sp, int per, int k) { return min(sp * per, (k + kBK - 1) / kBK * kBK); }

// What a workgroup multiplies next.  A tile of no steps is given one step of zeros.
struct Job {
    Operand A, B;
    int m0, n0, kbeg, kend;
};

// Planes are taken one pair after the other, a step of the same k each.
template <class T, Lay LA, Lay LB, int PA, int PB>
struct TileStream {
    using S = Big;
    static constexpr int kPairs = PA + PB - 1;     // (lo, hi) and (hi, lo), as far as there are any, and (hi, hi)
    Mover<LA, S::BM, S::T> ma;
    Mover<LB, S::BN, S::T> mb;
    Job job;
    int steps, parity, tid;
    bool edge;       // the lane offsets are those of a tile that lies across an edge (or of none)
    char* lds;       // S::kLds bytes that nothing else uses

    __device__ __forceinline__ void move(int s) {
        const int k0 = job.kbeg + s / kPairs * kBK, ph = s % kPairs;
        const unsigned buf = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds +
                             ((s + parity) & 1) * ((S::BM + S::BN) * kBK * 2);
        ma.move(job.A, job.m0, k0, PA == 2 && ph == 0, buf, tid);
        mb.move(job.B, job.n0, k0, PB == 2 && ph == PA - 1, buf + S::BM * kBK * 2, tid);
    }
    // takes up a job and sets its first step under way
    __device__ __forceinline__ void start(const Job& j) {
        job = j;
        const int n = (j.kend - j.kbeg + kBK - 1) / kBK * kPairs;
        steps = n > 0 ? n : 1;
        // lane offsets differ from the tile before only where one of the two lies across an edge
        const bool e = j.m0 + S::BM > (LA == kK ? j.A.outer : j.A.inner) || j.n0 + S::BN > (LB == kK ? j.B.outer : j.B.inner);
        if (e || edge) {
            ma.init(j.A, j.m0, tid);
            mb.init(j.B, j.n0, tid);
        }
        edge = e;
        move(0);
    }
    __device__ __forceinline__ TileStream(char* lds_, const Job& j) : parity(0), tid(threadIdx.x), edge(true), lds(lds_) { start(j); }

    __device__ __forceinline__ void fetch(const char* buf, int kk, const Fragments<LA, S::BM>& fa, const Fragments<LB, S::BN>& fb,
                                          s16x8 (&a)[S::FM], s16x8 (&b)[S::FN]) const {
#pragma unroll
        for (int j = 0; j < S::FN; ++j) b[j] = fb.get(buf + S::BM * kBK * 2, j, kk);
#pragma unroll
        for (int i = 0; i < S::FM; ++i) a[i] = fa.get(buf, i, kk);
    }
    template <bool ZERO>      // ZERO: the sums begin here
    __device__ __forceinline__ void add(const s16x8 (&a)[S::FM], const s16x8 (&b)[S::FN], f32x4 (&acc)[S::FM][S::FN]) const {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int j = 0; j < S::FN; ++j) acc[i][j] = mfma(a[i], b[j], ZERO ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[i][j], T());
        __builtin_amdgcn_s_setprio(0);
    }
    template <bool FIRST, class Next>
    __device__ __forceinline__ void step(int s, int n, int group, const Fragments<LA, S::BM>& fa, const Fragments<LB, S::BN>& fb,
                                         f32x4 (&acc)[S::FM][S::FN], Next& next) {
        const char* buf = lds + ((s + parity) & 1) * ((S::BM + S::BN) * kBK * 2);
        s16x8 a[S::FM], b[S::FN];
        fetch(buf, 0, fa, fb, a, b);
        // the other buffer was read for the last time in the turn before this one (group 1's second half of step s - 1)
        if (s + 1 < n) {
            move(s + 1);
        } else {
            Job j;
            if (next(j)) {
                parity = (parity + n) & 1;
                start(j);
            }
        }
        wait_lds();
        turn();
        add<FIRST>(a, b, acc);
        turn();
        fetch(buf, 1, fa, fb, a, b);
        wait_lds();
        // both groups' shares of the next step have arrived when the turn ends in which group 1 reads this step's last
        if (group == 1 && s + 1 < n) wait_dma();
        turn();
        add<false>(a, b, acc);
        if (group == 0 && s + 1 < n) wait_dma();
        turn();
    }

    // Multiplies the job that start() took up.  next(Job&) -> bool names the one after it, whose first step is then under way
    // on return (waiting for it here, so that the caller's stores need not be waited for with it, cost 4 %: 4.09 against
    // 4.25 ms for 8192 x 65536 x 1024).  All waves leave together; acc as in gemm_tile.
    template <class Next>
    __device__ __forceinline__ void multiply(f32x4 (&acc)[S::FM][S::FN], Next next) {
        const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = wave / S::WN;
        const int wm = group * S::FM * 16, wn = (wave % S::WN) * S::FN * 16;
        const Fragments<LA, S::BM> fa(wm, lane);
        const Fragments<LB, S::BN> fb(wn, lane);
        wait_dma();
        turn();
        if (group == 1) turn();       // half a step behind the other group from here on
        const int n = steps;
        step<true>(0, n, group, fa, fb, acc, next);
        // not unrolled, nor its last step peeled: the compiler would move all sums between two sets of registers
#pragma clang loop unroll(disable)
        for (int s = 1; s < n; ++s) step<false>(s, n, group, fa, fb, acc, next);
        if (group == 0) turn();
    }
};

// Tile t of mt x nt in the order in which they are taken: workgroup b runs on XCD b % 8, each with an L2 of its own, so every
// XCD gets a contiguous share (turn_of), and inside it bands of four tile columns are gone through row by row (at): the tiles in
// flight on an XCD share a few rows and columns.  Split sums count their splits as tile rows, split by split, so that an XCD
// works on few ranges of k at a time.  (No division but by the few columns of a last, narrower band: the next tile is looked up
// while a turn waits for it.)
struct Order {
    int tiles, mt, nt, q, r;
    float inv;       // 1 / (4 mt)
    __device__ __forceinline__ Order(int tiles_, int mt_, int nt_) : tiles(tiles_), mt(mt_), nt(nt_), q(tiles_ >> 3), r(tiles_ & 7) {
        inv = 1.f / (4.f * mt_);
    }
    __device__ __forceinline__ int turn_of(int t) const {
        const int x = t & 7;
        return x * q + (x < r ? x : r) + (t >> 3);
    }
    __device__ __forceinline__ void operator()(int t, int& m, int& n) const { at(turn_of(t), m, n); }
    __device__ __forceinline__ void at(int u, int& m, int& n) const {
        int band = __builtin_amdgcn_readfirstlane((int)((float)u * inv));      // off by one at most, or a little more far out
        while (band * 4 * mt > u) --band;
        while ((band + 1) * 4 * mt <= u) ++band;
        const int in = u - band * 4 * mt, w = nt - band * 4;
        if (w >= 4) {
            n = band * 4 + (in & 3);
            m = in >> 2;
        } else {
            n = band * 4 + in % w;
            m = in / w;
        }
    }
};

// x as two fp16 numbers: hi = x to 11 bits, lo = the rest to 11 bits.  Where hi is not finite lo is 0, so that an infinity
// stays one instead of becoming inf - inf.
__device__ __forceinline__ void split16(float x, f16& hi, f16& lo) {
    hi = (f16)x;
    const float h = (float)hi;
    lo = __builtin_isfinite(h) ? (f16)(x - h) : (f16)0.f;
}

// four consecutive values to 16-bit storage, one or two planes
template <int SPLIT>
__device__ __forceinline__ void put4(f16* p, long long lo, const float (&v)[4]) {
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (SPLIT == 3) {
            f16 a, b;
            split16(v[e], a, b);
            h[e] = a;
            l[e] = b;
        } else {
            h[e] = (f16)v[e];
        }
    }
    *reinterpret_cast<f16x4*>(p) = h;
    if (SPLIT == 3) *reinterpret_cast<f16x4*>(p + lo) = l;
}
// as split16, to 8 bits each
__device__ __forceinline__ void split16(float x, bf16& hi, bf16& lo) {
    hi = (bf16)x;
    const float h = (float)hi;
    lo = __builtin_isfinite(h) ? (bf16)(x - h) : (bf16)0.f;
}
template <int SPLIT>
__device__ __forceinline__ void put4(bf16* p, long long lo, const float (&v)[4]) {
    bf16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bf16 a, b;
        split16(v[e], a, b);
        h[e] = a;
        l[e] = b;
    }
    *reinterpret_cast<bf16x4*>(p) = h;
    if (SPLIT == 3) *reinterpret_cast<bf16x4*>(p + lo) = l;
}

// Fragments i and i + 1 of a row in 16 bits: lane group q holds four elements from 4 q of either (x, y) and gets eight
// consecutive ones of the 32, from 8 q: stores of 16 bytes a lane, 64 a row at a time, instead of 8 and 32.
__device__ __forceinline__ void eight_of(s16x4 x, s16x4 y, s16x8& out) {
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    const u2 a = __builtin_bit_cast(u2, x), b = __builtin_bit_cast(u2, y);
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        // groups 0 1 2 3 of a and b -> a0 a1 b0 b1 and a2 a3 b2 b3 -> a0 a2 b0 b2 and a1 a3 b1 b3
        const auto half = __builtin_amdgcn_permlane32_swap(a[k], b[k], false, false);
        const auto quarter = __builtin_amdgcn_permlane16_swap(half[0], half[1], false, false);
        w[k] = quarter[0];
        w[2 + k] = quarter[1];
    }
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    out = __builtin_bit_cast(s16x8, u4{w[0], w[1], w[2], w[3]});
}
template <class T>
__device__ __forceinline__ s16x4 round4(const f32x4& v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (T)v[e];
    return __builtin_bit_cast(s16x4, r);
}

// the low plane of four values
template <class T = f16>
__device__ __forceinline__ s16x4 rest4(const f32x4& v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        T h, l;
        split16(v[e], h, l);
        r[e] = l;
    }
    return __builtin_bit_cast(s16x4, r);
}

// up to four consecutive outputs of a row of `n` elements, at element c of the row; rows need only their type's alignment
template <class O>
__device__ __forceinline__ void put_row4(O* row, int c, int n, const float (&v)[4]) {
    if (c + 4 <= n) {
        typedef O o4 __attribute__((ext_vector_type(4)));
        typedef o4 loose __attribute__((aligned(sizeof(O))));
        o4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = (O)v[e];
        *reinterpret_cast<loose*>(row + c) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < n) row[c + e] = (O)v[e];
    }
}

// fragments i and i + 1 of a row of `n` elements of type O: x and y from element c + 4 (lane / 16) and 16 on, c that of the
// fragments' first element.  All four lane groups of a row call together.
template <class O>
__device__ __forceinline__ void put_row8(O* row, int c, int n, int lane, const f32x4& x, const f32x4& y) {
    if constexpr (sizeof(O) == 2) {
        typedef O o8 __attribute__((ext_vector_type(8)));
        typedef o8 loose __attribute__((aligned(sizeof(O))));
        s16x8 w;
        eight_of(round4<O>(x), round4<O>(y), w);
        const o8 v = __builtin_bit_cast(o8, w);
        c += (lane >> 4) * 8;
        if (c + 8 <= n) {
            *reinterpret_cast<loose*>(row + c) = v;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < n) row[c + e] = v[e];
        }
    } else {
        c += (lane >> 4) * 4;
        const float v[4] = {x[0], x[1], x[2], x[3]}, w[4] = {y[0], y[1], y[2], y[3]};
        put_row4(row, c, n, v);
        put_row4(row, c + 16, n, w);
    }
}

// the power of two that brings a largest magnitude `amax` into [2^14, 2^15): fp16 keeps a factor of two of headroom.  As an
// exponent, for ldexpf: that of the smallest float32 is 163, whose power is none
__device__ __forceinline__ int shift_for(float amax) { return amax > 0.f && __builtin_isfinite(amax) ? 14 - ilogbf(amax) : 0; }
__device__ __forceinline__ f32x4 scaled(const f32x4& v, int e) {
    return f32x4{ldexpf(v[0], e), ldexpf(v[1], e), ldexpf(v[2], e), ldexpf(v[3], e)};
}

// ---- which shape a product takes, and over how many workgroups its sum is split (host) -----------------------------------
enum ShapeId { kSq, kThin, kBig, kSmall, kTiny };
typedef Shape<128, 128, 4, 2> Sq;
typedef Shape<64, 64, 2, 2> Small;
typedef Shape<32, 32, 2, 2> Tiny;     // where there are fewer tiles than CUs: 512 x 512 x 512 of two planes 4.8 us, Small 7.5

inline int side_of(ShapeId s) {      // Thin: along m
    return s == kBig ? Big::BM : s == kSmall ? Small::BM : s == kTiny ? Tiny::BM : Sq::BM;
}

struct Cut {
    ShapeId shape;
    int splits;
};
// tiles(b): tiles of b x b; area: outputs; pairs: products a step (three of two planes each, two of two planes and one).
// strided: an operand is kM.  Its rows of 32 elements are half a cache line: 32 x 32 tiles take a quarter longer
// where several share a CU.
template <class Tiles>
inline Cut cut_of(Tiles tiles, double area, long long K, int pairs, bool may_split, bool strided, int cus) {
    // us a step of 64 k: `step` of a CU's time with `at_once` workgroups on it, `alone` at least; `ends`: start and end of a
    // tile.  Measured at k = 512 and 2048 with half a workgroup to sixteen a CU; in TFLOP/s of 16-bit products with the chip
    // full: 256 x 256 tiles 1330, 128 x 128 900, 64 x 64 660, 32 x 32 290; three products a step 1365, 1170, 780, 490 (two:
    // between).
    struct Cost {
        ShapeId id;
        int b, at_once;
        double step, alone, ends;
    };
    static const Cost one[4] = {{kBig, 256, 1, 1.5, 1.35, 4.5}, {kSq, 128, 2, 0.58, 0.66, 3.0},
                                {kSmall, 64, 4, 0.21, 0.52, 2.0}, {kTiny, 32, 8, 0.125, 0.23, 2.2}};
    static const Cost two[4] = {{kBig, 256, 1, 3.0, 2.7, 5.0}, {kSq, 128, 2, 0.94, 1.08, 3.0},
                                {kSmall, 64, 3, 0.37, 0.62, 2.5}, {kTiny, 32, 5, 0.19, 0.29, 2.2}};
    static const Cost three[4] = {{kBig, 256, 1, 4.5, 4.1, 5.0}, {kSq, 128, 2, 1.33, 1.50, 3.0},
                                  {kSmall, 64, 2, 0.53, 0.68, 2.5}, {kTiny, 32, 4, 0.25, 0.34, 2.2}};
    const long long steps = (K + kBK - 1) / kBK, most = may_split ? (steps < 256 ? steps : 256) : 1;
    Cut best{kSq, 1};
    double least = 1e300;
    for (int c = 0; c < 4; ++c) {
        const Cost& q = pairs == 1 ? one[c] : pairs == 2 ? two[c] : three[c];
        const long long t = tiles(q.b);
        for (long long s = 1; s <= most; s += s < 16 ? 1 : s / 8) {
            const double per = (double)((steps + s - 1) / s);
            const long long n = (t * s + cus - 1) / cus, full = n / q.at_once, rest = n % q.at_once;
            auto round = [&](long long k) {
                const double shared = (strided && q.id == kTiny ? 1.25 * q.step : q.step) * (double)k;
                return (shared > q.alone ? shared : q.alone) * per + q.ends;
            };
            // a split sum is written and read once more, 4 bytes an element at 4 TB/s, and takes one more launch
            const double time = (double)full * round(q.at_once) + (rest ? round(rest) : 0.0) +
                                (s > 1 ? 4.0 + 8e-6 * (double)s * area / 4.0 : 0.0);
            if (time < least) {
                least = time;
                best = Cut{q.id, (int)s};
            }
        }
    }
    return best;
}

}  // namespace ds
