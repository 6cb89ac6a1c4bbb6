// orth.hip — an update orthogonalised by Newton-Schulz products, for many matrices at once, and the optimiser step around it:
//     m <- mu m + g      U = g + mu m (nesterov) or m      X = U / (|U|_F + eps)
//     five times   X <- P(X X^T) X,  P(A) = a I + b A + c A^2          w <- w (1 - lr decay) - lr sqrt(max(1, rows / cols)) X
// with (a, b, c) the quintic whose iteration takes singular values of (0, 1] towards 1; a tall matrix is worked on transposed, so
// that A is the smaller (M x M) Gram matrix. The coefficients, the momentum rule and the scale of the update are those of the published
// Muon method (K. Jordan and others, 2024).
//
// Through the Gram matrix. Everything an iteration applies to X is a polynomial of A, and the next Gram matrix is P A P: up to three
// iterations run on M x M matrices alone (Q <- P Q collects what they apply, A <- P (P A)), then X <- Q X once. Five iterations in
// two runs (3 + 2) cost 6 M^2 N + 14 M^3 instead of the 15 M^2 N + 5 M^3 of forming X each time (all M x M results are symmetric:
// one triangle is computed): equal for square matrices, 2.5 times fewer operations for wide ones. But the Gram matrix holds squares, and
// what is rounded off beside the largest is amplified with the smallest: in fp32 all five in one run are up to 25 times further off than
// X formed each time, 3 + 2 up to three times for small square matrices and twice for wide ones. Runs of three are for matrices that
// are wide enough to gain by them (run_of).
//
// Precision. One product in bf16 per step leaves the result 1e-2 off on well conditioned gradients and 3e-1 on those with a few
// strong directions: what is lost next to the large singular values is amplified by a^5 = 485 where they are small. The operands
// are therefore kept as TWO fp16 planes each, v = hi + lo with hi = fp16(v), lo = fp16(v - hi): 22 bits and lo's sign for fp32's
// 24. A product is three MFMAs (hi hi, hi lo, lo hi; lo lo lies below the planes' own rounding), accumulated in fp32. The planes are
// scaled by powers of two so that entries far below 1 keep their low bits above fp16's subnormal step. Off the 64-bit result, beside
// the same five iterations in fp32 (gradients with four strong directions): 63 x 124 1.2e-6 and 1.4e-6, 128 x 128 0.7e-6 and 1.4e-6,
// 372 x 372 0.9e-6 and 2.0e-6, 4096 x 4096 3.3e-6 and 4.8e-6; in runs of three 248 x 1780 2.7e-6 and 2.1e-6, 1095 x 465 2.6e-6 and 2.9e-6,
// 1024 x 18432 1.4e-6 and 4.1e-6. Matrices of 16 to 32 with strong directions alone 3.5e-6 and 2.6e-6.
//
// All matrices of a call share each launch (a task list by value, no device tables): the products of one dependency level, of matrices
// with short and with long runs alike. Planes are padded to whole tiles with zeros, which stay zeros, so that the K loops have no
// bounds.
#include "common.h"
#include "../../include/cpcsv_hip.h"
#include <algorithm>
#include <climits>

namespace {
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
// Entries are bounded by spectral norms: |X| < 1.21, |A| and |P A| < 1.45, |P| < 3.45, |Q| < 3.45^k behind k iterations. The scaled
// values stay below fp16's 65504.
constexpr float SX = 16384.f, SA = 16384.f, SP = 8192.f;
constexpr float SQ[4] = {0.f, SP, 4096.f, 1024.f};
constexpr int RUN = 3;                         // most iterations between two X
constexpr int PAD = 128, MAXJ = CPCSV_ORTH_JOBS, MAXT = 2 * MAXJ, NORMB = 1024;      // NORMB: most blocks of a matrix' norm

struct Job {
    const void* g; float* m; void* out;       // gradient, momentum (NULL: none), weight or result
    long x, xt;                               // offsets in halves
    int rows, cols;                           // of the matrix
    int M, N, tall;                           // padded min / max side; tall: rows > cols
    int run;                                  // iterations between two X
    int t_norm, t_split;                      // first block of the job
};
struct Jobs {
    Job j[MAXJ];
    int n, dtype, nesterov;
    float mu, eps;
    double* part;
    _Float16* ws;
};

// all first blocks compared at once (a search is a chain of loads that wait half a microsecond each)
template <int Job::*FIRST> __device__ __forceinline__ int job_of(const Jobs& s) {
    static_assert(MAXJ == 16, "a quarter of the wavefront");
    const int l = threadIdx.x & 15, first = s.j[l].*FIRST;                   // (behind the last job: 0)
    return __popc((uint32_t)__ballot((int)blockIdx.x >= first && (first || !l)) & 0xffff) - 1;
}
__device__ __forceinline__ float ld_g(const void* p, int dtype, long i) {
    return dtype == CPCSV_F32 ? ((const float*)p)[i] : bf16_to_f32(((const bf16_t*)p)[i]);
}
__device__ __forceinline__ uint32_t split_of(float v) {           // hi | lo << 16
    union { _Float16 h[2]; uint32_t w; } p;
    p.h[0] = (_Float16)v;
    p.h[1] = (_Float16)(v - (float)p.h[0]);
    return p.w;
}
// An operand [rows][K] holds, of each row, 32 values' hi halves and then their lo halves, 128 bytes: a slice of 32 K is a cache line
// (planes apart, a product of 128 x 128 tiles asked for half lines and was bound by them: 64-byte rows 0.65 us for 32 KB a CU, 128-byte
// rows 0.43). Offset of (r, k)'s hi half; lo is 32 further.
__device__ __forceinline__ long at_of(long r, int k, int K) { return r * 2 * K + (k >> 5) * 64 + (k & 31); }
__device__ __forceinline__ void planes_of(const uint32_t* w, half8& hi, half8& lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        union { uint32_t w; _Float16 h[2]; } p;
        p.w = w[e];
        hi[e] = p.h[0]; lo[e] = p.h[1];
    }
}
__host__ __device__ inline int norm_blocks(int rows, int cols) {
    const long n = ((long)rows * cols + 4095) / 4096;
    return n < NORMB ? (int)n : NORMB;
}

// ---- momentum and |U|^2 (double: squares of any fp32 value) ----------------------------------------------------------
// Bound by HBM: 54 us for 25 M values (12 bytes each).
__global__ __launch_bounds__(256) void orth_norm_kernel(Jobs s) {
    const int k = job_of<&Job::t_norm>(s);
    const Job& j = s.j[k];
    const int blk = blockIdx.x - j.t_norm, nb = norm_blocks(j.rows, j.cols);
    const long n = (long)j.rows * j.cols;
    double q = 0.0;
    auto one = [&](float u, float& m) {
        if (j.m) {
            m = __fmaf_rn(s.mu, m, u);
            u = s.nesterov ? __fmaf_rn(s.mu, m, u) : m;
        }
        q += (double)u * (double)u;
    };
    const long step = (long)nb * 256, id = (long)blk * 256 + threadIdx.x;
    long i = id;
    if (((uintptr_t)j.g & 15) == 0 && ((uintptr_t)j.m & 15) == 0 && s.dtype == CPCSV_F32) {          // sixteen values a thread and turn
        const f32x4* g4 = (const f32x4*)j.g;
        f32x4* m4 = (f32x4*)j.m;
        long v = id;
        for (; v + 3 * step < n / 4; v += 4 * step) {
            f32x4 u[4], m[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u[k] = g4[v + k * step];
                if (j.m) m[k] = m4[v + k * step];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { float x = m[k][e]; one(u[k][e], x); m[k][e] = x; }
                if (j.m) m4[v + k * step] = m[k];
            }
        }
        for (; v < n / 4; v += step) {
            const f32x4 u = g4[v];
            f32x4 m = u;
            if (j.m) m = m4[v];
#pragma unroll
            for (int e = 0; e < 4; ++e) { float x = m[e]; one(u[e], x); m[e] = x; }
            if (j.m) m4[v] = m;
        }
        i = n / 4 * 4 + id;
    }
    for (; i < n; i += step) {
        float m = j.m ? j.m[i] : 0.f;
        one(ld_g(j.g, s.dtype, i), m);
        if (j.m) j.m[i] = m;
    }
    __shared__ double sh[256];
    sh[threadIdx.x] = q;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) s.part[k * NORMB + blk] = sh[0];
}

// ---- X_0 in both orientations, split, 64 x 64 tiles of the padded matrix ---------------------------------------------
// Bound by HBM: 81 us for 25 M values with momentum, 5.0 TB/s (every load is in flight before the norm's parts are added up).
__global__ __launch_bounds__(256) void orth_split_kernel(Jobs s) {
    __shared__ uint32_t t[64][65];
    __shared__ double sh[256];
    const int k = job_of<&Job::t_split>(s);
    const Job& j = s.j[k];
    const int PR = j.tall ? j.N : j.M, PC = j.tall ? j.M : j.N, tile = blockIdx.x - j.t_split;
    const int r0 = tile / (PC / 64) * 64, c0 = tile % (PC / 64) * 64;
    const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6, c = c0 + cl;
    float u[16], m[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + i * 4 + rl;
        const bool in = r < j.rows && c < j.cols;
        const long at = in ? (long)r * j.cols + c : 0;
        u[i] = in ? ld_g(j.g, s.dtype, at) : 0.f;
        m[i] = in && j.m ? j.m[at] : 0.f;
    }
    double sum = 0.0;
    for (int i = threadIdx.x; i < norm_blocks(j.rows, j.cols); i += 256) sum += s.part[k * NORMB + i];
    sh[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    // u SX / (|U| + eps), the factor as a power of two and the rest: by itself it leaves fp32's range where |U| is tiny (eps 0). Zeros
    // stay zeros whatever eps is.
    const double norm = sqrt(sh[0]) + (double)s.eps;
    int pow2 = 0;
    const float rest = norm > 0.0 ? (float)frexp((double)SX / norm, &pow2) : norm == 0.0 ? 0.f : (float)norm;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float v = !j.m ? u[i] : s.nesterov ? __fmaf_rn(s.mu, m[i], u[i]) : m[i];
        const bool in = r0 + i * 4 + rl < j.rows && c < j.cols;
        t[i * 4 + rl][cl] = split_of(in ? ldexpf(v, pow2) * rest : 0.f);
    }
    __syncthreads();
    _Float16 *own = s.ws + (j.tall ? j.xt : j.x), *turned = s.ws + (j.tall ? j.x : j.xt);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int line = i * 32 + (threadIdx.x >> 3), q = (threadIdx.x & 7) * 8;
#pragma unroll
        for (int way = 0; way < 2; ++way) {
            uint32_t w[8];
            half8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = way ? t[q + e][line] : t[line][q + e];
            planes_of(w, hi, lo);
            _Float16* d = way ? turned + at_of(c0 + line, r0 + q, PR) : own + at_of(r0 + line, c0 + q, PC);
            *(half8*)d = hi;
            *(half8*)(d + 32) = lo;
        }
    }
}

// ---- the products: D = alpha P Q^T + beta E + gamma I over two-plane operands [rows][K] ------------------------------
// D symmetric, lower triangle and its mirror image (SYMM_E: with E and I) | D and its transpose | the result | the weight. A launch has
// one kind and its own kernel: straight-line code for all of them was 68 KB, and what a block runs once comes cold from memory
// (MIXED: products of the first and the third kind, where jobs of short and of long runs share a call)
enum { SYMM, SYMM_E, BOTH, OUT, WEIGHT, MIXED };
__host__ __device__ constexpr bool symmetric(int kind) { return kind == SYMM || kind == SYMM_E; }
struct Task {
    long p, q, e, d, dt;       // offsets in halves; OUT, WEIGHT: d is the output's address
    long slab;                 // first partial tile, in floats
    int R, C, K;
    float alpha, beta, gamma;
    int shape, t0, tiles, whole, S, r0; // tile shape; first block; tiles, of which `whole` in one piece, the others in S slices of K; first joining block
    int steps, longer;         // K steps of a slice; slices that have one more
    int rows, cols, tall;                     // OUT, WEIGHT: of the output
    int symm;
};
constexpr bool result(int kind) { return kind == OUT || kind == WEIGHT; }
template <int KIND> __device__ __forceinline__ bool symm_of(const Task& t) { return KIND == MIXED ? t.symm != 0 : symmetric(KIND); }
struct Launch {
    int first[MAXT];           // block of each task (behind the last: none's)
    Task t[MAXT];
    int n, kind, dtype;
    float decay;
    const float* hyper;
    _Float16* ws;
    float* slabs;
};

// Tiles. A wavefront's share of a tile sets what it reads from LDS for each MFMA, and LDS bandwidth is what bounds the main loop of
// large products: 256 x 256 with 128 x 64 a wavefront runs 1245 TFLOP/s (three MFMAs a product counted) on 4096^3 against 860 for
// 128 x 128 with 64 x 64, which packs two blocks on a CU and fills the chip at half the tiles (1024 x 18432 x 1024: 962 against 757).
// Small products are bound by the latency of their K steps and of what stands before and behind them: 64 x 64 tiles, whose single
// block a wavefront keeps two accumulators (a chain of dependent MFMAs half as long) and has its entries of E loaded beforehand
// (512^3, all three with a loop of two stages: 6.7 us for the bare product against 13.3 and 34). A level of 384 x 384 results takes
// 8.5 us, of 1024 x 1024 12.7 us; of that the block's own time is 5 and 9.5 us, the rest is the launch.
template <int BM_, int WM_, int WN_, int RING_> struct Cfg {
    static constexpr int BM = BM_, WM = WM_, WN = WN_, BK = 32, RING = RING_, WC = BM / WN, NW = (BM / WM) * WC, T = NW * 64;
    static constexpr int CPR = BK / 4;                            // 16-byte chunks of a row's slice, both halves
    static constexpr int LD = BM * CPR / T;                       // loads a thread, operand and stage
    static constexpr int STAGE = 4 * BM * BK;                     // halves
    static constexpr int SW = WN < 64 ? WN : 64, NB = SW / 32;    // columns of an epilogue strip, their 32 x 32 blocks
    static constexpr int STRIP = 32 * (SW + 1);                   // words of a strip in LDS
    static constexpr int LDS = RING * STAGE * 2;
    static constexpr int MA = WM / 32, MB = WN / 32, STRIPS = MA * MB / NB;
    // chunk (16 bytes) q of LDS row r lives in slot q ^ swz(r): the rows a fragment read touches together fall into all banks. The
    // DMA writes LDS in lane order, so the permutation is on the source side.
    static __device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }
};
using Big = Cfg<256, 128, 64, 2>;
using Mid = Cfg<128, 64, 64, 2>;
using Small = Cfg<64, 32, 32, 4>;
static_assert(Big::LDS >= Big::NW * Big::STRIP * 4 && Mid::LDS >= Mid::NW * Mid::STRIP * 4 && Small::LDS >= Small::NW * Small::STRIP * 4, "strips fit");

// of place w in a lower triangle taken row by row (w < 2^20)
__device__ __forceinline__ unsigned triangle_row(unsigned w) {
    unsigned r = (unsigned)((__builtin_amdgcn_sqrtf(8.f * (float)w + 1.f) - 1.f) * 0.5f);
    r -= r * (r + 1) / 2 > w;
    r += (r + 1) * (r + 2) / 2 <= w;
    return __builtin_amdgcn_readfirstlane(r);
}
template <int KIND> __device__ __forceinline__ void tile_of(const Task& t, unsigned tile, unsigned bm, int& ti, int& tj) {
    const unsigned tm = (t.R + bm - 1) / bm;
    if (symm_of<KIND>(t)) {
        // lower triangle by blocks of g x g tiles, a row of blocks behind the other (the last one of h tile rows; on the diagonal
        // triangles): a run of tiles shares operand rows in L2. Row by row, every XCD read the whole operand.
        const unsigned lg = tm >= 24 ? 3 : 2, g = 1u << lg;
        const unsigned I = triangle_row(tile) >> lg;           // (the tiles above a row of blocks are as many as row by row)
        const unsigned rem = tile - I * g * (I * g + 1) / 2, h = min(g, tm - I * g);
        const unsigned J = min(h == g ? rem >> 2 * lg : rem / (g * h), I), w = rem - J * g * h;
        const unsigned r = J < I ? w >> lg : triangle_row(w);
        ti = I * g + r;
        tj = J * g + w - (J < I ? r * g : r * (r + 1) / 2);
    } else {                                     // bands of 8 tile rows, so that a run of tiles shares operand rows in L2
        const unsigned tn = (t.C + bm - 1) / bm, g = tile / (8 * tn), gr = min(8u, tm - g * 8), w = tile - g * 8 * tn;
        const unsigned q = gr == 8 ? w >> 3 : w / gr;
        ti = g * 8 + w - q * gr;
        tj = q;
    }
}

template <int I> struct Const { static constexpr int value = I; };
template <int N, typename F> __device__ __forceinline__ void static_for(F&& f) {
    if constexpr (N > 0) {
        static_for<N - 1>(f);
        f(Const<N - 1>{});
    }
}

// E (symmetric, bit for bit) in rows r..r + 3 of column c, r a multiple of 4: read along row c, hi and lo
struct Quad { half4 hi, lo; };
__device__ __forceinline__ Quad quad_of(const Launch& s, const Task& t, int r, int c) {
    const _Float16* o = s.ws + t.e + at_of(c, r, t.C);
    return Quad{*(const half4*)o, *(const half4*)(o + 32)};
}

// One wavefront's strip, 32 rows x SW columns from (r0, c0), -> D. A lane's 16 values of a 32 x 32 block: column lane % 32, rows
// 8 (i / 4) + 4 (lane / 32) + i % 4; they pass through the wavefront's own piece of LDS (to_lds) to leave as 16-byte pieces of rows in
// either orientation (leave).
template <typename C, int KIND, bool EARLY>
__device__ __forceinline__ void to_lds(const Launch& s, const Task& t, int r0, int c0, const f32x16 (&acc)[C::NB], uint32_t* buf, const Quad (&early)[4]) {
    const int lane = threadIdx.x & 63, fr = lane & 31, fk = lane >> 5;
#pragma unroll
    for (int b = 0; b < C::NB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int rl = g * 8 + fk * 4, cl = b * 32 + fr, r = r0 + rl, c = c0 + cl;
            Quad q{};
            if (KIND == SYMM_E) q = EARLY ? early[g] : quad_of(s, t, r, c);      // (early: one block a strip)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = acc[b][g * 4 + j] * t.alpha;
                if (KIND == SYMM_E) v += ((float)q.hi[j] + (float)q.lo[j]) * t.beta + (r + j == c ? t.gamma : 0.f);
                buf[(rl + j) * (C::SW + 1) + cl] = result(KIND) ? __float_as_uint(v) : split_of(v);
            }
        }
}

// a 32 x 32 block of the strip as rows of D from (r0, c0): itself, its transpose, or (on the diagonal) its lower triangle mirrored
enum { SELF, TURNED, MIRRORED };
template <typename C, int HOW> __device__ __forceinline__ void block_out(const uint32_t* z, _Float16* d, int r0, int c0, int K) {
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < 2; ++i) {
        const int line = i * 16 + lane / 4, q = lane % 4 * 8;
        uint32_t w[8];
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            w[e] = HOW == TURNED || (HOW == MIRRORED && line < q + e) ? z[(q + e) * (C::SW + 1) + line] : z[line * (C::SW + 1) + q + e];
        planes_of(w, hi, lo);
        _Float16* o = d + at_of(r0 + line, c0 + q, K);
        *(half8*)o = hi;
        *(half8*)(o + 32) = lo;
    }
}

template <typename C, int KIND>
__device__ __forceinline__ void leave(const Launch& s, const Task& t, int r0, int c0, const uint32_t* buf) {
    constexpr int SW = C::SW, LDW = SW + 1, NB = C::NB;
    const int lane = threadIdx.x & 63;
    if (result(KIND)) {
        // rows of the output run along the strip's columns, of a tall one's along its rows; GO rows at a time are read before they are
        // written (the weight's: one after the other they cost a memory latency each)
        constexpr int GO = 16;
        const int len = t.tall ? 32 : SW, per = 64 / len, sub = lane % len, R0 = (t.tall ? c0 : r0) + lane / len, Cc = (t.tall ? r0 : c0) + sub;
        const int sl = t.tall ? sub * LDW + lane / len : lane / len * LDW + sub, dl = t.tall ? per : per * LDW;
        const long at0 = (long)R0 * t.cols + Cc, step = (long)per * t.cols;
        const float lr = KIND == WEIGHT ? s.hyper[0] : 0.f;
        const float keep = 1.f - lr * s.decay, by = lr * sqrtf(fmaxf(1.f, (float)t.rows / (float)t.cols));
        const int n = Cc < t.cols && R0 < t.rows ? min(SW / 2, (t.rows - R0 + per - 1) / per) : 0;
        typedef __attribute__((address_space(1))) float gf;
        typedef __attribute__((address_space(1))) bf16_t gb;
        for (int i0 = 0; i0 < n; i0 += GO) {
            float old[GO];
            if (KIND == WEIGHT)
#pragma unroll
                for (int i = 0; i < GO; ++i) old[i] = ((gf*)t.d)[at0 + step * min(i0 + i, n - 1)];
#pragma unroll
            for (int i = 0; i < GO; ++i) {
                if (i0 + i >= n) continue;
                const float v = __uint_as_float(buf[sl + dl * (i0 + i)]);
                const long at = at0 + step * (i0 + i);
                if (KIND == WEIGHT) ((gf*)t.d)[at] = old[i] * keep - by * v;
                else if (s.dtype == CPCSV_F32) ((gf*)t.d)[at] = v;
                else ((gb*)t.d)[at] = f32_to_bf16(v);
            }
        }
        return;
    }
    _Float16 *const d = s.ws + t.d, *const turned = s.ws + (symm_of<KIND>(t) ? t.d : t.dt);             // (D^T [C][R])
    for (int b = 0; b < NB; ++b) {
        const int cb = c0 + b * 32;
        if (symm_of<KIND>(t) && cb > r0) continue;             // (above the diagonal)
        if (symm_of<KIND>(t) && cb == r0) {
            // on it: each pair of entries is taken from the lower one (the two sums are the same numbers in another order)
            block_out<C, MIRRORED>(buf + b * 32, d, r0, cb, t.C);
            continue;
        }
        block_out<C, SELF>(buf + b * 32, d, r0, cb, t.C);
        block_out<C, TURNED>(buf + b * 32, turned, cb, r0, t.R);
    }
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// (sides are multiples of a strip's)
template <int KIND> __device__ __forceinline__ bool outside(const Task& t, int r0, int c0) { return r0 >= t.R || c0 >= t.C || (symm_of<KIND>(t) && r0 + 31 < c0); }

// all but the N youngest loads have landed, the wavefront's LDS reads are done
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// The block's task (all first blocks compared at once). task_of: every lane holds one, so that finding it and reading it is one latency
// of the arguments' memory, half a microsecond; the larger tiles have no registers for that.
__device__ __forceinline__ int task_at(const Launch& s) {
    static_assert(MAXT == 32 && sizeof(Task) % 4 == 0 && sizeof(Launch) <= 4096, "a half of the wavefront; a kernel's arguments");
    return __popc((uint32_t)__ballot((int)blockIdx.x >= s.first[threadIdx.x & 31])) - 1;
}
__device__ __forceinline__ Task task_of(const Launch& s) {
    union { Task t; int w[sizeof(Task) / 4]; } mine, own;
    mine.t = s.t[threadIdx.x & 31];
    const int k = task_at(s);
#pragma unroll
    for (int i = 0; i < (int)sizeof(Task) / 4; ++i) own.w[i] = __builtin_amdgcn_readlane(mine.w[i], k);
    return own.t;
}

template <typename C, int KIND>
__device__ __forceinline__ void product(const Launch& s, const Task& t, unsigned char* smem) {
    _Float16* const lds = (_Float16*)smem;
    // the whole tiles first, then the others, slice by slice. Blocks go to the eight XCDs in turn: each gets a contiguous run of
    // either part, whose operands its L2 then holds, and a share of both
    const bool sliced = (int)blockIdx.x - t.t0 >= t.whole;
    const int from = t.t0 + (sliced ? t.whole : 0), cut = t.tiles - t.whole, n = sliced ? cut * t.S : t.whole, xcd = blockIdx.x & 7;
    auto more = [&](int v) { return (v >> 3) * (n & 7) + min(v & 7, n & 7); };        // of v XCDs, those that have a block more
    const int u = ((blockIdx.x - from) >> 3) + xcd * (n >> 3) + more((-from & 7) + xcd) - more(-from & 7);
    const int S = sliced ? t.S : 1, sl = sliced ? (unsigned)u / (unsigned)cut : 0, tile = sliced ? t.whole + u - sl * cut : u;
    int ti, tj;
    tile_of<KIND>(t, tile, C::BM, ti, tj);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), K = t.K;
    const int k0 = sliced ? sl * t.steps + min(sl, t.longer) : 0, k1 = sliced ? k0 + t.steps + (sl < t.longer) : K / C::BK;
    const _Float16* src[2] = {s.ws + t.p + (long)ti * C::BM * 2 * K, s.ws + t.q + (long)tj * C::BM * 2 * K};
    uint32_t off[2][C::LD];                      // in bytes (K <= 131072 and 256 rows: below 2^28)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int i = 0; i < C::LD; ++i) {
            const int idx = i * C::T + tid, row = idx / C::CPR, q = (idx % C::CPR) ^ C::swz(row);
            const int last = (o ? t.C - tj * C::BM : t.R - ti * C::BM) - 1;               // a tile may hang over the padded side
            off[o][i] = (uint32_t)(min(row, last) * 2 * K + q * 8) * 2;
        }
    auto load = [&](int buf, int kt, int o, int i) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)(src[o] + (long)kt * 2 * C::BK) + off[o][i]),
                                         (__attribute__((address_space(3))) void*)(lds + buf * C::STAGE + o * C::BM * 2 * C::BK +
                                                                                   (i * C::T + wave * 64) * 8), 16, 0, 0);
    };
    auto stage = [&](int buf, int kt) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < C::LD; ++i) load(buf, kt, o, i);
    };
    const int wm = wave / C::WC * C::WM, wn = wave % C::WC * C::WN, fr = lane & 31, fk = lane >> 5;
    f32x16 acc[C::MA][C::MB], low;               // low: the hi lo terms of a one-block wavefront
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        low[e] = 0.f;
#pragma unroll
        for (int a = 0; a < C::MA; ++a)
#pragma unroll
            for (int b = 0; b < C::MB; ++b) acc[a][b][e] = 0.f;
    }
    stage(0, k0);
    constexpr bool ONE = C::MA * C::MB == 1;
    Quad early[4] = {};
    if constexpr (ONE) {
        // One wavefront a SIMD: what bounds a step is what it has to issue. Unrolled over the ring, so that LDS addresses are constants;
        // all fragments first, the loads between the MFMAs; the RING - 1 stages in flight are behind a barrier of its own (one with
        // the compiler's fence would wait for them). 475 cycles a step, 384 of them LDS traffic, 550 where half the CUs are at work (16 KB
        // a step arrive at 30 bytes a cycle and CU); 725 with two stages and a loop.
        constexpr int KK = C::BK / 16, EACH = 2 * C::LD / KK, AHEAD = C::RING - 1;
#pragma unroll
        for (int i = 1; i < AHEAD; ++i) stage(i, k0 + i);                     // (a slice has RING K steps at least)
        if (KIND == SYMM_E && S == 1) {              // behind the stages: scattered over 32 rows, they come late
            const int r0 = ti * C::BM + wm, c0 = tj * C::BM + wn;
            if (r0 < t.R && c0 < t.C)
#pragma unroll
                for (int g = 0; g < 4; ++g) early[g] = quad_of(s, t, r0 + g * 8 + fk * 4, c0 + fr);
        }
        const _Float16 *fp0 = lds + (wm + fr) * 2 * C::BK, *fq0 = lds + (C::BM + wn + fr) * 2 * C::BK;
        auto step = [&](const _Float16* p0, const _Float16* q0, auto&& between) {
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            half8 fp[KK][2], fq[KK][2];
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int at = ((kk * 2 + p * 4 + fk) ^ C::swz(fr)) * 8;
                    fp[kk][p] = *(const half8*)(p0 + at);
                    fq[kk][p] = *(const half8*)(q0 + at);
                }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                between(kk);
                low = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk][0], fq[kk][1], low, 0, 0, 0);
                acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk][0], fq[kk][0], acc[0][0], 0, 0, 0);
                low = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[kk][1], fq[kk][0], low, 0, 0, 0);
            }
        };
        int kt = k0;
        bool on = true;
        do
            static_for<C::RING>([&](auto u) {
                if (!on) return;
                wait_loads<(AHEAD - 1) * 2 * C::LD>();
                step(fp0 + u.value * C::STAGE, fq0 + u.value * C::STAGE, [&](int kk) {
#pragma unroll
                    for (int e = 0; e < EACH; ++e) load((u.value + AHEAD) % C::RING, kt + AHEAD, (kk * EACH + e) / C::LD, (kk * EACH + e) % C::LD);
                });
                on = ++kt + AHEAD < k1;
            });
        while (on);
        static_for<AHEAD>([&](auto u) {
            wait_loads<(AHEAD - 1 - u.value) * 2 * C::LD>();
            const int buf = (kt + u.value - k0) % C::RING * C::STAGE;
            step(fp0 + buf, fq0 + buf, [](int) {});
        });
    } else
    for (int kt = k0; kt < k1; ++kt) {
        const int buf = (kt - k0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const _Float16* base = lds + buf * C::STAGE;
        auto frag = [&](int side, int row, int kk, int p) {
            return *(const half8*)(base + (side * C::BM + row) * 2 * C::BK + ((kk * 2 + p * 4 + fk) ^ C::swz(row)) * 8);
        };
        if (kt + 1 < k1) stage(buf ^ 1, kt + 1);
#pragma unroll
        for (int kk = 0; kk < C::BK / 16; ++kk) {
            half8 fp[2][C::MA], fq[2][C::MB];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int a = 0; a < C::MA; ++a) fp[p][a] = frag(0, wm + a * 32 + fr, kk, p);
#pragma unroll
                for (int b = 0; b < C::MB; ++b) fq[p][b] = frag(1, wn + b * 32 + fr, kk, p);
            }
#define FOR_ACC for (int a = 0; a < C::MA; ++a) _Pragma("unroll") for (int b = 0; b < C::MB; ++b)
#pragma unroll
            FOR_ACC acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][a], fq[1][b], acc[a][b], 0, 0, 0);
#pragma unroll
            FOR_ACC acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[1][a], fq[0][b], acc[a][b], 0, 0, 0);
#pragma unroll
            FOR_ACC acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][a], fq[0][b], acc[a][b], 0, 0, 0);
        }
    }
    __syncthreads();
    if (ONE) acc[0][0] += low;
    if (S > 1) {                                 // a slice's share of the tile, strip by strip in the order the registers hold it
        f32x4* d = (f32x4*)(s.slabs + t.slab) + ((long)(tile - t.whole) * S + sl) * (C::BM * C::BM / 4) + (long)wave * C::STRIPS * C::NB * 256 + lane;
#pragma unroll
        for (int a = 0; a < C::MA; ++a)
#pragma unroll
            for (int b = 0; b < C::MB; ++b)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    f32x4 v = {acc[a][b][h * 4], acc[a][b][h * 4 + 1], acc[a][b][h * 4 + 2], acc[a][b][h * 4 + 3]};
                    d[((a * C::MB + b) * 4 + h) * 64] = v;
                }
        return;
    }
    uint32_t* const buf = (uint32_t*)smem + wave * C::STRIP;
    for (int strip = 0; strip < C::STRIPS; ++strip) {
        const int r0 = ti * C::BM + wm + strip / (C::MB / C::NB) * 32, c0 = tj * C::BM + wn + strip % (C::MB / C::NB) * C::NB * 32;
        if (outside<KIND>(t, r0, c0)) continue;
        static_for<C::STRIPS>([&](auto i) {      // (registers need constant indices)
            if (i.value != strip) return;
            constexpr int a = decltype(i)::value / (C::MB / C::NB), b = decltype(i)::value % (C::MB / C::NB) * C::NB;
            f32x16 part[C::NB];
#pragma unroll
            for (int n = 0; n < C::NB; ++n) part[n] = acc[a][b + n];
            to_lds<C, KIND, ONE>(s, t, r0, c0, part, buf, early);
        });
        wave_sync();
        leave<C, KIND>(s, t, r0, c0, buf);
        wave_sync();
    }
}

// one launch serves the two shapes of 256 threads and 64 KB of LDS
template <int KIND>
__global__ __launch_bounds__(Mid::T, 2) void orth_gemm_kernel(Launch s) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    const Task t = task_of(s);
    if (t.shape == 1) product<Mid, KIND>(s, s.t[task_at(s)], smem);
    else product<Small, KIND>(s, t, smem);
}
template <int KIND>
__global__ __launch_bounds__(Big::T) void orth_gemm_big_kernel(Launch s) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    product<Big, KIND>(s, s.t[task_at(s)], smem);
}

// the slices of a tile, added in order: one wavefront a strip
template <typename C, int KIND> __device__ __forceinline__ void join(const Launch& s, const Task& t, uint32_t* buf) {
    const int id = blockIdx.x - t.r0, strip = id % (C::NW * C::STRIPS), cut = id / (C::NW * C::STRIPS), wave = strip / C::STRIPS;
    const int a = strip % C::STRIPS / (C::MB / C::NB), b = strip % (C::MB / C::NB) * C::NB;
    int ti, tj;
    tile_of<KIND>(t, t.whole + cut, C::BM, ti, tj);
    const int r0 = ti * C::BM + wave / C::WC * C::WM + a * 32, c0 = tj * C::BM + wave % C::WC * C::WN + b * 32;
    if (outside<KIND>(t, r0, c0)) return;
    const f32x4* d = (const f32x4*)(s.slabs + t.slab) + (long)cut * t.S * (C::BM * C::BM / 4) + (long)strip * C::NB * 256 + threadIdx.x;
    f32x16 acc[C::NB];
#pragma unroll
    for (int n = 0; n < C::NB; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[n][e] = 0.f;
#pragma unroll 4
    for (int sl = 0; sl < t.S; ++sl)
#pragma unroll
        for (int n = 0; n < C::NB; ++n)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const f32x4 v = d[(long)sl * (C::BM * C::BM / 4) + (n * 4 + h) * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[n][h * 4 + e] += v[e];
            }
    const Quad none[4] = {};
    to_lds<C, KIND, false>(s, t, r0, c0, acc, buf, none);
    wave_sync();
    leave<C, KIND>(s, t, r0, c0, buf);
}
template <int KIND>
__global__ __launch_bounds__(64) void orth_join_kernel(Launch s) {
    __shared__ uint32_t buf[Mid::STRIP];
    const Task t = task_of(s);
    if (t.shape == 0) join<Big, KIND>(s, t, buf);
    else if (t.shape == 1) join<Mid, KIND>(s, t, buf);
    else join<Small, KIND>(s, t, buf);
}
static_assert(Mid::T == Small::T && Mid::LDS == Small::LDS && Mid::STRIP >= Small::STRIP && Mid::STRIP >= Big::STRIP, "shared launches");

// ---- host: the schedule ---------------------------------------------------------------------------------------------
long tiles_of(int kind, long R, long C, int bm) {
    const long tm = (R + bm - 1) / bm, tn = (C + bm - 1) / bm;
    return symmetric(kind) ? tm * (tm + 1) / 2 : tm * tn;
}
// How a product is cut: the tile, and how many slices of K the tiles get that do not fill the last round of blocks over the 256 CUs
// (all of them, where there are few: 1024 x 18432 against itself has 36 of 128 x 128 and took 470 us in one piece). By the
// product's sides alone, so that a matrix has the same bits in any company. Least time by what a K step was measured to take (us;
// `two`: while two blocks share the CU) and a block's fixed part; a join reads and writes its slabs once.
struct Shape { int bm, bk, fit, strips; double one, two, fixed; };
constexpr Shape SHAPES[3] = {{256, 32, 1, Big::NW * Big::STRIPS, 2.5, 2.5, 30.0}, {128, 32, 2, Mid::NW * Mid::STRIPS, 0.9, 1.6, 10.0},
                             {64, 32, 2, Small::NW * Small::STRIPS, 0.285, 0.57, 7.0}};
struct Cut { int shape, whole, S; long slab; };               // slab: floats
Cut cut_of(int kind, long R, long C, long K) {
    Cut best{0, 0, 1, 0};
    double least = 1e30;
    for (int c = 0; c < 3; ++c) {
        const Shape& h = SHAPES[c];
        const long n = tiles_of(kind, R, C, h.bm), slots = 256L * h.fit, nk = K / h.bk, whole = n / slots * slots, rest = n - whole;
        const double base = (double)(whole / slots) * (nk * h.two + h.fixed);
        for (int S = 1; S <= 128 && (S == 1 || (rest && K / S >= 256 && rest * S <= slots)); ++S) {
            double us = base;
            if (rest) us += (double)((nk + S - 1) / S) * (rest * S <= 256 ? h.one : h.two) + h.fixed;
            if (S > 1) us += 8.0 + 2.0 * rest * S * h.bm * h.bm * 4 / 4e6;
            if (us < least) {
                least = us;
                best = Cut{c, (int)(S > 1 ? whole : n), S, S > 1 ? rest * S * h.bm * h.bm : 0};
            }
        }
    }
    return best;
}

// Iterations between two X of a matrix, by its own (padded) sides: runs on the Gram matrix where they save work. At M x (M + 512) the
// two ways take the same time (1024 x 1536 213 us either way; runs of one and of three: 1024 x 1024 175 and 198, 1024 x 2048 241 and
// 225, 4096 x 4096 3825 and 4070, 128 x 512 99 and 106, 128 x 2048 118 and 112). Up to 16 rows or columns X is formed each time
// however long the other side is: a few strong directions are most of such a matrix, and runs of three lose in accuracy (16 x 2048 2.1
// times fp32's distance from the 64-bit result, against 1.4; 117 us against 112).
int run_of(const Job& j) { return j.N - j.M <= 512 || min(j.rows, j.cols) <= 16 ? 1 : RUN; }

struct Plan { long planes, slabs, bytes; int norm, split; };
struct Scratch { long a, p0, p1, r, q0, q1, xt1; };          // M x M matrices of a job and the second X^T

int plan(Jobs& s, Scratch* sc, const long* dims, int njobs, Plan& p) {
    if (njobs <= 0 || njobs > MAXJ || !dims) return -1001;
    long at = 0, slabs = 0;
    p = Plan{0, 0, 0, 0, 0};
    for (int i = 0; i < njobs; ++i) {
        const long r = dims[2 * i], c = dims[2 * i + 1];
        if (r <= 0 || c <= 0 || r > CPCSV_ORTH_MAX_SIDE || c > CPCSV_ORTH_MAX_SIDE || min(r, c) > CPCSV_ORTH_MAX_MIN) return -1002;
        Job& j = s.j[i];
        j.rows = (int)r; j.cols = (int)c; j.tall = r > c;
        j.M = (int)((j.tall ? c : r) + PAD - 1) / PAD * PAD;
        j.N = (int)((j.tall ? r : c) + PAD - 1) / PAD * PAD;
        j.run = run_of(j);
        const long mn = 2L * j.M * j.N, mm = 2L * j.M * j.M;
        j.x = at; j.xt = at + mn; sc[i].xt1 = at + 2 * mn;
        at += 3 * mn;
        long* const m6[6] = {&sc[i].a, &sc[i].p0, &sc[i].p1, &sc[i].r, &sc[i].q0, &sc[i].q1};
        for (int k = 0; k < (j.run == 1 ? 2 : 6); ++k) { *m6[k] = at; at += mm; }
        j.t_norm = p.norm; j.t_split = p.split;
        p.norm += norm_blocks(j.rows, j.cols);
        const long t64 = (long)(j.M / 64) * (j.N / 64);
        if (p.split + t64 > (1L << 30)) return -1002;
        p.split += (int)t64;
        // (a level holds one product of a job, two of its M x M ones)
        slabs += max(max(cut_of(SYMM, j.M, j.M, j.N).slab, 2 * cut_of(SYMM, j.M, j.M, j.M).slab), cut_of(BOTH, j.M, j.N, j.M).slab);
    }
    s.n = njobs;
    p.planes = at;
    p.slabs = slabs;
    p.bytes = (long)MAXJ * NORMB * 8 + at * 2 + slabs * 4;
    return 0;
}

template <int KIND> int fire(const Launch& big, const Launch& rest, const Launch& join, long ubig, long urest, long joins, hipStream_t st) {
    if (big.n) {                                                // more than the default cap of dynamic LDS: raise it once
        static const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(orth_gemm_big_kernel<KIND>), hipFuncAttributeMaxDynamicSharedMemorySize, Big::LDS);
        if (e != hipSuccess) return -(int)e;
        orth_gemm_big_kernel<KIND><<<(int)ubig, Big::T, Big::LDS, st>>>(big);
    }
    if (rest.n) orth_gemm_kernel<KIND><<<(int)urest, Mid::T, Mid::LDS, st>>>(rest);
    if (join.n) orth_join_kernel<KIND><<<(int)joins, 64, 0, st>>>(join);
    CPCSV_CHECK_LAUNCH();
    return 0;
}
// the products of one level: a launch for those of the big tile, one for the others, one that joins slices
int run_level(const Launch& all, long slabs, hipStream_t st) {
    Launch big = all, rest = all, join = all;
    big.n = rest.n = join.n = 0;
    for (Launch* l : {&big, &rest, &join}) std::fill(l->first, l->first + MAXT, INT_MAX);
    long at = 0, units[2] = {0, 0}, joins = 0;
    for (int i = 0; i < all.n; ++i) {
        Task t = all.t[i];
        const int kind = all.kind != MIXED ? all.kind : t.symm ? SYMM : BOTH;
        const Cut cut = cut_of(kind, t.R, t.C, t.K);
        t.shape = cut.shape;
        t.tiles = (int)tiles_of(kind, t.R, t.C, SHAPES[cut.shape].bm);
        t.whole = cut.whole; t.S = cut.S; t.slab = at;
        t.steps = t.K / SHAPES[cut.shape].bk / t.S; t.longer = t.K / SHAPES[cut.shape].bk % t.S;
        at += cut.slab;
        long& u = units[cut.shape != 0];
        t.t0 = (int)u; t.r0 = (int)joins;
        u += t.whole + (long)(t.tiles - t.whole) * t.S;
        if (t.S > 1) joins += (long)(t.tiles - t.whole) * SHAPES[cut.shape].strips;
        if (u > (1L << 30) || joins > (1L << 30)) return -1002;
        auto put = [&](Launch& l, int first) { l.first[l.n] = first; l.t[l.n++] = t; };
        put(cut.shape ? rest : big, t.t0);
        if (t.S > 1) put(join, t.r0);
    }
    if (at > slabs) return -1004;
    switch (all.kind) {
        case SYMM: return fire<SYMM>(big, rest, join, units[0], units[1], joins, st);
        case SYMM_E: return fire<SYMM_E>(big, rest, join, units[0], units[1], joins, st);
        case BOTH: return fire<BOTH>(big, rest, join, units[0], units[1], joins, st);
        case MIXED: return fire<MIXED>(big, rest, join, units[0], units[1], joins, st);
        case OUT: return fire<OUT>(big, rest, join, units[0], units[1], joins, st);
        default: return fire<WEIGHT>(big, rest, join, units[0], units[1], joins, st);
    }
}

int iterate(Jobs& s, const Scratch* sc, const Plan& p, int steps, const float* hyper, float decay, void* ws, hipStream_t st) {
    s.part = (double*)ws;
    s.ws = (_Float16*)((char*)ws + (long)MAXJ * NORMB * 8);
    Launch L{};
    L.dtype = s.dtype; L.hyper = hyper; L.decay = decay; L.ws = s.ws; L.slabs = (float*)(s.ws + p.planes);
    orth_norm_kernel<<<p.norm, 256, 0, st>>>(s);
    orth_split_kernel<<<p.split, 256, 0, st>>>(s);
    CPCSV_CHECK_LAUNCH();
    auto add = [&](int kind, const Job& j, long pp, long q, long d, int C, int K, float alpha) -> Task& {
        Task& t = L.t[L.n++];
        t = Task{};
        t.p = pp; t.q = q; t.d = d; t.R = j.M; t.C = C; t.K = K; t.alpha = alpha; t.symm = symmetric(kind);
        return t;
    };
    // where a job stands. P_k in p0, p1 in turn; Q_1 = P_1, Q_2 = P_2 P_1 in q0, Q_3 = P_3 Q_2 in q1
    enum { GRAM, POLY, COLLECT, NEXT, APPLY, END };
    struct { int phase, done, run, k; bool odd; } at[MAXJ] = {};               // odd: which X^T is current
    auto kind_of = [&](int i) {
        const auto& w = at[i];
        return w.phase == END ? -1 : w.phase == POLY ? SYMM_E : w.phase != APPLY ? SYMM : w.done + w.run < steps ? BOTH : hyper ? WEIGHT : OUT;
    };
    auto emit = [&](int i) {
        const Job& j = s.j[i];
        const Scratch& c = sc[i];
        auto& w = at[i];
        const long pk = w.k & 1 ? c.p0 : c.p1;
        switch (w.phase) {
            case GRAM:
                w.run = min(j.run, steps - w.done);
                w.k = 1;
                add(SYMM, j, j.x, j.x, c.a, j.M, j.N, SA / (SX * SX));
                w.phase = POLY;
                return;
            case POLY: {
                Task& t = add(SYMM_E, j, c.a, c.a, pk, j.M, j.M, NS_C * SP / (SA * SA));
                t.e = c.a; t.beta = NS_B * SP / SA; t.gamma = NS_A * SP;
                w.phase = w.run > 1 ? COLLECT : APPLY;
                return;
            }
            case COLLECT:
                if (w.k < w.run) add(SYMM, j, pk, c.a, c.r, j.M, j.M, 1.f / SP);
                if (w.k > 1) add(SYMM, j, pk, w.k == 2 ? c.p0 : c.q0, w.k == 2 ? c.q0 : c.q1, j.M, j.M, SQ[w.k] / (SP * SQ[w.k - 1]));
                w.phase = w.k < w.run ? NEXT : APPLY;
                return;
            case NEXT:
                add(SYMM, j, pk, c.r, c.a, j.M, j.M, 1.f / SP);
                ++w.k;
                w.phase = POLY;
                return;
            default: {
                const long q = w.run == 1 ? c.p0 : w.run == 2 ? c.q0 : c.q1;
                Task& t = add(BOTH, j, q, w.odd ? c.xt1 : j.xt, j.x, j.N, j.M, 1.f / SQ[w.run]);
                w.done += w.run;
                if (w.done < steps) t.dt = w.odd ? j.xt : c.xt1;
                else { t.d = (long)j.out; t.alpha /= SX; t.rows = j.rows; t.cols = j.cols; t.tall = j.tall; }
                w.odd = !w.odd;
                w.phase = w.done < steps ? GRAM : END;
            }
        }
    };
    // A level: the next products of all jobs that stand before some without E; of those with E if there are none; of the last ones. Jobs
    // of the same runs go in step, and five iterations in runs of one and of three share 17 levels.
    for (;;) {
        auto rank = [&](int kind) { return kind < 0 ? 3 : kind == SYMM || kind == BOTH ? 0 : kind == SYMM_E ? 1 : 2; };
        int least = 3, kinds = 0;
        for (int i = 0; i < s.n; ++i) least = min(least, rank(kind_of(i)));
        if (least == 3) return 0;
        L.n = 0;
        for (int i = 0; i < s.n; ++i)
            if (rank(kind_of(i)) == least) {
                L.kind = kind_of(i);
                kinds |= 1 << L.kind;
                emit(i);
            }
        if (kinds == (1 << SYMM | 1 << BOTH)) L.kind = MIXED;
        if (int rc = run_level(L, p.slabs, st)) return rc;
    }
}
}  // namespace

extern "C" long cpcsv_orth_workspace(const long* dims, int njobs) {
    Jobs s{};
    Scratch sc[MAXJ];
    Plan p;
    const int rc = plan(s, sc, dims, njobs, p);
    return rc ? rc : p.bytes;
}

extern "C" int cpcsv_orthogonalize(const void* const* g, void* const* out, const long* dims, int njobs, int dtype, int steps, float eps, void* ws,
                                   void* stream) {
    Jobs s{};
    Scratch sc[MAXJ];
    Plan p;
    if (int rc = plan(s, sc, dims, njobs, p)) return rc;
    if ((dtype != CPCSV_F32 && dtype != CPCSV_BF16) || steps < 1) return -1001;
    if (!g || !out || !ws) return -1003;
    for (int i = 0; i < njobs; ++i) {
        if (!g[i] || !out[i]) return -1003;
        s.j[i].g = g[i]; s.j[i].out = out[i];
    }
    s.dtype = dtype; s.eps = eps;
    return iterate(s, sc, p, steps, nullptr, 0.f, ws, (hipStream_t)stream);
}

extern "C" int cpcsv_muon_step(float* const* w, const float* const* g, float* const* m, const long* dims, int njobs, const float* hyper, float momentum,
                               int nesterov, float decay, int steps, float eps, void* ws, void* stream) {
    Jobs s{};
    Scratch sc[MAXJ];
    Plan p;
    if (int rc = plan(s, sc, dims, njobs, p)) return rc;
    if (steps < 1) return -1001;
    if (!w || !g || !m || !hyper || !ws) return -1003;
    for (int i = 0; i < njobs; ++i) {
        if (!w[i] || !g[i] || !m[i]) return -1003;
        s.j[i].g = g[i]; s.j[i].m = m[i]; s.j[i].out = w[i];
    }
    s.dtype = CPCSV_F32; s.eps = eps; s.mu = momentum; s.nesterov = nesterov;
    return iterate(s, sc, p, steps, hyper, decay, ws, (hipStream_t)stream);
}
