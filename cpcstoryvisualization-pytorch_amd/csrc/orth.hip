// orth.hip — an update orthogonalised by Newton-Schulz products, for many matrices at once, and the optimiser step around it:
//     m <- mu m + g      U = g + mu m (nesterov) or m      X = U / (|U|_F + eps)
//     five times   X <- P(X X^T) X,  P(A) = a I + b A + c A^2          w <- w (1 - lr decay) - lr sqrt(max(1, rows / cols)) X
// with (a, b, c) the quintic whose iteration takes singular values of (0, 1] towards 1; a tall matrix is worked on transposed, so
// that A is the smaller (M x M) Gram matrix.
//
// Through the Gram matrix. Everything an iteration applies to X is a polynomial of A, and the next Gram matrix is P A P: up to three
// iterations run on M x M matrices alone (Q <- P Q collects what they apply, A <- P (P A)), then X <- Q X once. Five iterations in
// two runs (3 + 2) cost 6 M^2 N + 14 M^3 instead of the 15 M^2 N + 5 M^3 of forming X each time (all M x M results are symmetric:
// one triangle is computed): equal for square matrices, 2.5 times fewer operations for wide ones. Runs longer than three lose what
// lies far below the largest singular value (the Gram matrix holds its square): in fp32 all five in one run are up to 25 times
// further off than X formed each time, 3 + 2 at most twice.
//
// Precision. One product in bf16 per step leaves the result 1e-2 off on well conditioned gradients and 3e-1 on those with a few
// strong directions: what is lost next to the large singular values is amplified by a^5 = 485 where they are small. The operands
// are therefore kept as TWO fp16 planes each, v = hi + lo with hi = fp16(v), lo = fp16(v - hi): 22 bits and lo's sign, an fp32's
// accuracy. A product is three MFMAs (hi hi, hi lo, lo hi; lo lo lies below the planes' own rounding), accumulated in fp32. The
// planes are scaled by powers of two so that entries far below 1 keep their low bits above fp16's subnormal step.
//
// All matrices of a call share each launch (a task list by value, no device tables): the products of one dependency level. Planes
// are padded to whole tiles with zeros, which stay zeros, so that the K loops have no bounds.
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
// Entries are bounded by spectral norms: |X| < 1.21, |A| and |P A| < 1.45, |P| < 3.45, |Q| < 3.45^k behind k iterations. The scaled
// values stay below fp16's 65504.
constexpr float SX = 16384.f, SA = 16384.f, SP = 8192.f;
constexpr float SQ[4] = {0.f, SP, 4096.f, 1024.f};
constexpr int RUN = 3;                         // iterations between two X
constexpr int PAD = 128, MAXJ = CPCSV_ORTH_JOBS, MAXT = 2 * MAXJ, NORMB = 256;

struct Job {
    const void* g; float* m; void* out;       // gradient, momentum (NULL: none), weight or result
    long x, xt;                               // offsets of the hi planes in halves; the lo plane follows each
    int rows, cols;                           // of the matrix
    int M, N, tall;                           // padded min / max side; tall: rows > cols
    int t_norm, t_split;                      // first block of the job
};
struct Jobs {
    Job j[MAXJ];
    int n, dtype, nesterov;
    float mu, eps;
    double* part;
    _Float16* ws;
};

template <int Job::*FIRST> __device__ __forceinline__ int job_of(const Jobs& s, int block) {
    int k = 0;
    while (k + 1 < s.n && block >= s.j[k + 1].*FIRST) ++k;
    return k;
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
__global__ __launch_bounds__(256) void orth_norm_kernel(Jobs s) {
    const int k = job_of<&Job::t_norm>(s, blockIdx.x);
    const Job& j = s.j[k];
    const int blk = blockIdx.x - j.t_norm, nb = norm_blocks(j.rows, j.cols);
    const long n = (long)j.rows * j.cols;
    double q = 0.0;
    for (long i = (long)blk * 256 + threadIdx.x; i < n; i += (long)nb * 256) {
        float u = ld_g(j.g, s.dtype, i);
        if (j.m) {
            const float m = __fmaf_rn(s.mu, j.m[i], u);
            j.m[i] = m;
            u = s.nesterov ? __fmaf_rn(s.mu, m, u) : m;
        }
        q += (double)u * (double)u;
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
__global__ __launch_bounds__(256) void orth_split_kernel(Jobs s) {
    __shared__ uint32_t t[64][65];
    __shared__ double sh[256];
    const int k = job_of<&Job::t_split>(s, blockIdx.x);
    const Job& j = s.j[k];
    sh[threadIdx.x] = threadIdx.x < norm_blocks(j.rows, j.cols) ? s.part[k * NORMB + threadIdx.x] : 0.0;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    const float inv = (float)((double)SX / (sqrt(sh[0]) + (double)s.eps));
    const int PR = j.tall ? j.N : j.M, PC = j.tall ? j.M : j.N, tile = blockIdx.x - j.t_split;
    const int r0 = tile / (PC / 64) * 64, c0 = tile % (PC / 64) * 64;
    const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + i * 4 + rl, c = c0 + cl;
        float u = 0.f;
        if (r < j.rows && c < j.cols) {
            const long at = (long)r * j.cols + c;
            u = ld_g(j.g, s.dtype, at);
            if (j.m) u = s.nesterov ? __fmaf_rn(s.mu, j.m[at], u) : j.m[at];
            u *= inv;
        }
        t[i * 4 + rl][cl] = split_of(u);
    }
    __syncthreads();
    _Float16 *own = s.ws + (j.tall ? j.xt : j.x), *turned = s.ws + (j.tall ? j.x : j.xt);
    const long plane = (long)j.M * j.N;
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
            _Float16* d = way ? turned + (long)(c0 + line) * PR + r0 + q : own + (long)(r0 + line) * PC + c0 + q;
            *(half8*)d = hi;
            *(half8*)(d + plane) = lo;
        }
    }
}

// ---- the products: D = alpha P Q^T + beta E + gamma I over two-plane operands [rows][K] ------------------------------
enum { SYMM, BOTH, OUT };      // D symmetric: lower triangle and its mirror image | D and its transpose | the result or the weight
struct Task {
    long p, q, e, d, dt;       // offsets of the hi planes in halves (e < 0: none); OUT: d is the output's address
    long slab;                 // first partial tile, in floats
    int R, C, K;
    float alpha, beta, gamma;
    int kind, t0, tiles, S, r0;               // first block, tiles, slices of K, first block of the joining launch
    int rows, cols, tall;                     // OUT: of the output
};
struct Launch {
    Task t[MAXT];
    int n, dtype;
    float decay;
    const float* hyper;
    _Float16* ws;
    float* slabs;
};

// Tiles. A wavefront's share of a tile sets what it reads from LDS for each MFMA, and LDS bandwidth is what bounds the main loop:
// 256 x 256 with 128 x 64 a wavefront runs 1245 TFLOP/s (three MFMAs a product counted) on 4096^3 against 860 for 128 x 128 with
// 64 x 64, which packs two blocks on a CU and fills the chip at half the tiles (1024 x 18432 x 1024: 962 against 757), and 64 x 64
// has the shortest way through a few hundred K (512^3: 6.7 us against 13.3 and 34).
template <int BM_, int WM_, int WN_, int BK_> struct Cfg {
    static constexpr int BM = BM_, WM = WM_, WN = WN_, BK = BK_, WC = BM / WN, T = (BM / WM) * WC * 64, CPR = BK / 8;
    static constexpr int LD = BM * CPR / T;                       // 16-byte loads a thread, operand plane and stage
    static constexpr int STAGE = 4 * BM * BK;                     // halves
    static constexpr int SW = WN < 64 ? WN : 64;                  // columns of an epilogue strip
    static constexpr int LDS = 2 * STAGE * 2 > (T / 64) * 32 * (SW + 1) * 4 ? 2 * STAGE * 2 : (T / 64) * 32 * (SW + 1) * 4;
    static constexpr int MA = WM / 32, MB = WN / 32, ACC = MA * MB * 16;
    // chunk (16 bytes) q of LDS row r lives in slot q ^ swz(r): the rows a fragment read touches together fall into all banks. The
    // DMA writes LDS in lane order, so the permutation is on the source side.
    static __device__ __forceinline__ int swz(int r) { return CPR == 4 ? (r >> 2) & 3 : (r >> 1) & 7; }
};
using Big = Cfg<256, 128, 64, 32>;
using Mid = Cfg<128, 64, 64, 32>;
using Small = Cfg<64, 32, 32, 64>;

__device__ __forceinline__ void tile_of(const Task& t, int tile, int bm, int& ti, int& tj) {
    if (t.kind == SYMM) {                        // lower triangle, row by row
        ti = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {                                     // bands of 8 tile rows, so that a run of tiles shares operand rows in L2
        const int tm = (t.R + bm - 1) / bm, tn = (t.C + bm - 1) / bm, g = tile / (8 * tn), gr = min(8, tm - g * 8), w = tile - g * 8 * tn;
        ti = g * 8 + w % gr;
        tj = w / gr;
    }
}

// acc of one wavefront -> D. A lane's 16 values of a 32 x 32 block: column lane % 32, rows 8 (i / 4) + 4 (lane / 32) + i % 4; they
// pass through the wavefront's own piece of LDS, 32 rows x SW columns at a time, to leave as 16-byte pieces of rows in either
// orientation.
template <typename C>
__device__ __forceinline__ void finish(const Launch& s, const Task& t, int ti, int tj, const f32x16 (&acc)[C::MA][C::MB], uint32_t* lds) {
    constexpr int SW = C::SW, LDW = SW + 1, NB = SW / 32;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 31, fk = lane >> 5;
    uint32_t* buf = lds + wave * 32 * LDW;
    const long RC = (long)t.R * t.C;
    const float lr = t.kind == OUT && s.hyper ? s.hyper[0] : 0.f;
    const float keep = 1.f - lr * s.decay, step = lr * sqrtf(fmaxf(1.f, (float)t.rows / (float)t.cols));
#pragma unroll
    for (int a = 0; a < C::MA; ++a)
#pragma unroll
        for (int b0 = 0; b0 < C::MB; b0 += NB) {
            const int r0 = ti * C::BM + wave / C::WC * C::WM + a * 32, c0 = tj * C::BM + wave % C::WC * C::WN + b0 * 32;
            if (r0 >= t.R || c0 >= t.C || (t.kind == SYMM && r0 + 31 < c0)) continue;      // (sides are multiples of a strip's)
            const bool diag = t.kind == SYMM && r0 < c0 + SW;                              // the strip meets the diagonal
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int rl = (i >> 2) * 8 + fk * 4 + (i & 3), cl = b * 32 + fr, r = r0 + rl, c = c0 + cl;
                    float v = acc[a][b0 + b][i] * t.alpha;
                    if (t.e >= 0) {
                        const _Float16* o = s.ws + t.e + (long)r * t.C + c;
                        v += ((float)o[0] + (float)o[RC]) * t.beta + (r == c ? t.gamma : 0.f);
                    }
                    buf[rl * LDW + cl] = t.kind == OUT ? __float_as_uint(v) : split_of(v);
                }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            if (t.kind == OUT) {
                // rows of the output run along the strip's columns, of a tall one's along its rows
                const int len = t.tall ? 32 : SW, lines = t.tall ? SW : 32, per = 64 / len;
                const int sub = lane % len;
                for (int l = lane / len; l < lines; l += per) {
                    const float v = __uint_as_float(t.tall ? buf[sub * LDW + l] : buf[l * LDW + sub]);
                    const int R = (t.tall ? c0 : r0) + l, Cc = (t.tall ? r0 : c0) + sub;
                    if (R >= t.rows || Cc >= t.cols) continue;
                    const long at = (long)R * t.cols + Cc;
                    if (s.hyper) ((float*)t.d)[at] = ((float*)t.d)[at] * keep - step * v;
                    else if (s.dtype == CPCSV_F32) ((float*)t.d)[at] = v;
                    else ((bf16_t*)t.d)[at] = f32_to_bf16(v);
                }
                continue;
            }
            if (diag) {
                // each pair of entries is taken from the lower one: the two sums are the same numbers in another order
                for (int i = lane; i < 32 * SW; i += 64) {
                    const int rl = i / SW, cl = i % SW, r = r0 + rl, c = c0 + cl;
                    if (r < c) continue;
                    union { uint32_t w; _Float16 h[2]; } p;
                    p.w = buf[rl * LDW + cl];
                    _Float16* d = s.ws + t.d;
                    d[(long)r * t.C + c] = p.h[0];
                    d[(long)r * t.C + c + RC] = p.h[1];
                    d[(long)c * t.C + r] = p.h[0];
                    d[(long)c * t.C + r + RC] = p.h[1];
                }
                continue;
            }
            uint32_t w[8];
            half8 hi, lo;
            constexpr int PC = SW / 8, RP = 64 / PC;              // 16-byte pieces of a strip row, rows a pass
#pragma unroll
            for (int i = 0; i < 32 / RP; ++i) {
                const int rl = i * RP + lane / PC, cl = lane % PC * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = buf[rl * LDW + cl + e];
                planes_of(w, hi, lo);
                _Float16* d = s.ws + t.d + (long)(r0 + rl) * t.C + c0 + cl;
                *(half8*)d = hi;
                *(half8*)(d + RC) = lo;
            }
            _Float16* const turned = s.ws + (t.kind == SYMM ? t.d : t.dt);                 // (D^T [C][R]; R = C for a symmetric one)
#pragma unroll
            for (int i = 0; i < SW / 16; ++i) {
                const int cl = i * 16 + lane / 4, rl = lane % 4 * 8;
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = buf[(rl + e) * LDW + cl];
                planes_of(w, hi, lo);
                _Float16* d = turned + (long)(c0 + cl) * t.R + r0 + rl;
                *(half8*)d = hi;
                *(half8*)(d + RC) = lo;
            }
        }
}

template <typename C>
__global__ __launch_bounds__(C::T) void orth_gemm_kernel(Launch s) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    _Float16* const lds = (_Float16*)smem;
    // blocks go to the eight XCDs in turn: give each a contiguous run of tiles, whose operands its L2 then holds
    const int nb = gridDim.x, per = nb >> 3, rest = nb & 7, xcd = blockIdx.x & 7;
    const int unit = xcd * per + min(xcd, rest) + (blockIdx.x >> 3);
    int k = 0;
    while (k + 1 < s.n && unit >= s.t[k + 1].t0) ++k;
    const Task& t = s.t[k];
    const int tile = (unit - t.t0) % t.tiles, sl = (unit - t.t0) / t.tiles;
    int ti, tj;
    tile_of(t, tile, C::BM, ti, tj);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, K = t.K;
    const int nk = K / C::BK, k0 = (int)((long)nk * sl / t.S), k1 = (int)((long)nk * (sl + 1) / t.S);
    const _Float16* src[2] = {s.ws + t.p + (long)ti * C::BM * K, s.ws + t.q + (long)tj * C::BM * K};
    const long pl[2] = {(long)t.R * K, (long)t.C * K};
    int off[2][C::LD];                           // (K <= 131072 and 256 rows: below 2^31)
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int i = 0; i < C::LD; ++i) {
            const int idx = i * C::T + tid, row = idx / C::CPR, q = (idx % C::CPR) ^ C::swz(row);
            const int last = (o ? t.C - tj * C::BM : t.R - ti * C::BM) - 1;               // a tile may hang over the padded side
            off[o][i] = min(row, last) * K + q * 8;
        }
    auto stage = [&](int buf, int kt) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int i = 0; i < C::LD; ++i)
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[o] + (p ? pl[o] : 0) + off[o][i] + kt * C::BK),
                                                     (__attribute__((address_space(3))) void*)(lds + buf * C::STAGE + (o * 2 + p) * C::BM * C::BK +
                                                                                               (i * C::T + wave * 64) * 8), 16, 0, 0);
    };
    const int wm = wave / C::WC * C::WM, wn = wave % C::WC * C::WN, fr = lane & 31, fk = lane >> 5;
    f32x16 acc[C::MA][C::MB];
#pragma unroll
    for (int a = 0; a < C::MA; ++a)
#pragma unroll
        for (int b = 0; b < C::MB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
    if (k0 < k1) stage(0, k0);
    for (int kt = k0; kt < k1; ++kt) {
        const int buf = (kt - k0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (kt + 1 < k1) stage(buf ^ 1, kt + 1);
        const _Float16* base = lds + buf * C::STAGE;
#pragma unroll
        for (int kk = 0; kk < C::BK / 16; ++kk) {
            half8 fp[2][C::MA], fq[2][C::MB];
#pragma unroll
            for (int p = 0; p < 2; ++p) {
#pragma unroll
                for (int a = 0; a < C::MA; ++a) {
                    const int row = wm + a * 32 + fr;
                    fp[p][a] = *(const half8*)(base + p * C::BM * C::BK + row * C::BK + ((kk * 2 + fk) ^ C::swz(row)) * 8);
                }
#pragma unroll
                for (int b = 0; b < C::MB; ++b) {
                    const int row = wn + b * 32 + fr;
                    fq[p][b] = *(const half8*)(base + (2 + p) * C::BM * C::BK + row * C::BK + ((kk * 2 + fk) ^ C::swz(row)) * 8);
                }
            }
#pragma unroll
            for (int a = 0; a < C::MA; ++a)
#pragma unroll
                for (int b = 0; b < C::MB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][a], fq[1][b], acc[a][b], 0, 0, 0);
#pragma unroll
            for (int a = 0; a < C::MA; ++a)
#pragma unroll
                for (int b = 0; b < C::MB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[1][a], fq[0][b], acc[a][b], 0, 0, 0);
#pragma unroll
            for (int a = 0; a < C::MA; ++a)
#pragma unroll
                for (int b = 0; b < C::MB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fp[0][a], fq[0][b], acc[a][b], 0, 0, 0);
        }
    }
    if (t.S > 1) {                               // a slice's share of the tile, in the order the registers hold it
        f32x4* d = (f32x4*)(s.slabs + t.slab) + (long)(tile * t.S + sl) * (C::ACC / 4) * C::T + tid;
#pragma unroll
        for (int a = 0; a < C::MA; ++a)
#pragma unroll
            for (int b = 0; b < C::MB; ++b)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    f32x4 v = {acc[a][b][h * 4], acc[a][b][h * 4 + 1], acc[a][b][h * 4 + 2], acc[a][b][h * 4 + 3]};
                    d[((a * C::MB + b) * 4 + h) * C::T] = v;
                }
        return;
    }
    __syncthreads();
    finish<C>(s, t, ti, tj, acc, (uint32_t*)smem);
}

// slices of a tile, added in order
template <typename C>
__global__ __launch_bounds__(C::T) void orth_join_kernel(Launch s) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    int k = 0;
    while (k + 1 < s.n && (int)blockIdx.x >= s.t[k + 1].r0) ++k;
    const Task& t = s.t[k];
    const int tile = blockIdx.x - t.r0;
    int ti, tj;
    tile_of(t, tile, C::BM, ti, tj);
    const f32x4* d = (const f32x4*)(s.slabs + t.slab) + (long)tile * t.S * (C::ACC / 4) * C::T + threadIdx.x;
    f32x16 acc[C::MA][C::MB];
#pragma unroll
    for (int a = 0; a < C::MA; ++a)
#pragma unroll
        for (int b = 0; b < C::MB; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
    for (int sl = 0; sl < t.S; ++sl)
#pragma unroll
        for (int a = 0; a < C::MA; ++a)
#pragma unroll
            for (int b = 0; b < C::MB; ++b)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const f32x4 v = d[((long)sl * (C::ACC / 4) + (a * C::MB + b) * 4 + h) * C::T];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a][b][h * 4 + e] += v[e];
                }
    finish<C>(s, t, ti, tj, acc, (uint32_t*)smem);
}

// ---- host: the schedule ---------------------------------------------------------------------------------------------
// Slices of K depend on the product alone, so that a matrix has the same bits in any company: a product whose 128 x 128 tiles leave
// CUs idle is cut into enough slices to fill them twice, none shorter than 512. (1024 x 18432 against itself: 36 tiles took 470 us.)
int slices(int kind, long R, long C, long K) {
    const long tm = (R + 127) / 128, tn = (C + 127) / 128, tiles = kind == SYMM ? tm * (tm + 1) / 2 : tm * tn;
    return (int)max(1L, min((512 + tiles - 1) / tiles, K / 512 > 1 && K >= 2048 ? K / 512 : 1));
}
long tiles_of(const Task& t, int bm) {
    const long tm = (t.R + bm - 1) / bm, tn = (t.C + bm - 1) / bm;
    return t.kind == SYMM ? tm * (tm + 1) / 2 : tm * tn;
}
// The tile of a launch: the least of (whole rounds of blocks over 256 CUs) x (K steps) x (measured time of a step), with a block's
// fixed part. Times in us; `two`: of a step when two blocks share the CU (Big: one fits).
struct Shape { int bm, bk, fit; double one, two, fixed; };
constexpr Shape SHAPES[3] = {{256, 32, 1, 2.4, 2.4, 5.0}, {128, 32, 2, 0.72, 1.6, 3.0}, {64, 64, 2, 0.57, 1.14, 2.0}};
int pick(const Launch& s) {
    int best = 0;
    double least = 1e30;
    for (int c = 0; c < 3; ++c) {
        double units = 0, steps = 0, longest = 0;
        for (int i = 0; i < s.n; ++i) {
            const double u = (double)tiles_of(s.t[i], SHAPES[c].bm) * s.t[i].S, n = (double)s.t[i].K / SHAPES[c].bk / s.t[i].S;
            units += u;
            steps += u * n;
            longest = n > longest ? n : longest;
        }
        const double slots = 256.0 * SHAPES[c].fit, n = steps / units, full = (double)(long)(units / slots), rest = units - full * slots;
        double us = full * (n * SHAPES[c].two + SHAPES[c].fixed);
        if (rest > 0) us += (full ? n : longest) * (rest <= 256 ? SHAPES[c].one : SHAPES[c].two) + SHAPES[c].fixed;
        if (us < least) { least = us; best = c; }
    }
    return best;
}

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
        const long mn = 2L * j.M * j.N, mm = 2L * j.M * j.M;
        j.x = at; j.xt = at + mn; sc[i].xt1 = at + 2 * mn;
        at += 3 * mn;
        long* const m6[6] = {&sc[i].a, &sc[i].p0, &sc[i].p1, &sc[i].r, &sc[i].q0, &sc[i].q1};
        for (long* v : m6) { *v = at; at += mm; }
        j.t_norm = p.norm; j.t_split = p.split;
        p.norm += norm_blocks(j.rows, j.cols);
        const long t64 = (long)(j.M / 64) * (j.N / 64);
        if (p.split + t64 > (1L << 30)) return -1002;
        p.split += (int)t64;
        // (a tile of any shape has at most the slices' floats; sides hang over by less than a 256 tile)
        const long need = max((long)slices(SYMM, j.M, j.M, j.N) * (j.M + 256) * (j.M + 256) * (slices(SYMM, j.M, j.M, j.N) > 1),
                              max((long)slices(SYMM, j.M, j.M, j.M) * (j.M + 256) * (j.M + 256) * 2 * (slices(SYMM, j.M, j.M, j.M) > 1),
                                  (long)slices(BOTH, j.M, j.N, j.M) * (j.M + 256) * (j.N + 256) * (slices(BOTH, j.M, j.N, j.M) > 1)));
        slabs += need;
    }
    s.n = njobs;
    p.planes = at;
    p.slabs = slabs;
    p.bytes = (long)MAXJ * NORMB * 8 + at * 2 + slabs * 4;
    return 0;
}

template <typename C> int go(Launch& s, long slabs, hipStream_t st) {
    int units = 0, joins = 0;
    long at = 0;
    for (int i = 0; i < s.n; ++i) {
        Task& t = s.t[i];
        const long n = tiles_of(t, C::BM);
        t.tiles = (int)n;
        t.t0 = units; t.r0 = joins; t.slab = at;
        if (units + n * t.S > (1L << 30)) return -1002;
        units += (int)(n * t.S);
        if (t.S > 1) {
            joins += (int)n;
            at += n * t.S * C::BM * C::BM;
        }
    }
    if (at > slabs) return -1004;
    if (C::LDS > 64 * 1024) {                                   // more than the default cap of dynamic LDS: raise it once
        static const hipError_t a = hipFuncSetAttribute(reinterpret_cast<const void*>(orth_gemm_kernel<C>), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
        static const hipError_t b = hipFuncSetAttribute(reinterpret_cast<const void*>(orth_join_kernel<C>), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
        if (a != hipSuccess || b != hipSuccess) return -(int)(a != hipSuccess ? a : b);
    }
    orth_gemm_kernel<C><<<units, C::T, C::LDS, st>>>(s);
    if (joins) {
        Launch only = s;                                        // the sliced products alone
        only.n = 0;
        for (int i = 0; i < s.n; ++i)
            if (s.t[i].S > 1) only.t[only.n++] = s.t[i];
        orth_join_kernel<C><<<joins, C::T, (C::T / 64) * 32 * (C::SW + 1) * 4, st>>>(only);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}
int run_level(Launch& s, long slabs, hipStream_t st) {
    if (!s.n) return 0;
    const int c = pick(s);
    return c == 0 ? go<Big>(s, slabs, st) : c == 1 ? go<Mid>(s, slabs, st) : go<Small>(s, slabs, st);
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
        t.p = pp; t.q = q; t.d = d; t.e = -1; t.R = j.M; t.C = C; t.K = K; t.alpha = alpha; t.kind = kind;
        t.S = slices(kind, t.R, t.C, t.K);
        return t;
    };
    auto level = [&]() { const int rc = run_level(L, p.slabs, st); L.n = 0; return rc; };
#define LEVEL(...)                                                          \
    do {                                                                    \
        for (int i = 0; i < s.n; ++i) { const Job& j = s.j[i]; const Scratch& c = sc[i]; __VA_ARGS__ } \
        if (int rc = level()) return rc;                                    \
    } while (0)
    bool odd = false;                            // which X^T is current
    for (int done = 0; done < steps;) {
        const int run = min(RUN, steps - done);
        LEVEL(add(SYMM, j, j.x, j.x, c.a, j.M, j.N, SA / (SX * SX)););
        for (int k = 1; k <= run; ++k) {
            // P_k in p0, p1 in turn; Q_1 = P_1, Q_2 = P_2 P_1 in q0, Q_3 = P_3 Q_2 in q1
            LEVEL(Task& t = add(SYMM, j, c.a, c.a, k & 1 ? c.p0 : c.p1, j.M, j.M, NS_C * SP / (SA * SA));
                  t.e = c.a; t.beta = NS_B * SP / SA; t.gamma = NS_A * SP;);
            if (k > 1 || k < run)
                LEVEL(const long pk = k & 1 ? c.p0 : c.p1;
                      if (k < run) add(SYMM, j, pk, c.a, c.r, j.M, j.M, 1.f / SP);
                      if (k > 1) add(SYMM, j, pk, k == 2 ? c.p0 : c.q0, k == 2 ? c.q0 : c.q1, j.M, j.M, SQ[k] / (SP * SQ[k - 1])););
            if (k < run) LEVEL(add(SYMM, j, k & 1 ? c.p0 : c.p1, c.r, c.a, j.M, j.M, 1.f / SP););
        }
        done += run;
        LEVEL(const long q = run == 1 ? c.p0 : run == 2 ? c.q0 : c.q1;
              Task& t = add(done < steps ? BOTH : OUT, j, q, odd ? c.xt1 : j.xt, j.x, j.N, j.M, 1.f / SQ[run]);
              if (done < steps) t.dt = odd ? j.xt : c.xt1;
              else { t.d = (long)j.out; t.alpha /= SX; t.rows = j.rows; t.cols = j.cols; t.tall = j.tall; });
        odd = !odd;
    }
#undef LEVEL
    return 0;
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
