// orth.hip — an update orthogonalised by Newton-Schulz products, for many matrices at once, and the optimiser step around it:
//     m <- mu m + g      U = g + mu m (nesterov) or m      X_0 = U / (|U|_F + eps)
//     five times   A = X X^T    B = b A + c A^2    X <- a X + B X        w <- w (1 - lr decay) - lr sqrt(max(1, rows / cols)) X
// with (a, b, c) the quintic whose iteration takes singular values of (0, 1] towards 1; a tall matrix is worked on transposed, so
// that A is the smaller Gram matrix. Singular values stay below 1.21, entries too.
//
// Precision. One product in bf16 per step leaves the result 1e-2 off on well conditioned gradients and 3e-1 on those with a few
// strong directions: what is lost next to the large singular values is amplified by a^5 = 485 where they are small. The operands
// are therefore kept as TWO fp16 planes each, v = hi + lo with hi = fp16(v), lo = fp16(v - hi): 22 bits and lo's sign, an fp32's
// accuracy. A product is three MFMAs (hi hi, hi lo, lo hi; lo lo lies below the planes' own rounding), accumulated in fp32. The
// planes are scaled by powers of two so that entries far below 1 keep their low bits above fp16's subnormal step.
//
// All matrices of a call share each launch (a job list by value, no device tables). Planes are padded to whole tiles with zeros,
// which stay zeros, so that the K loops have no bounds.
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
typedef __attribute__((ext_vector_type(8))) _Float16 half8;
typedef __attribute__((ext_vector_type(4))) _Float16 half4;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
// |X| < 1.21, |A| < 1.45, |B| < 2.81 entrywise (each is bounded by the spectral norm): the scaled values stay below fp16's 65504
constexpr float SX = 16384.f, SA = 16384.f, SB = 4096.f;
constexpr int TILE = 128, BK = 32, MAXJ = CPCSV_ORTH_JOBS, NORMB = 256;

struct Job {
    const void* g; float* m; void* out;       // gradient, momentum (NULL: none), weight or result
    long x, xt0, xt1, a, b;                   // offsets of the hi planes in halves; the lo plane follows each
    int rows, cols;                           // of the matrix
    int M, N, tall;                           // padded min / max side; tall: rows > cols
    int t_norm, t_split, t_sym, t_x;          // first block of the job in each kind of launch
};
struct Jobs {
    Job j[MAXJ];
    int n, dtype, nesterov;
    float mu, eps, decay;
    const float* hyper;
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
__device__ __forceinline__ void split_of(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
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
        _Float16 hi, lo;
        split_of(u, hi, lo);
        union { _Float16 h[2]; uint32_t w; } p;
        p.h[0] = hi; p.h[1] = lo;
        t[i * 4 + rl][cl] = p.w;
    }
    __syncthreads();
    _Float16 *own = s.ws + (j.tall ? j.xt0 : j.x), *turned = s.ws + (j.tall ? j.x : j.xt0);
    const long plane = (long)j.M * j.N;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int line = i * 32 + (threadIdx.x >> 3), q = (threadIdx.x & 7) * 8;
#pragma unroll
        for (int way = 0; way < 2; ++way) {
            half8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                union { uint32_t w; _Float16 h[2]; } p;
                p.w = way ? t[q + e][line] : t[line][q + e];
                hi[e] = p.h[0]; lo[e] = p.h[1];
            }
            _Float16* d = way ? turned + (long)(c0 + line) * PR + r0 + q : own + (long)(r0 + line) * PC + c0 + q;
            *(half8*)d = hi;
            *(half8*)(d + plane) = lo;
        }
    }
}

// ---- the products: D = P Q^T over two-plane operands, 128 x 128 tiles, K in slices of 32 ------------------------------
// SYM_A: A = X X^T    SYM_B: B = b A + c A A    UPDATE: X <- a X + B X    LAST: the same, into the result or the weight
enum { SYM_A, SYM_B, UPDATE, LAST };

template <int KIND>
__global__ __launch_bounds__(256, 2) void orth_gemm_kernel(Jobs s, int flip) {
    __shared__ __attribute__((aligned(16))) _Float16 lds[2][4][TILE * BK];
    constexpr bool SYM = KIND == SYM_A || KIND == SYM_B;
    const int k = SYM ? job_of<&Job::t_sym>(s, blockIdx.x) : job_of<&Job::t_x>(s, blockIdx.x);
    const Job& j = s.j[k];
    int ti, tj;
    if (SYM) {                                   // lower triangle of tiles, row by row
        int t = blockIdx.x - j.t_sym;
        ti = 0;
        while (t > ti) { t -= ti + 1; ++ti; }
        tj = t;
    } else {
        const int t = blockIdx.x - j.t_x, tm = j.M / TILE;
        ti = t % tm;
        tj = t / tm;
    }
    const long MN = (long)j.M * j.N, MM = (long)j.M * j.M;
    const _Float16 *P, *Q;
    long pl, ql;                                 // plane sizes
    int K;                                       // = the operands' leading dimension
    _Float16* const X = s.ws + j.x;
    _Float16* const XT = s.ws + (flip ? j.xt1 : j.xt0);
    if (KIND == SYM_A) { P = X; Q = X; pl = ql = MN; K = j.N; }
    else if (KIND == SYM_B) { P = Q = s.ws + j.a; pl = ql = MM; K = j.M; }
    else { P = s.ws + j.b; Q = XT; pl = MM; ql = MN; K = j.M; }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const _Float16* src[4];
    src[0] = P + (long)ti * TILE * K;
    src[1] = src[0] + pl;
    src[2] = Q + (long)tj * TILE * K;
    src[3] = src[2] + ql;
    // a row of a slice is four 16-byte chunks; chunk q of row r lives in slot q ^ ((r >> 2) & 3), so that the 16 rows a fragment read
    // touches at one time fall into all of the banks. The DMA writes LDS in lane order: the swizzle is on the source side.
    auto stage = [&](int buf, int k0) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int idx = i * 256 + tid, row = idx >> 2, q = (idx & 3) ^ ((row >> 2) & 3);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[p] + (long)row * K + k0 + q * 8),
                                                 (__attribute__((address_space(3))) void*)(&lds[buf][p][(i * 256 + wave * 64) * 8]), 16, 0, 0);
            }
    };
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64, fr = lane & 31, fk = lane >> 5;
    f32x16 acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;
    stage(0, 0);
    const int nk = K / BK;
    for (int kt = 0; kt < nk; ++kt) {
        const int buf = kt & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (kt + 1 < nk) stage(buf ^ 1, (kt + 1) * BK);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            half8 f[4][2];
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const int row = (p < 2 ? wm : wn) + a * 32 + fr, q = (kk * 2 + fk) ^ ((row >> 2) & 3);
                    f[p][a] = *(const half8*)&lds[buf][p][row * BK + q * 8];
                }
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[0][a], f[3][b], acc[a][b], 0, 0, 0);
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[1][a], f[2][b], acc[a][b], 0, 0, 0);
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[0][a], f[2][b], acc[a][b], 0, 0, 0);
                }
        }
    }
    // a lane's 16 values of a 32 x 32 block: column lane % 32, rows 8 (e / 4) + 4 (lane / 32) + e % 4
    const float lr = KIND == LAST && s.hyper ? s.hyper[0] : 0.f;
    const float keep = 1.f - lr * s.decay, step = lr * sqrtf(fmaxf(1.f, (float)j.rows / (float)j.cols));
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const int r = ti * TILE + wm + a * 32 + h * 8 + fk * 4, c = tj * TILE + wn + b * 32 + fr;
                half4 vh, vl;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = acc[a][b][h * 4 + e];
                    if (KIND == SYM_A) v[e] = x * (SA / (SX * SX));
                    else if (KIND == SYM_B) {
                        const _Float16* o = s.ws + j.a + (long)(r + e) * j.M + c;
                        v[e] = ((float)o[0] + (float)o[MM]) * (NS_B * SB / SA) + x * (NS_C * SB / (SA * SA));
                    } else {
                        const _Float16* o = X + (long)(r + e) * j.N + c;
                        const float old = (float)o[0] + (float)o[MN];
                        v[e] = KIND == LAST ? old * (NS_A / SX) + x * (1.f / (SB * SX)) : old * NS_A + x * (1.f / SB);
                    }
                    _Float16 hi, lo;
                    split_of(v[e], hi, lo);
                    vh[e] = hi; vl[e] = lo;
                }
                if (SYM) {
                    // the tile and its mirror image; on the diagonal each pair of entries is taken from one of its two sums
                    _Float16* d = s.ws + (KIND == SYM_A ? j.a : j.b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (r + e >= c) { d[(long)(r + e) * j.M + c] = vh[e]; d[(long)(r + e) * j.M + c + MM] = vl[e]; }
                        if (r + e > c) { d[(long)c * j.M + r + e] = vh[e]; d[(long)c * j.M + r + e + MM] = vl[e]; }
                    }
                } else if (KIND == UPDATE) {
                    _Float16* t = s.ws + (flip ? j.xt0 : j.xt1) + (long)c * j.M + r;
                    *(half4*)t = vh;
                    *(half4*)(t + MN) = vl;
#pragma unroll
                    for (int e = 0; e < 4; ++e) { X[(long)(r + e) * j.N + c] = vh[e]; X[(long)(r + e) * j.N + c + MN] = vl[e]; }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int R = j.tall ? c : r + e, C = j.tall ? r + e : c;
                        if (R >= j.rows || C >= j.cols) continue;
                        const long at = (long)R * j.cols + C;
                        if (s.hyper) ((float*)j.out)[at] = ((float*)j.out)[at] * keep - step * v[e];
                        else if (s.dtype == CPCSV_F32) ((float*)j.out)[at] = v[e];
                        else ((bf16_t*)j.out)[at] = f32_to_bf16(v[e]);
                    }
                }
            }
}

struct Plan { long bytes; int norm, split, sym, x; };
int plan(Jobs& s, const long* dims, int njobs, Plan& p) {
    if (njobs <= 0 || njobs > MAXJ || !dims) return -1001;
    long at = 0;
    p = Plan{0, 0, 0, 0, 0};
    for (int i = 0; i < njobs; ++i) {
        const long r = dims[2 * i], c = dims[2 * i + 1];
        if (r <= 0 || c <= 0 || r > CPCSV_ORTH_MAX_SIDE || c > CPCSV_ORTH_MAX_SIDE) return -1002;
        Job& j = s.j[i];
        j.rows = (int)r; j.cols = (int)c; j.tall = r > c;
        j.M = (int)((j.tall ? c : r) + TILE - 1) / TILE * TILE;
        j.N = (int)((j.tall ? r : c) + TILE - 1) / TILE * TILE;
        const long mn = (long)j.M * j.N, mm = (long)j.M * j.M;
        j.x = at; j.xt0 = at + 2 * mn; j.xt1 = at + 4 * mn; j.a = at + 6 * mn; j.b = j.a + 2 * mm;
        at = j.b + 2 * mm;
        const long tm = j.M / TILE, tn = j.N / TILE;
        j.t_norm = p.norm; j.t_split = p.split; j.t_sym = p.sym; j.t_x = p.x;
        p.norm += norm_blocks(j.rows, j.cols);
        if (p.split + tm * tn * 4 > (1L << 30)) return -1002;
        p.split += (int)(tm * tn * 4);
        p.sym += (int)(tm * (tm + 1) / 2);
        p.x += (int)(tm * tn);
    }
    s.n = njobs;
    p.bytes = at * 2 + (long)MAXJ * NORMB * 8;
    return 0;
}

int iterate(Jobs& s, const Plan& p, int steps, void* ws, hipStream_t st) {
    s.part = (double*)ws;
    s.ws = (_Float16*)((char*)ws + (long)MAXJ * NORMB * 8);
    orth_norm_kernel<<<p.norm, 256, 0, st>>>(s);
    orth_split_kernel<<<p.split, 256, 0, st>>>(s);
    for (int i = 0; i < steps; ++i) {
        orth_gemm_kernel<SYM_A><<<p.sym, 256, 0, st>>>(s, i & 1);
        orth_gemm_kernel<SYM_B><<<p.sym, 256, 0, st>>>(s, i & 1);
        if (i + 1 < steps) orth_gemm_kernel<UPDATE><<<p.x, 256, 0, st>>>(s, i & 1);
        else orth_gemm_kernel<LAST><<<p.x, 256, 0, st>>>(s, i & 1);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}
}  // namespace

extern "C" long cpcsv_orth_workspace(const long* dims, int njobs) {
    Jobs s{};
    Plan p;
    const int rc = plan(s, dims, njobs, p);
    return rc ? rc : p.bytes;
}

extern "C" int cpcsv_orthogonalize(const void* const* g, void* const* out, const long* dims, int njobs, int dtype, int steps, float eps, void* ws,
                                   void* stream) {
    Jobs s{};
    Plan p;
    if (int rc = plan(s, dims, njobs, p)) return rc;
    if ((dtype != CPCSV_F32 && dtype != CPCSV_BF16) || steps < 1) return -1001;
    if (!g || !out || !ws) return -1003;
    for (int i = 0; i < njobs; ++i) {
        if (!g[i] || !out[i]) return -1003;
        s.j[i].g = g[i]; s.j[i].out = out[i];
    }
    s.dtype = dtype; s.eps = eps;
    return iterate(s, p, steps, ws, (hipStream_t)stream);
}

extern "C" int cpcsv_muon_step(float* const* w, const float* const* g, float* const* m, const long* dims, int njobs, const float* hyper, float momentum,
                               int nesterov, float decay, int steps, float eps, void* ws, void* stream) {
    Jobs s{};
    Plan p;
    if (int rc = plan(s, dims, njobs, p)) return rc;
    if (steps < 1) return -1001;
    if (!w || !g || !m || !hyper || !ws) return -1003;
    for (int i = 0; i < njobs; ++i) {
        if (!w[i] || !g[i] || !m[i]) return -1003;
        s.j[i].g = g[i]; s.j[i].m = m[i]; s.j[i].out = w[i];
    }
    s.dtype = CPCSV_F32; s.eps = eps; s.mu = momentum; s.nesterov = nesterov; s.decay = decay; s.hyper = hyper;
    return iterate(s, p, steps, ws, (hipStream_t)stream);
}
