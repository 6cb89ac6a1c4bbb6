// blocknorm.hip — the root-mean-square norms before and after a block, fused with the block's gate and residual scale:
//     uh = u ru,  ru = (mean u^2 + eps)^-1/2        x' = x + scale * gate * w_post * uh
//     xh = x' rx, rx = (mean x'^2 + eps)^-1/2       z  = w_next * xh
// (u the block's output, x the residual stream, z the next block's input), and their gradients. With g = dz w_next:
//     dx = dx' + rx (g - xh mean(g xh))             q = dx scale gate w_post       du = ru (q - uh mean(q uh))
//     dgate = dx scale w_post uh    dw_next = sum dz xh    dw_post = scale sum(dx gate uh)    dscale = w_post sum(dx gate uh)
// HBM-bound: every tensor is read or written once. x' is formed again in the backward pass from x and u (the same bytes as reading
// it, and exactly the forward's fp32 value rather than its rounded copy), the row statistics are two floats a row.
// A row is owned by `tpr` threads (64: one wavefront, no barrier; up to 512 for wide rows) that keep it in registers between the
// two reductions, with their share of the weights beside it: blocks walk many rows, so the weights are read once a block. The
// weight gradients' column sums accumulate in registers over a block's rows and are joined by a second launch in a fixed order.
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
constexpr int MAXB = 1024;         // blocks of the backward kernel (and partial rows the second launch sums)

template <typename T, int VEC> struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) word { T d[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ word<T, VEC> ldw(const T* p) { return *reinterpret_cast<const word<T, VEC>*>(p); }

struct NormArgs {
    const void *x, *u, *gate; const float *scale, *w_post, *w_next;
    void *xo, *z; float *ru, *rx;
    const void *dxo, *dz; void *dx, *du, *dgate; float *partE, *partF;
    long rows, T; int D, gmode, tpr, S, items; float eps;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// sum over the row's threads, the same value (and bits) in all of them. `slot` alternates so that one barrier a reduction suffices:
// a slot is written again only behind the barrier of the reduction in between.
__device__ __forceinline__ float row_sum(float v, int tpr, float (*red)[8], int& slot) {
    v = wave_sum(v);
    if (tpr == 64) return v;
    const int nw = tpr >> 6;
    if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < nw; ++w) v += red[slot][w];
    slot ^= 1;
    return v;
}

template <int VEC, int NV> struct Cols {
    float s[NV * VEC], wp[NV * VEC], wn[NV * VEC];
    __device__ __forceinline__ void load(const NormArgs& a, int lr) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * a.tpr + lr) * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const bool in = c < a.D;
                s[j * VEC + k] = in && a.scale ? a.scale[c + k] : 1.f;
                wp[j * VEC + k] = in && a.w_post ? a.w_post[c + k] : 0.f;
                wn[j * VEC + k] = in && a.w_next ? a.w_next[c + k] : 0.f;
            }
        }
    }
};
template <typename T, int VEC, int NV> struct Row {
    word<T, VEC> r[NV];
    __device__ __forceinline__ void load(const void* p, long off, const NormArgs& a, int lr, bool on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * a.tpr + lr) * VEC;
            if (on && c < a.D) r[j] = ldw<T, VEC>((const T*)p + off + c);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) elem<T>::st(&r[j].d[k], 0.f);
        }
    }
    __device__ __forceinline__ float at(int i) const { return elem<T>::ld(&r[i / VEC].d[i % VEC]); }
};
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(void* p, long off, const float* v, const NormArgs& a, int lr, bool on) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * a.tpr + lr) * VEC;
        if (on && c < a.D) {
            word<T, VEC> w;
#pragma unroll
            for (int k = 0; k < VEC; ++k) elem<T>::st(&w.d[k], v[j * VEC + k]);
            *reinterpret_cast<word<T, VEC>*>((T*)p + off + c) = w;
        }
    }
}
__device__ __forceinline__ long gate_off(const NormArgs& a, long row) { return (a.gmode == 2 ? row / a.T : row) * a.D; }
// the residual sum, its roundings pinned: forward and backward form the same x'
__device__ __forceinline__ float residual(float x, float s, float g, float wp, float uh) { return __fmaf_rn(__fmul_rn(__fmul_rn(s, g), wp), uh, x); }

template <typename XT, typename UT, int VEC, int NV>
__global__ __launch_bounds__(512) void norm_fwd_kernel(NormArgs a) {
    __shared__ float red[2][8];
    constexpr int E = NV * VEC;
    const int lr = threadIdx.x % a.tpr, rid = threadIdx.x / a.tpr, rpb = blockDim.x / a.tpr;
    const float inv = 1.f / (float)a.D;
    int slot = 0;
    Cols<VEC, NV> w;
    w.load(a, lr);
    for (long row0 = (long)blockIdx.x * rpb; row0 < a.rows; row0 += (long)gridDim.x * rpb) {
        const long row = row0 + rid;
        const bool on = row < a.rows;
        Row<XT, VEC, NV> x;
        Row<UT, VEC, NV> u, g;
        x.load(a.x, row * a.D, a, lr, on);
        float x1[E];
        if (a.u) {
            u.load(a.u, row * a.D, a, lr, on);
            if (a.gmode) g.load(a.gate, on ? gate_off(a, row) : 0, a, lr, on);
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) q = __fmaf_rn(u.at(i), u.at(i), q);
            const float ru = rsqrtf(row_sum(q, a.tpr, red, slot) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = residual(x.at(i), w.s[i], a.gmode ? g.at(i) : 1.f, w.wp[i], __fmul_rn(u.at(i), ru));
            store_row<XT, VEC, NV>(a.xo, row * a.D, x1, a, lr, on);
            if (on && lr == 0) a.ru[row] = ru;
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = x.at(i);
        }
        if (a.w_next) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) q = __fmaf_rn(x1[i], x1[i], q);
            const float rx = rsqrtf(row_sum(q, a.tpr, red, slot) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = x1[i] * rx * w.wn[i];
            store_row<UT, VEC, NV>(a.z, row * a.D, x1, a, lr, on);
            if (on && lr == 0) a.rx[row] = rx;
        }
    }
}

// items: with a gate a sample, (sample, segment) pairs of consecutive rows - E is kept apart for each; otherwise one item a block,
// its rows a grid apart
template <typename XT, typename UT, int VEC, int NV>
__global__ __launch_bounds__(512) void norm_bwd_kernel(NormArgs a) {
    __shared__ float red[2][8];
    __shared__ float fold[NV * VEC == 8 ? 64 * 4 * 8 : 1];      // (several rows a block only at 8 values a thread)
    constexpr int E = NV * VEC;
    const int lr = threadIdx.x % a.tpr, rid = threadIdx.x / a.tpr, rpb = blockDim.x / a.tpr;
    const float inv = 1.f / (float)a.D;
    int slot = 0;
    Cols<VEC, NV> w;
    w.load(a, lr);
    float accE[E], accF[E];
#pragma unroll
    for (int i = 0; i < E; ++i) accF[i] = 0.f;
    // block sums of a per-thread column share -> dst (the rows of a block with one wavefront a row are joined in LDS, in order)
    auto flush = [&](const float* acc, float* dst) {
        float v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = acc[i];
        if (E == 8 && rpb > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i) fold[(rid * E + i) * 64 + lr] = acc[i];
            __syncthreads();
            if (rid) return;
            for (int r = 1; r < rpb; ++r)
#pragma unroll
                for (int i = 0; i < E; ++i) v[i] += fold[(r * E + i) * 64 + lr];
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * a.tpr + lr) * VEC;
            if (c < a.D)
#pragma unroll
                for (int k = 0; k < VEC; ++k) dst[c + k] = v[j * VEC + k];
        }
    };
    for (int item = blockIdx.x; item < a.items; item += gridDim.x) {
        long lo = (long)item * rpb, hi = a.rows, step = (long)gridDim.x * rpb;
        if (a.gmode == 2) {
            const long b = item / a.S, seg = item % a.S, per = (a.T + a.S - 1) / a.S;
            lo = b * a.T + min(seg * per, a.T);
            hi = b * a.T + min((seg + 1) * per, a.T);
            step = rpb;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) accE[i] = 0.f;
        for (long row0 = lo; row0 < hi; row0 += step) {
            const long row = row0 + rid;
            const bool on = row < hi;
            Row<XT, VEC, NV> x, dxo;
            Row<UT, VEC, NV> u, g, dz;
            float x1[E], uh[E], dx[E], ru = 0.f;
            x.load(a.x, row * a.D, a, lr, on);
            if (a.dxo) dxo.load(a.dxo, row * a.D, a, lr, on);
            if (a.dz) dz.load(a.dz, row * a.D, a, lr, on);
            if (a.u) {
                u.load(a.u, row * a.D, a, lr, on);
                if (a.gmode) g.load(a.gate, on ? gate_off(a, row) : 0, a, lr, on);
                ru = on ? a.ru[row] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x1[i] = x.at(i);
                if (a.u) {
                    uh[i] = __fmul_rn(u.at(i), ru);
                    x1[i] = residual(x1[i], w.s[i], a.gmode ? g.at(i) : 1.f, w.wp[i], uh[i]);
                }
                dx[i] = a.dxo ? dxo.at(i) : 0.f;
            }
            if (a.dz) {
                const float rx = on ? a.rx[row] : 0.f;
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    x1[i] *= rx;
                    q += dz.at(i) * w.wn[i] * x1[i];
                    accF[i] += dz.at(i) * x1[i];
                }
                q = row_sum(q, a.tpr, red, slot) * inv;
#pragma unroll
                for (int i = 0; i < E; ++i) dx[i] += rx * (dz.at(i) * w.wn[i] - x1[i] * q);
            }
            store_row<XT, VEC, NV>(a.dx, row * a.D, dx, a, lr, on);
            if (a.u) {
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float gt = a.gmode ? g.at(i) : 1.f, t = dx[i] * uh[i];
                    accE[i] += a.gmode == 1 ? t * gt : t;
                    x1[i] = t * w.s[i] * w.wp[i];                          // (x1: the gate's gradient from here)
                    dx[i] *= w.s[i] * gt * w.wp[i];
                    q += dx[i] * uh[i];
                }
                if (a.gmode == 1 && a.dgate) store_row<UT, VEC, NV>(a.dgate, row * a.D, x1, a, lr, on);
                q = row_sum(q, a.tpr, red, slot) * inv;
#pragma unroll
                for (int i = 0; i < E; ++i) dx[i] = ru * (dx[i] - uh[i] * q);
                if (a.du) store_row<UT, VEC, NV>(a.du, row * a.D, dx, a, lr, on);
            }
        }
        if (a.partE) flush(accE, a.partE + (long)item * a.D);
    }
    if (a.partF) flush(accF, a.partF + (long)blockIdx.x * a.D);
}

// a gate a sample: E of the sample's segments -> its gradient; the first segment's row becomes gate * E for the sums over samples
template <typename UT>
__global__ __launch_bounds__(256) void norm_gate_kernel(const UT* gate, const float* scale, const float* w_post, float* partE, UT* dgate, int B, int S, int D) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= (long)B * D) return;
    const long b = id / D;
    const int c = (int)(id - b * D);
    float e = 0.f;
    for (int s = 0; s < S; ++s) e += partE[(b * S + s) * D + c];
    if (dgate) elem<UT>::st(dgate + id, e * (scale ? scale[c] : 1.f) * w_post[c]);
    partE[b * S * D + c] = e * elem<UT>::ld(gate + id);
}

// column sums of the partial rows (nE of them strideE rows apart; nF): 32 columns x 32 row lanes a block
__global__ __launch_bounds__(1024) void norm_cols_kernel(const float* partE, int nE, int strideE, const float* partF, int nF, const float* scale,
                                                         const float* w_post, float* dscale, float* dw_post, float* dw_next, int D) {
    __shared__ float sh[32][33];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
    for (int which = 0; which < 2; ++which) {
        const float* part = which ? partF : partE;
        if (!part) continue;
        const int n = which ? nF : nE;
        const long ld = (long)(which ? 1 : strideE) * D;
        float v = 0.f;
        if (c < D)
            for (int r = rl; r < n; r += 32) v += part[r * ld + c];
        __syncthreads();
        sh[rl][cl] = v;
        __syncthreads();
        if (rl == 0 && c < D) {
            v = 0.f;
#pragma unroll
            for (int r = 0; r < 32; ++r) v += sh[r][cl];
            if (which) { if (dw_next) dw_next[c] = v; }
            else {
                if (dw_post) dw_post[c] = v * (scale ? scale[c] : 1.f);
                if (dscale) dscale[c] = v * w_post[c];
            }
        }
    }
}

// 8 elements a load where every row starts at a 16-byte boundary, single elements otherwise
bool vec8(int D, const NormArgs& a) {
    const uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.u | (uintptr_t)a.gate | (uintptr_t)a.xo | (uintptr_t)a.z | (uintptr_t)a.dxo |
                          (uintptr_t)a.dz | (uintptr_t)a.dx | (uintptr_t)a.du | (uintptr_t)a.dgate;
    return D % 8 == 0 && (all & 15) == 0;
}
int tpr_of(int D, int per) {                // threads a row: the fewest wavefronts whose registers hold it
    int t = 64;
    while (t < 512 && (long)t * per < D) t <<= 1;
    return t;
}
int check(const NormArgs& a, int xdt, int udt, int gmode) {
    if (!((xdt == CPCSV_F32 || xdt == CPCSV_BF16) && (udt == CPCSV_F32 || udt == CPCSV_BF16)) || (xdt == CPCSV_BF16 && udt == CPCSV_F32)) return -1001;
    if (a.rows <= 0 || a.D <= 0 || a.D > CPCSV_NORM_MAX_D || gmode < 0 || gmode > 2 || (gmode == 2 && (a.T <= 0 || a.rows % a.T))) return -1002;
    if (!a.x || (a.u && !a.w_post) || (gmode && (!a.gate || !a.u)) || (!a.u && !a.w_next)) return -1003;
    return 0;
}
int segments(long B, long T) { return B >= MAXB ? 1 : (int)min((MAXB + B - 1) / B, T); }

template <typename XT, typename UT>
void launch(NormArgs& a, bool bwd, hipStream_t st, int& blocks) {
    const bool v8 = vec8(a.D, a);
    const int per = a.D <= 4096 ? 8 : (a.D <= 8192 ? 16 : 32);
    a.tpr = tpr_of(a.D, per);
    const int threads = a.tpr == 64 ? 256 : a.tpr, rpb = threads / a.tpr;
    if (!bwd) blocks = (int)min((a.rows + rpb - 1) / rpb, (long)MAXB * 1024 / threads);
    else {
        if (a.gmode != 2) a.items = (int)min((a.rows + rpb - 1) / rpb, (long)MAXB);
        blocks = min(a.items, MAXB);
    }
#define GO(V, N) (bwd ? norm_bwd_kernel<XT, UT, V, N><<<blocks, threads, 0, st>>>(a) : norm_fwd_kernel<XT, UT, V, N><<<blocks, threads, 0, st>>>(a))
    if (v8) per == 8 ? GO(8, 1) : per == 16 ? GO(8, 2) : GO(8, 4);
    else per == 8 ? GO(1, 8) : per == 16 ? GO(1, 16) : GO(1, 32);
#undef GO
}
void dispatch(NormArgs& a, int xdt, int udt, bool bwd, hipStream_t st, int& blocks) {
    if (xdt == CPCSV_F32 && udt == CPCSV_F32) launch<float, float>(a, bwd, st, blocks);
    else if (xdt == CPCSV_F32) launch<float, bf16_t>(a, bwd, st, blocks);
    else launch<bf16_t, bf16_t>(a, bwd, st, blocks);
}
}  // namespace

extern "C" int cpcsv_norm_residual_fwd(const void* x, const void* u, const void* gate, const float* scale, const float* w_post, const float* w_next,
                                       void* xo, void* z, float* ru, float* rx, long rows, int D, int xdt, int udt, int gate_mode, long T, float eps,
                                       void* stream) {
    NormArgs a{};
    a.x = x; a.u = u; a.gate = gate; a.scale = scale; a.w_post = w_post; a.w_next = w_next; a.xo = xo; a.z = z; a.ru = ru; a.rx = rx;
    a.rows = rows; a.D = D; a.gmode = gate_mode; a.T = T; a.eps = eps;
    if (int rc = check(a, xdt, udt, gate_mode)) return rc;
    if ((u && (!xo || !ru)) || (w_next && (!z || !rx))) return -1003;
    int blocks = 0;
    dispatch(a, xdt, udt, false, (hipStream_t)stream, blocks);
    CPCSV_CHECK_LAUNCH();
    return 0;
}

extern "C" long cpcsv_norm_residual_part(long rows, int D, int gate_mode, long T) {
    if (rows <= 0 || D <= 0) return 0;
    const long B = gate_mode == 2 && T > 0 ? rows / T : 0;
    return (B + 2L * MAXB) * D;
}

extern "C" int cpcsv_norm_residual_bwd(const void* x, const void* u, const void* gate, const float* scale, const float* w_post, const float* w_next,
                                       const float* ru, const float* rx, const void* dxo, const void* dz, void* dx, void* du, void* dgate,
                                       float* dscale, float* dw_post, float* dw_next, float* part, long rows, int D, int xdt, int udt, int gate_mode,
                                       long T, void* stream) {
    NormArgs a{};
    a.x = x; a.u = u; a.gate = gate; a.scale = scale; a.w_post = w_post; a.w_next = w_next; a.ru = (float*)ru; a.rx = (float*)rx;
    a.dxo = dxo; a.dz = w_next ? dz : nullptr; a.dx = dx; a.du = u ? du : nullptr; a.dgate = gate_mode ? dgate : nullptr;
    a.rows = rows; a.D = D; a.gmode = gate_mode; a.T = T;
    if (int rc = check(a, xdt, udt, gate_mode)) return rc;
    const bool needE = u && (dscale || dw_post || (gate_mode == 2 && dgate)), needF = dw_next && a.dz;
    if (!dx || (u && !ru) || (a.dz && !rx) || ((needE || needF) && !part)) return -1003;
    const long B = gate_mode == 2 ? rows / T : 0;
    if (gate_mode == 2) { a.S = segments(B, T); a.items = (int)(B * a.S); }
    const long itemsMax = gate_mode == 2 ? B * a.S : MAXB;
    if (needE) a.partE = part;
    if (needF) a.partF = part + itemsMax * D;
    hipStream_t st = (hipStream_t)stream;
    int blocks = 0;
    dispatch(a, xdt, udt, true, st, blocks);
    CPCSV_CHECK_LAUNCH();
    if (needE && gate_mode == 2) {
        const int n = cdiv(B * D, 256);
        if (udt == CPCSV_F32) norm_gate_kernel<float><<<n, 256, 0, st>>>((const float*)gate, scale, w_post, part, (float*)dgate, (int)B, a.S, D);
        else norm_gate_kernel<bf16_t><<<n, 256, 0, st>>>((const bf16_t*)gate, scale, w_post, part, (bf16_t*)dgate, (int)B, a.S, D);
        CPCSV_CHECK_LAUNCH();
    }
    if ((needE && (dscale || dw_post)) || needF) {
        norm_cols_kernel<<<cdiv(D, 32), 1024, 0, st>>>(a.partE, gate_mode == 2 ? (int)B : blocks, gate_mode == 2 ? a.S : 1, a.partF, blocks,
                                                       scale, w_post, dscale, dw_post, dw_next, D);
        CPCSV_CHECK_LAUNCH();
    }
    return 0;
}
