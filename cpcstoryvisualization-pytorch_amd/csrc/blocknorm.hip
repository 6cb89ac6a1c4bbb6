// blocknorm.hip — the root-mean-square norms before and after a block, fused with the block's gate and residual scale:
//     uh = u ru,  ru = (mean u^2 + eps)^-1/2        x' = x + scale * gate * w_post * uh
//     xh = x' rx, rx = (mean x'^2 + eps)^-1/2       z  = w_next * xh
// (u the block's output, x the residual stream, z the next block's input), and their gradients. With g = dz w_next:
//     dx = dx' + rx (g - xh mean(g xh))             q = dx scale gate w_post       du = ru (q - uh mean(q uh))
//     dgate = dx scale w_post uh    dw_next = sum dz xh    dw_post = scale sum(dx gate uh)    dscale = w_post sum(dx gate uh)
// HBM-bound: every tensor is read or written once (but for spilled registers, below). x' is formed again in the backward pass from x and u (the same bytes as reading
// it, and exactly the forward's fp32 value rather than its rounded copy), the row statistics are two floats a row.
// A row is owned by `tpr` threads (64: one wavefront, no barrier; up to 1024 for wide rows) that keep 8 values each (16 above 8192
// columns) in registers between the two reductions, with their share of the weights beside them: blocks walk many rows, so the weights
// are read once a block, and the next row is loaded before this one's reductions. 32768 rows of 2048 in bf16 with a gate a token:
// forward 135 us, 5.0 TB/s; backward 224 us, 4.8 TB/s (a large copy: 4.9 to 5.4). 8192 rows of 8192, an fp32 stream: 182 and 289 us,
// 4.4 and 4.2 TB/s.
// One bound of 1024 threads a block serves all widths: 128 registers, and the backward kernel needs more. Only its 16-byte bf16 form of
// 8 values has no scratch; bytes a lane elsewhere: 16-byte rows up to 8192 columns 28 (fp32 stream, bf16 branch) and 120 (all fp32), odd
// rows 64 to 132, rows above 8192 columns 188 to 308, odd ones 632 to 744 (their forward 8 to 72). What that costs, both ways, no gate,
// against the bytes at 5.0 TB/s: 32768 x 2048 in fp32 583 us and 537; 12276 x 365 53 to 65 and 18 to 36 (value-by-value loads too);
// 8192 x 12288 1080 to 1490 and 400 to 810; 8192 x 16384 1260 to 1750 and 540 to 1070; 2048 x 16383 860 to 960 and 130 to 270.
// Squares are summed in fp32: entries above about 1e17 leave its range (1/rms becomes 0), as do rows below 1e-19 if eps is 0.
// The weight gradients' column sums accumulate in registers over a block's rows and are joined by a second launch (8 us) in a fixed
// order.
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
constexpr int MAXB = 1024;         // blocks of the backward kernel (and partial rows the second launch sums)

template <typename T, int VEC> struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) word { T d[VEC]; };
template <typename T, int VEC> __device__ __forceinline__ word<T, VEC> ldw(const T* p) { return *reinterpret_cast<const word<T, VEC>*>(p); }
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
template <typename T, int VEC> __device__ __forceinline__ void stw(T* p, const float* v) {
    word<T, VEC> w;
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {            // (one conversion of two values, rounded to nearest even)
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
            const bf16x2 r = __builtin_convertvector((f32x2{v[k], v[k + 1]}), bf16x2);
            __builtin_memcpy(&w.d[k], &r, 4);
        }
    } else
#pragma unroll
        for (int k = 0; k < VEC; ++k) elem<T>::st(&w.d[k], v[k]);
    *reinterpret_cast<word<T, VEC>*>(p) = w;
}

struct NormArgs {
    const void *x, *u, *gate; const float *scale, *w_post, *w_next;
    void *xo, *z; float *ru, *rx;
    const void *dxo, *dz; void *dx, *du, *dgate; float *partE, *partF, *partE0;
    long rows, T; int D, gmode, tpr, S, items; float eps;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// sum over the row's threads, the same value (and bits) in all of them. `slot` alternates so that one barrier a reduction suffices:
// a slot is written again only behind the barrier of the reduction in between.
__device__ __forceinline__ float row_sum(float v, int tpr, float (*red)[16], int& slot) {
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

template <int VEC, int NV> struct Cols {            // f = scale w_post
    float f[NV * VEC], wn[NV * VEC];
    __device__ __forceinline__ void load(const NormArgs& a, int lr) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * a.tpr + lr) * VEC;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const bool in = c < a.D;
                f[j * VEC + k] = in && a.w_post ? __fmul_rn(a.scale ? a.scale[c + k] : 1.f, a.w_post[c + k]) : 0.f;
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
            const unsigned c = (j * a.tpr + lr) * VEC;
            if (on && c < (unsigned)a.D) r[j] = ldw<T, VEC>((const T*)p + off + c);
            else
#pragma unroll
                for (int k = 0; k < VEC; ++k) elem<T>::st(&r[j].d[k], 0.f);
        }
    }
    __device__ __forceinline__ float at(int i) const { return elem<T>::ld(&r[i / VEC].d[i % VEC]); }
    // what was unpacked so far is not kept: unpacking 16-bit values again costs an instruction, holding them unpacked a register each
    __device__ __forceinline__ void forget() {
        if constexpr (sizeof(T) == 2 && VEC == 8)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                u32x4 w;
                __builtin_memcpy(&w, &r[j], 16);
                asm volatile("" : "+v"(w));
                __builtin_memcpy(&r[j], &w, 16);
            }
    }
};
template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(void* p, long off, const float* v, const NormArgs& a, int lr, bool on) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const unsigned c = (j * a.tpr + lr) * VEC;
        if (on && c < (unsigned)a.D) stw<T, VEC>((T*)p + off + c, v + j * VEC);
    }
}
__device__ __forceinline__ long gate_off(const NormArgs& a, long row) { return (a.gmode == 2 ? row / a.T : row) * a.D; }
// the residual sum, its roundings pinned: forward and backward form the same x'
__device__ __forceinline__ float residual(float x, float g, float f, float uh) { return __fmaf_rn(__fmul_rn(g, f), uh, x); }

template <typename XT, typename UT, int VEC, int NV> struct FwdRows {
    Row<XT, VEC, NV> x;
    Row<UT, VEC, NV> u, g;
    __device__ __forceinline__ void load(const NormArgs& a, long row, long end, int lr) {
        const bool on = row < end;
        const long off = on ? row * a.D : 0;
        x.load(a.x, off, a, lr, on);
        if (a.u) u.load(a.u, off, a, lr, on);
        if (a.gmode) g.load(a.gate, on ? gate_off(a, row) : 0, a, lr, on);
    }
};

template <typename XT, typename UT, int VEC, int NV>
__global__ __launch_bounds__(1024) void norm_fwd_kernel(NormArgs a) {
    __shared__ float red[2][16];
    constexpr int E = NV * VEC;
    // (a wavefront lies in one row: its address arithmetic is scalar)
    const int lr = threadIdx.x % a.tpr, rid = __builtin_amdgcn_readfirstlane(threadIdx.x / a.tpr), rpb = blockDim.x / a.tpr;
    const float inv = 1.f / (float)a.D;
    const long step = (long)gridDim.x * rpb;
    int slot = 0;
    constexpr bool AHEAD = E == 8 && VEC == 8;                  // (elsewhere two rows would not fit the registers)
    FwdRows<XT, UT, VEC, NV> cur, next;
    if (AHEAD) cur.load(a, (long)blockIdx.x * rpb + rid, a.rows, lr);
    Cols<VEC, NV> w;
    w.load(a, lr);
    for (long row0 = (long)blockIdx.x * rpb; row0 < a.rows; row0 += step) {
        const long row = row0 + rid;
        const bool on = row < a.rows;
        if (!AHEAD) cur.load(a, row, a.rows, lr);
        else if (row0 + step < a.rows) next.load(a, row + step, a.rows, lr);
        float x1[E];
        if (a.u) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) q = __fmaf_rn(cur.u.at(i), cur.u.at(i), q);
            const float ru = rsqrtf(row_sum(q, a.tpr, red, slot) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = residual(cur.x.at(i), a.gmode ? cur.g.at(i) : 1.f, w.f[i], __fmul_rn(cur.u.at(i), ru));
            store_row<XT, VEC, NV>(a.xo, row * a.D, x1, a, lr, on);
            if (on && lr == 0 && a.ru) a.ru[row] = ru;
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = cur.x.at(i);
        }
        if (a.w_next) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) q = __fmaf_rn(x1[i], x1[i], q);
            const float rx = rsqrtf(row_sum(q, a.tpr, red, slot) * inv + a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x1[i] = x1[i] * rx * w.wn[i];
            store_row<UT, VEC, NV>(a.z, row * a.D, x1, a, lr, on);
            if (on && lr == 0 && a.rx) a.rx[row] = rx;
        }
        if (AHEAD) cur = next;
    }
}

template <typename XT, typename UT, int VEC, int NV> struct BwdRows {
    Row<XT, VEC, NV> x, dxo;
    Row<UT, VEC, NV> u, g, dz;
    float ru, rx;
    __device__ __forceinline__ void load(const NormArgs& a, long row, long end, int lr) {
        const bool on = row < end;
        const long off = on ? row * a.D : 0;
        x.load(a.x, off, a, lr, on);
        if (a.dxo) dxo.load(a.dxo, off, a, lr, on);
        if (a.dz) dz.load(a.dz, off, a, lr, on);
        if (a.u) u.load(a.u, off, a, lr, on);
        if (a.gmode) g.load(a.gate, on ? gate_off(a, row) : 0, a, lr, on);
        ru = on && a.u ? a.ru[row] : 0.f;
        rx = on && a.dz ? a.rx[row] : 0.f;
    }
};

// items: with a gate a sample, (sample, segment) pairs of consecutive rows - E is kept apart for each; otherwise one item a block,
// its rows a grid apart
template <typename XT, typename UT, int VEC, int NV>
__global__ __launch_bounds__(1024) void norm_bwd_kernel(NormArgs a) {
    __shared__ float red[2][16];
    __shared__ float fold[NV * VEC == 8 ? 64 * 4 * 8 : 1];      // (several rows a block only at 8 values a thread)
    constexpr int E = NV * VEC;
    // (a wavefront lies in one row: its address arithmetic is scalar)
    const int lr = threadIdx.x % a.tpr, rid = __builtin_amdgcn_readfirstlane(threadIdx.x / a.tpr), rpb = blockDim.x / a.tpr;
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
        constexpr bool AHEAD = E == 8 && VEC == 8;
        BwdRows<XT, UT, VEC, NV> cur, next;
        if (AHEAD) cur.load(a, lo + rid, hi, lr);
        for (long row0 = lo; row0 < hi; row0 += step) {
            const long row = row0 + rid;
            const bool on = row < hi;
            if (!AHEAD) cur.load(a, row, hi, lr);
            else if (row0 + step < hi) next.load(a, row + step, hi, lr);
            float xh[E], dx[E];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                xh[i] = cur.x.at(i);
                if (a.u) xh[i] = residual(xh[i], a.gmode ? cur.g.at(i) : 1.f, w.f[i], __fmul_rn(cur.u.at(i), cur.ru));
                dx[i] = a.dxo ? cur.dxo.at(i) : 0.f;
            }
            if (a.dz) {
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    xh[i] *= cur.rx;
                    q += cur.dz.at(i) * w.wn[i] * xh[i];
                    accF[i] += cur.dz.at(i) * xh[i];
                }
                cur.dz.forget();
                q = row_sum(q, a.tpr, red, slot) * inv;
#pragma unroll
                for (int i = 0; i < E; ++i) dx[i] += cur.rx * (cur.dz.at(i) * w.wn[i] - xh[i] * q);
            }
            store_row<XT, VEC, NV>(a.dx, row * a.D, dx, a, lr, on);
            cur.u.forget();
            cur.g.forget();
            if (a.u) {
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const float gt = a.gmode ? cur.g.at(i) : 1.f, uh = __fmul_rn(cur.u.at(i), cur.ru), t = dx[i] * uh;
                    accE[i] += a.gmode == 1 ? t * gt : t;
                    xh[i] = t * w.f[i];                                    // (the gate's gradient from here)
                    dx[i] *= gt * w.f[i];
                    q += dx[i] * uh;
                }
                if (a.gmode == 1 && a.dgate) store_row<UT, VEC, NV>(a.dgate, row * a.D, xh, a, lr, on);
                cur.u.forget();
                q = row_sum(q, a.tpr, red, slot) * inv;
#pragma unroll
                for (int i = 0; i < E; ++i) dx[i] = cur.ru * (dx[i] - __fmul_rn(cur.u.at(i), cur.ru) * q);
                if (a.du) store_row<UT, VEC, NV>(a.du, row * a.D, dx, a, lr, on);
            }
            if (AHEAD) cur = next;
        }
        if (a.partE) flush(accE, a.partE + (long)item * a.D);
    }
    if (a.partF) flush(accF, a.partF + (long)blockIdx.x * a.D);
}

// 16 columns x 64 row lanes a block: the sum of n rows of `part` ld values apart, from column c; in the first row lane
__device__ __forceinline__ float column_sum(const float* part, int n, long ld, int c, int D, float (*sh)[17]) {
    const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
    float v = 0.f;
    if (c < D)
        for (int r = rl; r < n; r += 64) v += part[r * ld + c];
    sh[rl][cl] = v;
    __syncthreads();
    v = 0.f;
    if (rl == 0)
#pragma unroll
        for (int r = 0; r < 64; ++r) v += sh[r][cl];
    return v;
}

// a gate a sample: E of the sample's segments -> its gradient; the first segment's row becomes gate * E for the sums over samples
template <typename UT>
__global__ __launch_bounds__(1024) void norm_gate_kernel(const UT* gate, const float* scale, const float* w_post, float* partE, UT* dgate, int S, int D) {
    __shared__ float sh[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15);
    const long b = blockIdx.y;
    const float e = column_sum(partE + b * S * D, S, D, c, D, sh);
    if (threadIdx.x >= 16 || c >= D) return;
    if (dgate) elem<UT>::st(dgate + b * D + c, e * __fmul_rn(scale ? scale[c] : 1.f, w_post[c]));
    partE[b * S * D + c] = e * elem<UT>::ld(gate + b * D + c);
}

// column sums of the partial rows (nE of them strideE rows apart; nF)
__global__ __launch_bounds__(1024) void norm_cols_kernel(const float* partE, int nE, int strideE, const float* partF, int nF, const float* scale,
                                                         const float* w_post, float* dscale, float* dw_post, float* dw_next, int D) {
    __shared__ float sh[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15);
    const bool which = blockIdx.y != 0;
    if (!(which ? partF : partE)) return;
    const float v = column_sum(which ? partF : partE, which ? nF : nE, (long)(which ? 1 : strideE) * D, c, D, sh);
    if (threadIdx.x >= 16 || c >= D) return;
    if (which) { if (dw_next) dw_next[c] = v; }
    else {
        if (dw_post) dw_post[c] = v * (scale ? scale[c] : 1.f);
        if (dscale) dscale[c] = v * w_post[c];
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
    while (t < 1024 && (long)t * per < D) t <<= 1;
    return t;
}
int check(const NormArgs& a, int xdt, int udt, int gmode) {
    if (!((xdt == CPCSV_F32 || xdt == CPCSV_BF16) && (udt == CPCSV_F32 || udt == CPCSV_BF16)) || (xdt == CPCSV_BF16 && udt == CPCSV_F32)) return -1001;
    if (a.rows <= 0 || a.D <= 0 || a.D > CPCSV_NORM_MAX_D || gmode < 0 || gmode > 2 || (gmode == 2 && (a.T <= 0 || a.rows % a.T || a.rows / a.T > (1L << 30))))
        return -1002;
    if (!a.x || (a.u && !a.w_post) || (gmode && (!a.gate || !a.u)) || (!a.u && !a.w_next)) return -1003;
    return 0;
}
template <typename XT, typename UT>
void launch(NormArgs& a, bool bwd, hipStream_t st, int& blocks) {
    const bool v8 = vec8(a.D, a);
    const int per = a.D <= 8192 ? 8 : 16;
    a.tpr = tpr_of(a.D, per);
    const int threads = a.tpr == 64 ? 256 : a.tpr, rpb = threads / a.tpr;
    const long fit = min((long)MAXB, 256L * 1024 / threads);             // blocks that the chip holds at once
    blocks = (int)min((a.rows + rpb - 1) / rpb, fit);
    if (bwd) {
        a.items = blocks;
        if (a.gmode == 2) {
            const long B = a.rows / a.T;
            a.S = B >= fit ? 1 : (int)min((fit + B - 1) / B, a.T);
            a.items = (int)(B * a.S);
            blocks = (int)min((long)a.items, fit);
        }
        if (a.partF) a.partF = a.partE0 + (a.partE ? (long)a.items * a.D : 0);
    }
#define GO(V, N) (bwd ? norm_bwd_kernel<XT, UT, V, N><<<blocks, threads, 0, st>>>(a) : norm_fwd_kernel<XT, UT, V, N><<<blocks, threads, 0, st>>>(a))
    if (v8) per == 8 ? GO(8, 1) : GO(8, 2);
    else per == 8 ? GO(1, 8) : GO(1, 16);
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
    if ((u && !xo) || (w_next && !z)) return -1003;
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
    a.partE0 = part;                          // E's rows (an item each), then F's (a block each)
    if (needE) a.partE = part;
    if (needF) a.partF = part;
    hipStream_t st = (hipStream_t)stream;
    int blocks = 0;
    dispatch(a, xdt, udt, true, st, blocks);
    CPCSV_CHECK_LAUNCH();
    if (needE && gate_mode == 2) {
        for (long b0 = 0; b0 < B; b0 += 65535) {                          // (the grid's second dimension)
            const dim3 n(cdiv(D, 16), (unsigned)min(65535L, B - b0));
            float* e = part + b0 * a.S * D;
            if (udt == CPCSV_F32) norm_gate_kernel<float><<<n, 1024, 0, st>>>((const float*)gate + b0 * D, scale, w_post, e, dgate ? (float*)dgate + b0 * D : nullptr, a.S, D);
            else norm_gate_kernel<bf16_t><<<n, 1024, 0, st>>>((const bf16_t*)gate + b0 * D, scale, w_post, e, dgate ? (bf16_t*)dgate + b0 * D : nullptr, a.S, D);
        }
        CPCSV_CHECK_LAUNCH();
    }
    if ((needE && (dscale || dw_post)) || needF) {
        norm_cols_kernel<<<dim3(cdiv(D, 16), 2), 1024, 0, st>>>(needE ? part : nullptr, gate_mode == 2 ? (int)B : blocks, gate_mode == 2 ? a.S : 1, a.partF, blocks,
                                                       scale, w_post, dscale, dw_post, dw_next, D);
        CPCSV_CHECK_LAUNCH();
    }
    return 0;
}
