// scan.hip — gated linear recurrence over a packed projection p = [f | v | o] (three column blocks of H; two without an output gate):
//     z_t = sigmoid(f_t)     h_t = z_t h_{t-1} + (1 - z_t) v_t     y_t = h_t silu(o_t)
// and its gradients. With D_t = dL/dh_t (every later use included) and C_t = z_t D_t:
//     D_t = dy_t silu(o_t) + C_{t+1}      dv_t = (1 - z_t) D_t      df_t = D_t (h_{t-1} - v_t) z_t (1 - z_t)
//     do_t = dy_t h_t silu'(o_t)          dh_0 = C_1
// Both directions are first-order linear recurrences with a coefficient per token and channel, so a run of tokens acts on what
// enters it as an affine map (A = product of its z, plus what it leaves from zero): a long time axis is cut into chunks of CH
// tokens whose maps are formed independently, joined, and applied. 1 - z is sigmoid(-f), not a difference: it keeps its relative
// accuracy where the gate is nearly closed or open.
//
// A thread owns the VEC channels of one 4-byte word and one chunk: the chunk's words of every operand sit in registers (all
// loads issued before the first use), the recurrence runs over them. States, maps and their products are fp32 whatever the
// storage type. No atomics: every sum has one order.
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
constexpr int CH = 32;      // tokens per chunk
constexpr int TB = 256;

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) word { T d[VEC]; };

struct Gate { float s, c; };                                   // sigmoid(x), sigmoid(-x)
__device__ __forceinline__ Gate gate_of(float x) {
    const float e = __expf(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
    return x >= 0.f ? Gate{r, q} : (x < 0.f ? Gate{q, r} : Gate{x, x});          // (NaN stays NaN)
}

// one step of the recurrence, its roundings pinned (no contraction choices): a sequence read token by token, in one call, or run
// again by the backward kernel has the same bits wherever the chunks fall alike
__device__ __forceinline__ float advance(const Gate& z, float h, float v) { return __fmaf_rn(z.s, h, __fmul_rn(z.c, v)); }

struct Dims { int B, T, H, G, NC; long sb, st; const int* len; };

struct Item { int b, c, ch, t0, n; bool ok; };                 // n = tokens of the chunk that are alive
template <int VEC, int L>
__device__ __forceinline__ Item item_of(const Dims& d) {
    Item it;
    const long id = (long)blockIdx.x * TB + threadIdx.x, rest = id / d.G;
    it.ch = (int)(id - rest * d.G) * VEC;
    it.b = (int)(rest / d.NC);
    it.c = (int)(rest - (long)it.b * d.NC);
    it.ok = it.b < d.B;
    it.t0 = it.c * L;
    int len = d.T;
    if (it.ok && d.len) len = min(max(d.len[it.b], 0), d.T);
    it.n = min(max(len - it.t0, 0), L);
    return it;
}

template <typename T, int VEC, int L, bool FULL>
__device__ __forceinline__ void load_rows(word<T, VEC>* r, const T* p, long st, int n) {
#pragma unroll
    for (int i = 0; i < L; ++i)
        if (FULL || i < n) r[i] = *reinterpret_cast<const word<T, VEC>*>(p + i * st);
}

// ---- forward --------------------------------------------------------------------------------------------------------
// the chunk's map: A = prod z, Hl = state left from zero
template <typename T, int VEC, bool FULL>
__device__ __forceinline__ void fwd_map(const T* p, long st, int H, int n, float* A, float* Hl) {
    word<T, VEC> f[CH], v[CH];
    load_rows<T, VEC, CH, FULL>(f, p, st, n);
    load_rows<T, VEC, CH, FULL>(v, p + H, st, n);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (!FULL && i >= n) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
            A[k] *= z.s;
            Hl[k] = advance(z, Hl[k], elem<T>::ld(&v[i].d[k]));
        }
    }
}

template <typename T, int VEC>
__global__ __launch_bounds__(TB) void scan_map_kernel(const T* __restrict__ p, float* __restrict__ sA, float* __restrict__ sH, Dims d) {
    const Item it = item_of<VEC, CH>(d);
    if (!it.ok) return;
    float A[VEC], Hl[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) { A[k] = 1.f; Hl[k] = 0.f; }
    const T* q = p + it.b * d.sb + it.t0 * d.st + it.ch;
    if (it.n == CH) fwd_map<T, VEC, true>(q, d.st, d.H, it.n, A, Hl);
    else fwd_map<T, VEC, false>(q, d.st, d.H, it.n, A, Hl);
    const long o = ((long)it.b * d.NC + it.c) * d.H + it.ch;
#pragma unroll
    for (int k = 0; k < VEC; ++k) { sA[o + k] = A[k]; sH[o + k] = Hl[k]; }
}

// joins the maps of a channel: sH[c] becomes what ENTERS chunk c (c ascending, or descending for the backward direction), `last`
// what leaves the final one
__global__ __launch_bounds__(64) void scan_join_kernel(const float* __restrict__ sA, float* __restrict__ sH, const float* __restrict__ first,
                                                       float* __restrict__ last, int B, int NC, int H, int reverse) {
    const long id = (long)blockIdx.x * 64 + threadIdx.x;
    if (id >= (long)B * H) return;
    const int b = (int)(id / H), ch = (int)(id - (long)b * H);
    float h = first ? first[id] : 0.f;
    const long base = (long)b * NC * H + ch;
    constexpr int U = 16;
    for (int c0 = 0; c0 < NC; c0 += U) {
        float a[U], x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int c = reverse ? NC - 1 - (c0 + i) : c0 + i;
            const bool in = c0 + i < NC;
            a[i] = in ? sA[base + (long)c * H] : 1.f;
            x[i] = in ? sH[base + (long)c * H] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int c = reverse ? NC - 1 - (c0 + i) : c0 + i;
            if (c0 + i < NC) {
                sH[base + (long)c * H] = h;
                h = a[i] * h + x[i];
            }
        }
    }
    if (last) last[id] = h;
}

template <typename T, int VEC, int L, bool GATE, bool FULL>
__device__ __forceinline__ void fwd_apply(const T* p, long st, int H, int n, float* h, T* y, int rows) {
    word<T, VEC> f[L], v[L], o[GATE ? L : 1];
    load_rows<T, VEC, L, FULL>(f, p, st, n);
    load_rows<T, VEC, L, FULL>(v, p + H, st, n);
    if (GATE) load_rows<T, VEC, L, FULL>(o, p + 2 * (long)H, st, n);
#pragma unroll
    for (int i = 0; i < L; ++i) {
        if (!FULL && i >= rows) continue;
        word<T, VEC> out;
        if (FULL || i < n) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                h[k] = advance(z, h[k], elem<T>::ld(&v[i].d[k]));
                float r = h[k];
                if (GATE) {
                    const float g = elem<T>::ld(&o[i].d[k]);
                    r = __fmul_rn(r, __fmul_rn(g, gate_of(g).s));
                }
                elem<T>::st(&out.d[k], r);
            }
        } else {                                               // behind the story's end: zeros, the state stays
#pragma unroll
            for (int k = 0; k < VEC; ++k) elem<T>::st(&out.d[k], 0.f);
        }
        *reinterpret_cast<word<T, VEC>*>(y + (long)i * H) = out;
    }
}

// L = CH: chunk c from its entering state hin (h0 when there is one chunk). L = 1: single tokens (T = 1), h0 may be h_last.
template <typename T, int VEC, int L, bool GATE>
__global__ __launch_bounds__(TB) void scan_apply_kernel(const T* __restrict__ p, const float* h0, const float* __restrict__ hin,
                                                        T* __restrict__ y, float* h_last, Dims d) {
    const Item it = item_of<VEC, L>(d);
    if (!it.ok) return;
    float h[VEC];
    const long so = (long)it.b * d.H + it.ch, ho = ((long)it.b * d.NC + it.c) * d.H + it.ch;
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[k] = hin ? hin[ho + k] : (h0 ? h0[so + k] : 0.f);
    const T* q = p + it.b * d.sb + it.t0 * d.st + it.ch;
    T* yo = y + ((long)it.b * d.T + it.t0) * d.H + it.ch;
    const int rows = min(L, d.T - it.t0);
    if (it.n == L) fwd_apply<T, VEC, L, GATE, true>(q, d.st, d.H, it.n, h, yo, rows);
    else fwd_apply<T, VEC, L, GATE, false>(q, d.st, d.H, it.n, h, yo, rows);
    if (!hin && h_last)
#pragma unroll
        for (int k = 0; k < VEC; ++k) h_last[so + k] = h[k];
}

// ---- backward -------------------------------------------------------------------------------------------------------
template <typename T, int VEC, bool GATE, bool FULL>
__device__ __forceinline__ void bwd_map(const T* p, const T* dy, long st, int H, int n, float* A, float* Cl) {
    word<T, VEC> f[CH], o[GATE ? CH : 1], g[CH];
    load_rows<T, VEC, CH, FULL>(f, p, st, n);
    if (GATE) load_rows<T, VEC, CH, FULL>(o, p + 2 * (long)H, st, n);
    load_rows<T, VEC, CH, FULL>(g, dy, H, n);
#pragma unroll
    for (int i = CH - 1; i >= 0; --i) {
        if (!FULL && i >= n) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
            float u = elem<T>::ld(&g[i].d[k]);
            if (GATE) {
                const float x = elem<T>::ld(&o[i].d[k]);
                u *= x * gate_of(x).s;
            }
            A[k] *= z.s;
            Cl[k] = z.s * (Cl[k] + u);
        }
    }
}

template <typename T, int VEC, bool GATE>
__global__ __launch_bounds__(TB) void scan_bwd_map_kernel(const T* __restrict__ p, const T* __restrict__ dy, float* __restrict__ sA,
                                                          float* __restrict__ sC, Dims d) {
    const Item it = item_of<VEC, CH>(d);
    if (!it.ok) return;
    float A[VEC], Cl[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) { A[k] = 1.f; Cl[k] = 0.f; }
    const T* q = p + it.b * d.sb + it.t0 * d.st + it.ch;
    const T* g = dy + ((long)it.b * d.T + it.t0) * d.H + it.ch;
    if (it.n == CH) bwd_map<T, VEC, GATE, true>(q, g, d.st, d.H, it.n, A, Cl);
    else bwd_map<T, VEC, GATE, false>(q, g, d.st, d.H, it.n, A, Cl);
    const long o = ((long)it.b * d.NC + it.c) * d.H + it.ch;
#pragma unroll
    for (int k = 0; k < VEC; ++k) { sA[o + k] = A[k]; sC[o + k] = Cl[k]; }
}

// h of the chunk is run again from its entering state (kept in registers), then the chunk is walked backwards
template <typename T, int VEC, bool GATE, bool FULL>
__device__ __forceinline__ void bwd_apply(const T* p, const T* dy, long st, int H, int n, float* h, float* C, T* dp, int rows) {
    constexpr int K = GATE ? 3 : 2;
    word<T, VEC> f[CH], v[CH], o[GATE ? CH : 1], g[CH];
    load_rows<T, VEC, CH, FULL>(f, p, st, n);
    load_rows<T, VEC, CH, FULL>(v, p + H, st, n);
    if (GATE) load_rows<T, VEC, CH, FULL>(o, p + 2 * (long)H, st, n);
    load_rows<T, VEC, CH, FULL>(g, dy, H, n);
    float before[CH][VEC];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (!FULL && i >= n) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
            before[i][k] = h[k];
            h[k] = advance(z, h[k], elem<T>::ld(&v[i].d[k]));
        }
    }
#pragma unroll
    for (int i = CH - 1; i >= 0; --i) {
        if (!FULL && i >= rows) continue;
        word<T, VEC> wf, wv, wo;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            float df = 0.f, dv = 0.f, dO = 0.f;
            if (FULL || i < n) {
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                const float gy = elem<T>::ld(&g[i].d[k]);
                float u = gy;
                if (GATE) {
                    const float x = elem<T>::ld(&o[i].d[k]);
                    const Gate s = gate_of(x);
                    u *= x * s.s;
                    dO = gy * h[k] * s.s * (1.f + x * s.c);
                }
                const float D = u + C[k];
                dv = D * z.c;
                C[k] = D * z.s;
                df = C[k] * z.c * (before[i][k] - elem<T>::ld(&v[i].d[k]));
                h[k] = before[i][k];
            }
            elem<T>::st(&wf.d[k], df);
            elem<T>::st(&wv.d[k], dv);
            elem<T>::st(&wo.d[k], dO);
        }
        T* row = dp + (long)i * K * H;
        *reinterpret_cast<word<T, VEC>*>(row) = wf;
        *reinterpret_cast<word<T, VEC>*>(row + H) = wv;
        if (GATE) *reinterpret_cast<word<T, VEC>*>(row + 2 * (long)H) = wo;
    }
}

template <typename T, int VEC, bool GATE>
__global__ __launch_bounds__(TB) void scan_bwd_apply_kernel(const T* __restrict__ p, const T* __restrict__ dy, const float* __restrict__ h0,
                                                            const float* __restrict__ hin, const float* __restrict__ dh_last,
                                                            const float* __restrict__ cin, T* __restrict__ dp, float* __restrict__ dh0, Dims d) {
    const Item it = item_of<VEC, CH>(d);
    if (!it.ok) return;
    float h[VEC], C[VEC];
    const long so = (long)it.b * d.H + it.ch, ho = ((long)it.b * d.NC + it.c) * d.H + it.ch;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        h[k] = hin ? hin[ho + k] : (h0 ? h0[so + k] : 0.f);
        C[k] = cin ? cin[ho + k] : (dh_last ? dh_last[so + k] : 0.f);
    }
    const T* q = p + it.b * d.sb + it.t0 * d.st + it.ch;
    const long row = (long)it.b * d.T + it.t0;
    T* out = dp + row * (GATE ? 3 : 2) * d.H + it.ch;
    const int rows = min(CH, d.T - it.t0);
    if (it.n == CH) bwd_apply<T, VEC, GATE, true>(q, dy + row * d.H + it.ch, d.st, d.H, it.n, h, C, out, rows);
    else bwd_apply<T, VEC, GATE, false>(q, dy + row * d.H + it.ch, d.st, d.H, it.n, h, C, out, rows);
    if (!cin && dh0)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dh0[so + k] = C[k];
}

template <typename T, int VEC, bool GATE>
int run_fwd(const T* p, const float* h0, T* y, float* h_last, float* hin, float* sA, const Dims& d, hipStream_t st) {
    const int blocks = cdiv((long)d.B * d.NC * d.G, TB);
    if (d.T == 1) {
        scan_apply_kernel<T, VEC, 1, GATE><<<blocks, TB, 0, st>>>(p, h0, nullptr, y, h_last, d);
    } else if (d.NC == 1) {
        scan_apply_kernel<T, VEC, CH, GATE><<<blocks, TB, 0, st>>>(p, h0, nullptr, y, h_last, d);
    } else {
        scan_map_kernel<T, VEC><<<blocks, TB, 0, st>>>(p, sA, hin, d);
        scan_join_kernel<<<cdiv((long)d.B * d.H, 64), 64, 0, st>>>(sA, hin, h0, h_last, d.B, d.NC, d.H, 0);
        scan_apply_kernel<T, VEC, CH, GATE><<<blocks, TB, 0, st>>>(p, h0, hin, y, h_last, d);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}

template <typename T, int VEC, bool GATE>
int run_bwd(const T* p, const float* h0, const float* hin, const T* dy, const float* dh_last, T* dp, float* dh0, float* sA, float* sC,
            const Dims& d, hipStream_t st) {
    const int blocks = cdiv((long)d.B * d.NC * d.G, TB);
    if (d.NC == 1) {
        scan_bwd_apply_kernel<T, VEC, GATE><<<blocks, TB, 0, st>>>(p, dy, h0, nullptr, dh_last, nullptr, dp, dh0, d);
    } else {
        scan_bwd_map_kernel<T, VEC, GATE><<<blocks, TB, 0, st>>>(p, dy, sA, sC, d);
        scan_join_kernel<<<cdiv((long)d.B * d.H, 64), 64, 0, st>>>(sA, sC, dh_last, dh0, d.B, d.NC, d.H, 1);
        scan_bwd_apply_kernel<T, VEC, GATE><<<blocks, TB, 0, st>>>(p, dy, h0, hin, dh_last, sC, dp, dh0, d);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}

bool pairs_ok(int dtype, int H, long sb, long st, const void* a, const void* b, const void* c) {
    return dtype == CPCSV_BF16 && H % 2 == 0 && sb % 2 == 0 && st % 2 == 0 && (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0;
}

int dims_of(Dims& d, int dtype, int B, int T, int H, long sb, long st, const int* len, int vec) {
    if ((dtype != CPCSV_F32 && dtype != CPCSV_BF16) || B <= 0 || T <= 0 || H <= 0) return -1001;
    d = Dims{B, T, H, H / vec, (T + CH - 1) / CH, sb, st, len};
    if ((long)B * d.NC * d.G > (1L << 38)) return -1002;
    return 0;
}
}  // namespace

extern "C" int cpcsv_scan_chunks(int T) { return T > 0 ? (T + CH - 1) / CH : 0; }

extern "C" int cpcsv_scan_fwd(const void* p, int dtype, long psb, long pst, const float* h0, const int* lengths, void* y, float* h_last,
                              float* hin, float* sA, int B, int T, int H, int out_gate, void* stream) {
    const bool two = pairs_ok(dtype, H, psb, pst, p, y, nullptr);
    Dims d;
    if (int rc = dims_of(d, dtype, B, T, H, psb, pst, lengths, two ? 2 : 1)) return rc;
    if (!p || !y || (d.NC > 1 && (!hin || !sA))) return -1003;
    hipStream_t st = (hipStream_t)stream;
#define GO(T_, V) (out_gate ? run_fwd<T_, V, true>((const T_*)p, h0, (T_*)y, h_last, hin, sA, d, st) \
                            : run_fwd<T_, V, false>((const T_*)p, h0, (T_*)y, h_last, hin, sA, d, st))
    if (dtype == CPCSV_F32) return GO(float, 1);
    return two ? GO(bf16_t, 2) : GO(bf16_t, 1);
#undef GO
}

extern "C" int cpcsv_scan_bwd(const void* p, int dtype, long psb, long pst, const float* h0, const int* lengths, const float* hin,
                              const void* dy, const float* dh_last, void* dp, float* dh0, float* sA, float* sC, int B, int T, int H,
                              int out_gate, void* stream) {
    const bool two = pairs_ok(dtype, H, psb, pst, p, dy, dp);
    Dims d;
    if (int rc = dims_of(d, dtype, B, T, H, psb, pst, lengths, two ? 2 : 1)) return rc;
    if (!p || !dy || !dp || (d.NC > 1 && (!hin || !sA || !sC))) return -1003;
    hipStream_t st = (hipStream_t)stream;
#define GO(T_, V) (out_gate ? run_bwd<T_, V, true>((const T_*)p, h0, hin, (const T_*)dy, dh_last, (T_*)dp, dh0, sA, sC, d, st) \
                            : run_bwd<T_, V, false>((const T_*)p, h0, hin, (const T_*)dy, dh_last, (T_*)dp, dh0, sA, sC, d, st))
    if (dtype == CPCSV_F32) return GO(float, 1);
    return two ? GO(bf16_t, 2) : GO(bf16_t, 1);
#undef GO
}
