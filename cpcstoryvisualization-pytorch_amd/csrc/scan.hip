// scan.hip — gated linear recurrence over a packed projection p = [f | v | o] (three column blocks of H; two without an output gate):
//     z_t = sigmoid(f_t)     h_t = z_t h_{t-1} + (1 - z_t) v_t     y_t = h_t silu(o_t)
// and its gradients. With D_t = dL/dh_t (every later use included) and C_t = z_t D_t:
//     D_t = dy_t silu(o_t) + C_{t+1}      dv_t = (1 - z_t) D_t      df_t = D_t (h_{t-1} - v_t) z_t (1 - z_t)
//     do_t = dy_t h_t silu'(o_t)          dh_0 = C_1
// Both directions are first-order linear recurrences with a coefficient per token and channel, so a run of tokens acts on what
// enters it as an affine map x -> A x + X (A the product of its z). 1 - z is sigmoid(-f), not a difference: it keeps its relative
// accuracy where the gate is nearly closed or open. States, maps and their products are fp32 whatever the storage type.
//
// One pass over the data. A wavefront holds CH tokens of the channels of one 4-byte word a lane in registers, a block a tile of
// several such chunks; the maps of the chunks meet in LDS, those of the tiles in memory: a block publishes its tile's map, reads the
// maps of the tiles before it and applies them IN ORDER, so that a result does not depend on who was ready when. Behind every SB
// tiles the state itself is published and the reading starts there. Tiles are handed out by a counter in the order of the
// recurrence: whatever a block waits for belongs to a block that has started before it and publishes its map without waiting (and,
// by induction over the counter, its state), so every wait ends. A published word is its own flag: 64 (state: 32) bits written and
// read as one, all ones until then; a NaN is published as another pattern.
// Bound by HBM: p, y (dy, dp) once each. 8 x 4096 x 2048 in bf16 (a large copy: 4.9 to 5.4 TB/s): forward 127 us, 4.2 TB/s; backward
// 209 us, 4.5 TB/s; one sequence of 32768 x 2048: 128 us (fp32: 198 us, 5.4 TB/s). Two launches (the words are armed first, 2 to 5 us); T <= SHORT runs as one,
// from start to end in registers, bit for bit what single tokens give (64 x 512, one token: 3 us; 12 x 5 x 365 in fp32: 6 us, both ways
// 12; 64 x 32 x 2048 in bf16: 17 and 41 us for bytes of 7 and 19 at 5.0 TB/s - one thread walks the sequence, latency).
#include "common.h"
#include "../../include/cpcsv_hip.h"

namespace {
constexpr int CH = 16;               // tokens a wavefront holds
constexpr int FW = 8, BW = 4;        // wavefronts (chunks) of a tile, forward and backward: what the registers hold twice on a CU
constexpr int SB = 8;                // tiles between published states (training batch of 8 x 4096 x 2048, both directions: 16 tiles 341 us,
                                     // 8 322, 4 315; but a state has to pass T / (SB tiles) hands, and fewer of them is safer for long T)
constexpr int SHORT = 32;
constexpr int TB = 256;
constexpr int POLLS = 1 << 20;       // of a wait (about a second): a bound that no run comes near

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) word { T d[VEC]; };
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

template <typename T, int VEC> __device__ __forceinline__ void store_word(T* p, const float (&v)[VEC]) {
    word<T, VEC> w;
    if constexpr (sizeof(T) == 2 && VEC == 2) {                // (one conversion of two values, rounded to nearest even)
        const bf16x2 r = __builtin_convertvector((f32x2{v[0], v[1]}), bf16x2);
        __builtin_memcpy(&w, &r, 4);
    } else
#pragma unroll
        for (int k = 0; k < VEC; ++k) elem<T>::st(&w.d[k], v[k]);
    *reinterpret_cast<word<T, VEC>*>(p) = w;
}

struct Gate { float s, c; };                                   // sigmoid(x), sigmoid(-x)
__device__ __forceinline__ Gate gate_of(float x) {
    const float e = __expf(-fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
    return x >= 0.f ? Gate{r, q} : Gate{q, r};
}
// one step of the recurrence, its roundings pinned (no contraction choices): a sequence read token by token, in one call, or run
// again by the backward kernel has the same bits wherever the chunks fall alike
__device__ __forceinline__ float advance(float s, float h, float b) { return __fmaf_rn(s, h, b); }        // b = (1 - z) v, rounded

struct Dims { int B, T, H, G, NT, NCH; long sb, st; const int* len; };
__device__ __forceinline__ int length_of(const Dims& d, int b) { return d.len ? min(max(d.len[b], 0), d.T) : d.T; }

template <typename T, int VEC, int L, bool FULL>
__device__ __forceinline__ void load_rows(word<T, VEC>* r, const T* p, long st, int n) {
#pragma unroll
    for (int i = 0; i < L; ++i)
        if (FULL || i < n) r[i] = *reinterpret_cast<const word<T, VEC>*>(p + i * st);
}

// ---- up to SHORT tokens, single tokens: one thread a word of channels, from start to end ------------------------------
template <typename T, int VEC, int L, bool GATE>
__global__ __launch_bounds__(TB) void scan_short_kernel(const T* __restrict__ p, const float* h0, T* __restrict__ y, float* h_last, Dims d) {
    const long id = (long)blockIdx.x * TB + threadIdx.x;
    const int b = (int)(id / d.G), ch = (int)(id - (long)b * d.G) * VEC;
    if (b >= d.B) return;
    const int n = length_of(d, b);
    const T* q = p + b * d.sb + ch;
    word<T, VEC> f[L], v[L], o[GATE ? L : 1];
    load_rows<T, VEC, L, false>(f, q, d.st, n);
    load_rows<T, VEC, L, false>(v, q + d.H, d.st, n);
    if (GATE) load_rows<T, VEC, L, false>(o, q + 2 * (long)d.H, d.st, n);
    const long so = (long)b * d.H + ch;
    float h[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[k] = h0 ? h0[so + k] : 0.f;
    T* out = y + (long)b * d.T * d.H + ch;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        if (i >= d.T) continue;
        float r[VEC] = {};
        if (i < n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                r[k] = h[k] = advance(z.s, h[k], __fmul_rn(z.c, elem<T>::ld(&v[i].d[k])));
                if (GATE) {
                    const float g = elem<T>::ld(&o[i].d[k]);
                    r[k] = __fmul_rn(r[k], __fmul_rn(g, gate_of(g).s));
                }
            }
        store_word<T, VEC>(out + (long)i * d.H, r);            // (behind the sequence's end: zeros, the state stays)
    }
    if (h_last)
#pragma unroll
        for (int k = 0; k < VEC; ++k) h_last[so + k] = h[k];
}

template <typename T, int VEC, bool GATE>
__global__ __launch_bounds__(TB) void scan_short_bwd_kernel(const T* __restrict__ p, const float* __restrict__ h0, const T* __restrict__ dy,
                                                            const float* __restrict__ dh_last, T* __restrict__ dp, float* __restrict__ dh0, Dims d) {
    constexpr int L = SHORT, K = GATE ? 3 : 2;
    const long id = (long)blockIdx.x * TB + threadIdx.x;
    const int b = (int)(id / d.G), ch = (int)(id - (long)b * d.G) * VEC;
    if (b >= d.B) return;
    const int n = length_of(d, b);
    const T* q = p + b * d.sb + ch;
    word<T, VEC> f[L], v[L], o[GATE ? L : 1], g[L];
    load_rows<T, VEC, L, false>(f, q, d.st, n);
    load_rows<T, VEC, L, false>(v, q + d.H, d.st, n);
    if (GATE) load_rows<T, VEC, L, false>(o, q + 2 * (long)d.H, d.st, n);
    load_rows<T, VEC, L, false>(g, dy + (long)b * d.T * d.H + ch, d.H, n);
    const long so = (long)b * d.H + ch;
    float h[VEC], C[VEC], before[L][VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        h[k] = h0 ? h0[so + k] : 0.f;
        C[k] = dh_last ? dh_last[so + k] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < L; ++i)
        if (i < n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                before[i][k] = h[k];
                h[k] = advance(z.s, h[k], __fmul_rn(z.c, elem<T>::ld(&v[i].d[k])));
            }
    T* out = dp + (long)b * d.T * K * d.H + ch;
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
        if (i >= d.T) continue;
        float df[VEC] = {}, dv[VEC] = {}, dO[VEC] = {};
        if (i < n)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                const float gy = elem<T>::ld(&g[i].d[k]);
                float u = gy;
                if (GATE) {
                    const float x = elem<T>::ld(&o[i].d[k]);
                    const Gate s = gate_of(x);
                    u *= x * s.s;
                    dO[k] = gy * h[k] * s.s * (1.f + x * s.c);
                }
                const float D = u + C[k];
                dv[k] = D * z.c;
                C[k] = D * z.s;
                df[k] = C[k] * z.c * (before[i][k] - elem<T>::ld(&v[i].d[k]));
                h[k] = before[i][k];
            }
        T* row = out + (long)i * K * d.H;
        store_word<T, VEC>(row, df);
        store_word<T, VEC>(row + d.H, dv);
        if (GATE) store_word<T, VEC>(row + 2 * (long)d.H, dO);
    }
    if (dh0)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dh0[so + k] = C[k];
}

// ---- tiles ------------------------------------------------------------------------------------------------------------
struct Look {                        // armed with ones before each use
    unsigned* ticket;
    unsigned* state;                 // [B][tiles / SB][H] what enters the tiles behind each run of SB
    unsigned long long* map;         // [B][tiles][H] {A, X}
};
struct Map { float a, x; };
// A product of gates that underflows is not zero: 0 would turn an infinite state into NaN. It stays at fp32's smallest number instead,
// which adds 2^-149 |h| to a finite state's result: less than 2^-49 for any |h| below 2^100. (A gate that is 0 in fp32, f below about
// -87, is 0: it makes NaN of an infinite state here as token by token.)
constexpr float LEAST = 0x1p-149f;
__device__ __forceinline__ float product(float a, float b) {
    const float r = a * b;
    return r == 0.f && a != 0.f && b != 0.f ? LEAST : r;
}
// of a chunk, whose gates are multiplied without that test; least: the smallest of them
__device__ __forceinline__ float whole_product(float a, float least) { return a == 0.f && least > 0.f ? LEAST : a; }
__device__ __forceinline__ float plain_nan(float v) { return v == v ? v : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ void publish(unsigned long long* p, float a, float x) {
    const unsigned long long w = (unsigned long long)__float_as_uint(plain_nan(a)) | (unsigned long long)__float_as_uint(plain_nan(x)) << 32;
    __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(unsigned* p, float x) {
    __hip_atomic_store(p, __float_as_uint(plain_nan(x)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// the published words of VEC channels (ok: the lane has some); NaN should the wait ever run out
template <int VEC, typename W> __device__ __forceinline__ void await(const W* p, bool ok, W (&w)[VEC]) {
    for (int i = 0; i < POLLS; ++i) {
        bool there = true;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            w[k] = ok ? __hip_atomic_load(p + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : (W)0;
            there = there && w[k] != ~(W)0;
        }
        if (__all(there)) return;
        __builtin_amdgcn_s_sleep(2);
    }
}

__global__ __launch_bounds__(256) void scan_arm_kernel(uint4* w, long n) {
    const long id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id < n) w[id] = uint4{~0u, ~0u, ~0u, ~0u};
}

// What a tile's blocks share, and the state that enters a wavefront's chunk. `tile` counts in the direction of the recurrence, as do
// the wavefronts. Every thread of the block calls it.
template <int W, int VEC> struct Joint {
    Map own[W][64 * VEC], seen[SB][64 * VEC];
    float start[64 * VEC];
    unsigned ticket;

    __device__ __forceinline__ void enter(const Look& lk, const Dims& d, int b, int tile, int ch, bool ok, const float (&A)[VEC], const float (&X)[VEC],
                                          const float* first, float (&h)[VEC]) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, at = lane * VEC, sb0 = tile / SB * SB;
#pragma unroll
        for (int k = 0; k < VEC; ++k) own[w][at + k] = Map{A[k], X[k]};
        __syncthreads();
        Map whole[VEC];
        unsigned long long* const maps = lk.map + (long)b * d.NT * d.H + ch;
        if (w == 0) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                whole[k] = own[0][at + k];
                for (int j = 1; j < W; ++j) {
                    const Map m = own[j][at + k];
                    whole[k] = Map{product(m.a, whole[k].a), __fmaf_rn(m.a, whole[k].x, m.x)};
                }
                if (ok && tile % SB != SB - 1 && tile + 1 < d.NT) publish(maps + (long)tile * d.H + k, whole[k].a, whole[k].x);
            }
        }
        for (int t = sb0 + w; t < tile; t += W) {
            unsigned long long m[VEC];
            await<VEC>(maps + (long)t * d.H, ok, m);
#pragma unroll
            for (int k = 0; k < VEC; ++k) seen[t - sb0][at + k] = Map{__uint_as_float((unsigned)m[k]), __uint_as_float((unsigned)(m[k] >> 32))};
        }
        if (w == W - 1) {
            if (sb0) {
                unsigned m[VEC];
                await<VEC>(lk.state + ((long)b * (d.NT / SB) + sb0 / SB - 1) * d.H + ch, ok, m);
#pragma unroll
                for (int k = 0; k < VEC; ++k) start[at + k] = __uint_as_float(m[k]);
            } else
#pragma unroll
                for (int k = 0; k < VEC; ++k) start[at + k] = first && ok ? first[(long)b * d.H + ch + k] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = start[at + k];
        for (int t = 0; t < tile - sb0; ++t)
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = __fmaf_rn(seen[t][at + k].a, h[k], seen[t][at + k].x);
        if (w == 0 && ok && tile % SB == SB - 1 && tile + 1 < d.NT)
#pragma unroll
            for (int k = 0; k < VEC; ++k) publish(lk.state + ((long)b * (d.NT / SB) + tile / SB) * d.H + ch + k, __fmaf_rn(whole[k].a, h[k], whole[k].x));
        for (int j = 0; j < w; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = __fmaf_rn(own[j][at + k].a, h[k], own[j][at + k].x);
    }
};

// the block's place: tiles in the order of the recurrence, of a tile all rows and channel groups
template <int W, int VEC> __device__ __forceinline__ void place_of(const Look& lk, const Dims& d, unsigned& ticket, int& b, int& tile, int& ch) {
    if (threadIdx.x == 0) ticket = atomicAdd(lk.ticket, 1u) + 1u;
    __syncthreads();
    const unsigned unit = ticket, groups = (unsigned)((d.G + 63) / 64);
    ch = (int)(unit % groups) * 64 * VEC + (int)(threadIdx.x & 63) * VEC;
    b = (int)(unit / groups % (unsigned)d.B);
    tile = (int)(unit / groups / (unsigned)d.B);
}

template <typename T, int VEC, bool GATE>
__global__ __launch_bounds__(FW * 64, 4) void scan_fwd_kernel(const T* __restrict__ p, const float* __restrict__ h0, T* __restrict__ y,
                                                              float* __restrict__ h_last, float* __restrict__ hin, Look lk, Dims d) {
    __shared__ Joint<FW, VEC> sh;
    int b, tile, ch;
    place_of<FW, VEC>(lk, d, sh.ticket, b, tile, ch);
    const bool ok = ch < d.H;
    const int chunk = tile * FW + (threadIdx.x >> 6), t0 = chunk * CH, n = min(max(length_of(d, b) - t0, 0), CH), rows = min(max(d.T - t0, 0), CH);
    float zs[CH][VEC], in[CH][VEC], act[GATE ? CH : 1][VEC], A[VEC], X[VEC], least[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) { A[k] = least[k] = 1.f; X[k] = 0.f; }
    {
        word<T, VEC> f[CH], v[CH], o[GATE ? CH : 1];
        const T* q = p + b * d.sb + t0 * d.st + (ok ? ch : 0);          // (lanes without channels read the row's first and store nothing)
        if (n == CH) {
            load_rows<T, VEC, CH, true>(f, q, d.st, n);
            load_rows<T, VEC, CH, true>(v, q + d.H, d.st, n);
            if (GATE) load_rows<T, VEC, CH, true>(o, q + 2 * (long)d.H, d.st, n);
        } else {
            load_rows<T, VEC, CH, false>(f, q, d.st, n);
            load_rows<T, VEC, CH, false>(v, q + d.H, d.st, n);
            if (GATE) load_rows<T, VEC, CH, false>(o, q + 2 * (long)d.H, d.st, n);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const bool on = i < n;                                   // (behind the end: the identity)
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                zs[i][k] = on ? z.s : 1.f;
                in[i][k] = on ? __fmul_rn(z.c, elem<T>::ld(&v[i].d[k])) : 0.f;
                if (GATE) {
                    const float g = elem<T>::ld(&o[i].d[k]);
                    act[i][k] = on ? __fmul_rn(g, gate_of(g).s) : 0.f;
                }
                A[k] *= zs[i][k];
                least[k] = fminf(least[k], zs[i][k]);
                X[k] = __fmaf_rn(zs[i][k], X[k], in[i][k]);
            }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = whole_product(A[k], least[k]);
    float h[VEC];
    sh.enter(lk, d, b, tile, ch, ok, A, X, h0, h);
    if (!ok || !rows) return;
    if (hin)
#pragma unroll
        for (int k = 0; k < VEC; ++k) hin[((long)b * d.NCH + chunk) * d.H + ch + k] = h[k];
    T* out = y + ((long)b * d.T + t0) * d.H + ch;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (i >= rows) continue;
        float r[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            h[k] = advance(zs[i][k], h[k], in[i][k]);
            r[k] = GATE ? __fmul_rn(h[k], act[i][k]) : (i < n ? h[k] : 0.f);
        }
        store_word<T, VEC>(out + (long)i * d.H, r);
    }
    if (h_last && chunk == d.NCH - 1)
#pragma unroll
        for (int k = 0; k < VEC; ++k) h_last[(long)b * d.H + ch + k] = h[k];
}

// h of the chunk is run again from its entering state; what does not wait for D leaves at once (do), the rest is kept as
// u = dy silu(o), z, 1 - z and z (1 - z) (h_{t-1} - v). Tiles and wavefronts count from the sequence's end.
template <typename T, int VEC, bool GATE>
__global__ __launch_bounds__(BW * 64, 2) void scan_bwd_kernel(const T* __restrict__ p, const float* __restrict__ hin, const T* __restrict__ dy,
                                                              const float* __restrict__ dh_last, T* __restrict__ dp, float* __restrict__ dh0, Look lk, Dims d) {
    constexpr int K = GATE ? 3 : 2;
    __shared__ Joint<BW, VEC> sh;
    int b, tile, ch;
    place_of<BW, VEC>(lk, d, sh.ticket, b, tile, ch);
    const bool ok = ch < d.H;
    const int chunk = (d.NT - 1 - tile) * BW + BW - 1 - (int)(threadIdx.x >> 6), t0 = chunk * CH;
    const int n = min(max(length_of(d, b) - t0, 0), CH), rows = ok ? min(max(d.T - t0, 0), CH) : 0;
    float zs[CH][VEC], zc[CH][VEC], q[CH][VEC], u[CH][VEC], A[VEC], X[VEC], least[VEC];
    const long row0 = (long)b * d.T + t0;
    T* out = dp + row0 * K * d.H + ch;
    {
        word<T, VEC> f[CH], v[CH], o[GATE ? CH : 1], g[CH];
        const T* src = p + b * d.sb + t0 * d.st + (ok ? ch : 0);
        const T* gy = dy + row0 * d.H + (ok ? ch : 0);
        if (n == CH) {
            load_rows<T, VEC, CH, true>(f, src, d.st, n);
            load_rows<T, VEC, CH, true>(v, src + d.H, d.st, n);
            if (GATE) load_rows<T, VEC, CH, true>(o, src + 2 * (long)d.H, d.st, n);
            load_rows<T, VEC, CH, true>(g, gy, d.H, n);
        } else {
            load_rows<T, VEC, CH, false>(f, src, d.st, n);
            load_rows<T, VEC, CH, false>(v, src + d.H, d.st, n);
            if (GATE) load_rows<T, VEC, CH, false>(o, src + 2 * (long)d.H, d.st, n);
            load_rows<T, VEC, CH, false>(g, gy, d.H, n);
        }
        float h[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = n ? hin[((long)b * d.NCH + chunk) * d.H + (ok ? ch : 0) + k] : 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            float dO[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const bool on = i < n;
                const Gate z = gate_of(elem<T>::ld(&f[i].d[k]));
                const float x = elem<T>::ld(&v[i].d[k]), gr = elem<T>::ld(&g[i].d[k]);
                q[i][k] = on ? z.s * z.c * (h[k] - x) : 0.f;
                zs[i][k] = on ? z.s : 1.f;
                zc[i][k] = on ? z.c : 0.f;
                if (on) h[k] = advance(z.s, h[k], __fmul_rn(z.c, x));
                if (GATE) {
                    const float w = elem<T>::ld(&o[i].d[k]);
                    const Gate s = gate_of(w);
                    u[i][k] = on ? gr * (w * s.s) : 0.f;
                    dO[k] = on ? gr * h[k] * s.s * (1.f + w * s.c) : 0.f;
                } else u[i][k] = on ? gr : 0.f;
            }
            if (GATE && i < rows) store_word<T, VEC>(out + (long)i * K * d.H + 2 * (long)d.H, dO);
        }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) { A[k] = least[k] = 1.f; X[k] = 0.f; }
#pragma unroll
    for (int i = CH - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            A[k] *= zs[i][k];
            least[k] = fminf(least[k], zs[i][k]);
            X[k] = zs[i][k] * (X[k] + u[i][k]);
        }
#pragma unroll
    for (int k = 0; k < VEC; ++k) A[k] = whole_product(A[k], least[k]);
    float C[VEC];
    sh.enter(lk, d, b, tile, ch, ok, A, X, dh_last, C);
    // u of a token behind the end is 0, its z 1: C passes it unchanged, as the map says
#pragma unroll
    for (int i = CH - 1; i >= 0; --i) {
        if (i >= rows) continue;
        float df[VEC], dv[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float D = u[i][k] + C[k];
            df[k] = D * q[i][k];
            dv[k] = D * zc[i][k];
            C[k] = D * zs[i][k];
        }
        store_word<T, VEC>(out + (long)i * K * d.H, df);
        store_word<T, VEC>(out + (long)i * K * d.H + d.H, dv);
    }
    if (dh0 && ok && chunk == 0)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dh0[(long)b * d.H + ch + k] = C[k];
}

// ---- host -------------------------------------------------------------------------------------------------------------
int tiles_of(int T, int waves) { return (int)(((long)T + waves * CH - 1) / (waves * CH)); }
// ticket (16 bytes), states, maps: a whole number of 16-byte pieces
long look_bytes(int B, int T, int H, int waves) {
    const long nt = tiles_of(T, waves), st = ((long)B * (nt / SB) * H * 4 + 15) / 16 * 16;
    return 16 + st + ((long)B * nt * H * 8 + 15) / 16 * 16;
}
Look look_of(void* ws, const Dims& d) {
    char* c = (char*)ws;
    return Look{(unsigned*)c, (unsigned*)(c + 16), (unsigned long long*)(c + 16 + ((long)d.B * (d.NT / SB) * d.H * 4 + 15) / 16 * 16)};
}
int arm(void* ws, long bytes, hipStream_t st) {
    scan_arm_kernel<<<cdiv(bytes / 16, 256), 256, 0, st>>>((uint4*)ws, bytes / 16);
    CPCSV_CHECK_LAUNCH();
    return 0;
}

template <typename T, int VEC, bool GATE>
int run_fwd(const T* p, const float* h0, T* y, float* h_last, float* hin, void* ws, Dims d, hipStream_t st) {
    const int blocks = cdiv((long)d.B * d.G, TB);
    if (d.T == 1) scan_short_kernel<T, VEC, 1, GATE><<<blocks, TB, 0, st>>>(p, h0, y, h_last, d);
    else if (d.T <= SHORT) scan_short_kernel<T, VEC, SHORT, GATE><<<blocks, TB, 0, st>>>(p, h0, y, h_last, d);
    else {
        d.NT = tiles_of(d.T, FW);
        if (int rc = arm(ws, look_bytes(d.B, d.T, d.H, FW), st)) return rc;
        scan_fwd_kernel<T, VEC, GATE><<<(unsigned)((long)d.NT * d.B * ((d.G + 63) / 64)), FW * 64, 0, st>>>(p, h0, y, h_last, hin, look_of(ws, d), d);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}

template <typename T, int VEC, bool GATE>
int run_bwd(const T* p, const float* h0, const float* hin, const T* dy, const float* dh_last, T* dp, float* dh0, void* ws, Dims d, hipStream_t st) {
    if (d.T <= SHORT) scan_short_bwd_kernel<T, VEC, GATE><<<cdiv((long)d.B * d.G, TB), TB, 0, st>>>(p, h0, dy, dh_last, dp, dh0, d);
    else {
        d.NT = tiles_of(d.T, BW);
        if (int rc = arm(ws, look_bytes(d.B, d.T, d.H, BW), st)) return rc;
        scan_bwd_kernel<T, VEC, GATE><<<(unsigned)((long)d.NT * d.B * ((d.G + 63) / 64)), BW * 64, 0, st>>>(p, hin, dy, dh_last, dp, dh0, look_of(ws, d), d);
    }
    CPCSV_CHECK_LAUNCH();
    return 0;
}

// two bf16 channels a word where every row starts at a 4-byte boundary, single elements otherwise
bool pairs_ok(int dtype, int H, long sb, long st, const void* a, const void* b, const void* c) {
    return dtype == CPCSV_BF16 && H % 2 == 0 && sb % 2 == 0 && st % 2 == 0 && (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 3) == 0;
}
int dims_of(Dims& d, int dtype, int B, int T, int H, long sb, long st, const int* len, int vec) {
    if ((dtype != CPCSV_F32 && dtype != CPCSV_BF16) || B <= 0 || T <= 0 || H <= 0 || T > CPCSV_SCAN_MAX_T) return -1001;
    d = Dims{B, T, H, H / vec, 0, (T + CH - 1) / CH, sb, st, len};
    // a launch holds fewer than 2^32 threads
    const long groups = (d.G + 63L) / 64, threads = T <= SHORT ? (long)B * d.G : max((long)tiles_of(T, FW) * FW, (long)tiles_of(T, BW) * BW) * 64;
    if (threads >= (1L << 32) - TB || (T > SHORT && threads * B >= (1L << 32) / groups)) return -1002;
    return 0;
}
}  // namespace

extern "C" int cpcsv_scan_states(int T) { return T > SHORT && T <= CPCSV_SCAN_MAX_T ? (T + CH - 1) / CH : 0; }

extern "C" long cpcsv_scan_workspace(int B, int T, int H, int backward) {
    return B > 0 && T > SHORT && T <= CPCSV_SCAN_MAX_T && H > 0 ? look_bytes(B, T, H, backward ? BW : FW) : 0;
}

extern "C" int cpcsv_scan_fwd(const void* p, int dtype, long psb, long pst, const float* h0, const int* lengths, void* y, float* h_last,
                              float* hin, void* ws, int B, int T, int H, int out_gate, void* stream) {
    const bool two = pairs_ok(dtype, H, psb, pst, p, y, nullptr);
    Dims d;
    if (int rc = dims_of(d, dtype, B, T, H, psb, pst, lengths, two ? 2 : 1)) return rc;
    if (!p || !y || (T > SHORT && (!ws || ((uintptr_t)ws & 15)))) return -1003;
    hipStream_t st = (hipStream_t)stream;
#define GO(T_, V) (out_gate ? run_fwd<T_, V, true>((const T_*)p, h0, (T_*)y, h_last, hin, ws, d, st) \
                            : run_fwd<T_, V, false>((const T_*)p, h0, (T_*)y, h_last, hin, ws, d, st))
    if (dtype == CPCSV_F32) return GO(float, 1);
    return two ? GO(bf16_t, 2) : GO(bf16_t, 1);
#undef GO
}

extern "C" int cpcsv_scan_bwd(const void* p, int dtype, long psb, long pst, const float* h0, const int* lengths, const float* hin,
                              const void* dy, const float* dh_last, void* dp, float* dh0, void* ws, int B, int T, int H,
                              int out_gate, void* stream) {
    const bool two = pairs_ok(dtype, H, psb, pst, p, dy, dp);
    Dims d;
    if (int rc = dims_of(d, dtype, B, T, H, psb, pst, lengths, two ? 2 : 1)) return rc;
    if (!p || !dy || !dp || (T > SHORT && (!hin || !ws || ((uintptr_t)ws & 15)))) return -1003;
    hipStream_t st = (hipStream_t)stream;
#define GO(T_, V) (out_gate ? run_bwd<T_, V, true>((const T_*)p, h0, hin, (const T_*)dy, dh_last, (T_*)dp, dh0, ws, d, st) \
                            : run_bwd<T_, V, false>((const T_*)p, h0, hin, (const T_*)dy, dh_last, (T_*)dp, dh0, ws, d, st))
    if (dtype == CPCSV_F32) return GO(float, 1);
    return two ? GO(bf16_t, 2) : GO(bf16_t, 1);
#undef GO
}
