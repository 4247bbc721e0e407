// eventad_amd/csrc/rmsnorm.hip -- root-mean-square norm of rows with the residual's addition, its gradient, and the form
// with an 8-bit output.
//
//   h = round(x + residual),   r = 1 / sqrt(mean(h^2) + eps),   y = h r w
//   8 bit: scale = max|y| / 448 per row,  q = e4m3(y / scale)
//
// h is rounded to the activations' type before it is used, because it is what the next layer reads and what the backward pass
// has: norm and gradient are those of the stored sum.  Gradient, with e = dy w:
//   dh = r (e - h r^2 mean(e h)) + dsum   (the gradient of x and of residual),   dw = sum over rows of dy h r
//
// Bound by bytes.  LANES lanes hold a row in registers (ITERS 16-byte pieces each), so every array is read and written once;
// sums over a row go through DPP / shuffles, over more than a wave through LDS.  Rows too long for registers are read twice.
// bf16 with residual, 400,000 x 256: 819 MB in 130 us (6.3 TB/s), the gradient 819 MB in 173 us (4.7 TB/s; a copy of 4 GiB runs
// at 4.75); 8 bits, 16,384 x 2048: 235 MB in 48 us (4.9 TB/s), 100,000 x 2048 1434 MB in 272 (5.3).
#include "seq.h"

struct NormArgs {
    const void *x, *res; int64_t ldx, ldr;
    const float* w;
    void *sum, *y; int64_t lds, ldy;
    uint8_t* q; int64_t ldq; float* scale;
    int64_t rows; int channels; float eps;
    // gradient
    const void *dy, *dsum; int64_t lddy, ldds;
    void* dh; int64_t lddh;
    float* part;                                     // [workgroups][channels]
};

// A piece of a row: V elements from column c on.  U: rows start anywhere and end inside a piece; whole pieces are still one access
// each (global memory takes any address), the last one goes element by element.  (12,000 x 8191 bf16: forward 193 us, with gradient 600; x 8192
// 150 and 294.  The gradient then takes 258 registers, one wave per SIMD.)
template <typename T, int V> struct NormAny { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T, int V, bool U> __device__ __forceinline__ typename SeqRaw<T, V>::type norm_raw(const T* __restrict__ row, int c, int D) {
    if constexpr (!U) return seq_raw<T, V>(row + min(c, D - V));
    else {
        typename SeqRaw<T, V>::type v = {};
        if (c + V <= D) {
            const typename NormAny<T, V>::type w = *(const typename NormAny<T, V>::type*)(row + c);
            v = w;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) if (c + i < D) v[i] = row[c + i];
        }
        return v;
    }
}
template <typename T, int V, bool U> __device__ __forceinline__ void norm_load(const T* __restrict__ row, int c, int D, float (&out)[V]) {
    if constexpr (!U) seq_load<T, V>(row + c, out);
    else seq_unpack<T, V>(norm_raw<T, V, U>(row, c, D), out);
}
template <typename T, int V, bool U> __device__ __forceinline__ void norm_store(T* __restrict__ row, int c, int D, const float (&in)[V]) {
    if constexpr (!U) seq_store<T, V>(row + c, in);
    else if (c + V <= D) {
        typename NormAny<T, V>::type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)in[i];
        *(typename NormAny<T, V>::type*)(row + c) = v;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (c + i < D) row[c + i] = (T)in[i];
    }
}
template <int V, bool U> __device__ __forceinline__ void norm_weights(const float* __restrict__ w, int c, int D, float (&out)[V]) {
    if (!U || c + V <= D) {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = w[c + i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = c + i < D ? w[c + i] : 0.f;
    }
}

// Sums over the LANES lanes that share a row.  More than a wave exchanges them in s, which a workgroup may use again after one
// more barrier (two halves in turn, in a loop).
template <int LANES> __device__ __forceinline__ float row_sum(float v, float* s) {
    v = seq_lane_sum<LANES < 64 ? LANES : 64>(v);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
    }
    return v;
}
template <int LANES> __device__ __forceinline__ void row_sums(float& v, float& u, float* s) {
    v = seq_lane_sum<LANES < 64 ? LANES : 64>(v);
    u = seq_lane_sum<LANES < 64 ? LANES : 64>(u);
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) { s[threadIdx.x >> 6] = v; s[4 + (threadIdx.x >> 6)] = u; }
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
        u = (s[4] + s[5]) + (s[6] + s[7]);
    }
}
// a sum and the maximum of the bit patterns of non-negative floats (NaN is above all numbers and stays)
__device__ __forceinline__ unsigned most_of(unsigned a, unsigned b) { return a > b ? a : b; }
template <int LANES> __device__ __forceinline__ void row_sum_max(float& v, unsigned& u, float* s) {
    v = seq_lane_sum<LANES < 64 ? LANES : 64>(v);
    u = most_of(u, seq_dpp_bits<0xB1>(u));
    u = most_of(u, seq_dpp_bits<0x4E>(u));
    u = most_of(u, seq_dpp_bits<0x141>(u));
    u = most_of(u, seq_dpp_bits<0x140>(u));
    if constexpr (LANES >= 32) { const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false); u = most_of(r[0], r[1]); }
    if constexpr (LANES >= 64) { const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false); u = most_of(r[0], r[1]); }
    if constexpr (LANES > 64) {
        if ((threadIdx.x & 63) == 0) { s[threadIdx.x >> 6] = v; s[4 + (threadIdx.x >> 6)] = __uint_as_float(u); }
        __syncthreads();
        v = (s[0] + s[1]) + (s[2] + s[3]);
        const unsigned* m = (const unsigned*)s + 4;
        u = most_of(most_of(m[0], m[1]), most_of(m[2], m[3]));
    }
}

// LOOP: the row does not fit ITERS pieces per lane and is read again for every pass over it.
template <typename T, int V, bool U, int LANES, int ITERS, bool LOOP>
__global__ __launch_bounds__(256) void k_norm_fwd(NormArgs a) {
    __shared__ __attribute__((aligned(16))) float s_red[4];
    constexpr int PER = 256 / LANES;
    const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES, D = a.channels;
    const bool in = row < a.rows;
    const int64_t r = in ? row : a.rows - 1;
    const T* x = (const T*)a.x + r * a.ldx;
    const T* res = a.res ? (const T*)a.res + r * a.ldr : nullptr;
    float h[ITERS][V];
    auto piece = [&](int c, float (&v)[V], bool store) {         // h of the piece at column c
        norm_load<T, V, U>(x, c, D, v);
        if (res) {
            float e[V];
            norm_load<T, V, U>(res, c, D, e);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (float)(T)(v[i] + e[i]);
            if (store) norm_store<T, V, U>((T*)a.sum + r * a.lds, c, D, v);
        }
    };
    float ss = 0.f;
    if constexpr (LOOP) {
        for (int c = lane * V; c < D; c += LANES * V) {
            float v[V];
            piece(c, v, in);
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(v[i], v[i], ss);
        }
    } else {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int c = (k * LANES + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) h[k][i] = 0.f;
            if (c < D) piece(c, h[k], in);
        }
#pragma unroll
        for (int k = 0; k < ITERS; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(h[k][i], h[k][i], ss);
    }
    ss = row_sum<LANES>(ss, s_red);
    const float inv = 1.f / sqrtf(ss / (float)D + a.eps);
    if (!in) return;
    auto finish = [&](int c, const float (&v)[V]) {
        float y[V], w[V];
        norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = v[i] * inv * w[i];
        norm_store<T, V, U>((T*)a.y + r * a.ldy, c, D, y);
    };
    if constexpr (LOOP) { for (int c = lane * V; c < D; c += LANES * V) { float v[V]; piece(c, v, false); finish(c, v); } }
    else {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) { const int c = (k * LANES + lane) * V; if (c < D) finish(c, h[k]); }
    }
}

// ---- 8 bits ----------------------------------------------------------------------------------------------------------------
// y / scale = 448 p / max|p| with p = h w needs no r.  A value next to a border of the 8-bit grid has to fall on the side the
// definition says, so the quotient is formed in float32 (p, its maximum, 448 / maximum and the product: error below 5 units in the
// last place) and, where it lies within 8 of a border, again in float64, where p is exact.  One value in 60,000 of ordinary data
// does.  A row with max|p| below 2^-100 is formed in float64 altogether: 448 / max|p| leaves float32 at 1.3e-36, and below 1.2e-38 p
// has not all its bits; so is its scale.

// v rounded towards the odd neighbour, so that a second rounding to fewer bits is the one rounding of v: e4m3 keeps 4 of the
// 24 bits of a float
__device__ __forceinline__ float norm_to_odd(double v) {
    const float f = (float)v;
    const double back = (double)f;
    if (back == v || !(fabs(v) < 1e30)) return f;
    unsigned u = __float_as_uint(f);
    if (fabs(back) > fabs(v)) --u;                               // towards zero
    return __uint_as_float(u | 1u);
}

template <typename T, int V, bool U, int LANES, int ITERS, bool LOOP>
__global__ __launch_bounds__(256) void k_norm_fp8(NormArgs a) {
    __shared__ __attribute__((aligned(16))) float s_red[8];
    __shared__ unsigned long long s_exact[LANES > 64 ? 4 : 1];
    constexpr int PER = 256 / LANES;
    const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / LANES;
    const int lane = threadIdx.x % LANES, D = a.channels;
    const bool in = row < a.rows;
    const int64_t r = in ? row : a.rows - 1;
    const T* x = (const T*)a.x + r * a.ldx;
    const T* res = a.res ? (const T*)a.res + r * a.ldr : nullptr;
    float p[ITERS][V];
    auto piece = [&](int c, float (&v)[V], bool store) {         // h of the piece at column c
        norm_load<T, V, U>(x, c, D, v);
        if (res) {
            float e[V];
            norm_load<T, V, U>(res, c, D, e);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (float)(T)(v[i] + e[i]);
            if (store) norm_store<T, V, U>((T*)a.sum + r * a.lds, c, D, v);
        }
    };
    float ss = 0.f, top = 0.f, poison = 0.f;
    auto fold = [&](int c, float (&v)[V]) {                      // h -> p
        float w[V];
        norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            ss = fmaf(v[i], v[i], ss);
            v[i] *= w[i];
            top = fmaxf(top, fabsf(v[i]));
            poison = fmaf(v[i], 0.f, poison);                    // NaN if anything is not finite
        }
    };
    if constexpr (LOOP) { for (int c = lane * V; c < D; c += LANES * V) { float v[V]; piece(c, v, in); fold(c, v); } }
    else {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int c = (k * LANES + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) p[k][i] = 0.f;
            if (c < D) piece(c, p[k], in);
        }
#pragma unroll
        for (int k = 0; k < ITERS; ++k) { const int c = (k * LANES + lane) * V; if (c < D) fold(c, p[k]); }
    }
    const unsigned own = __float_as_uint(poison == 0.f ? top : __builtin_nanf(""));
    unsigned most = own;
    row_sum_max<LANES>(ss, most, s_red);
    const float inv = 1.f / sqrtf(ss / (float)D + a.eps);
    float scale = __uint_as_float(most) * inv / 448.f;
    const bool zero = !(scale >= 1.17549435e-38f) && scale == scale;             // a row of zeros (or next to it)
    if (zero) scale = 1.f;
    const float by32 = zero ? inv : 448.f / __uint_as_float(most);
    const bool tiny = !zero && most < 0x0d800000u;               // 2^-100
    // p -> q of a piece; true if a value lies too close to a border
    auto divide = [&](const float (&v)[V], float (&q)[V]) {
        unsigned near = 0xffffffffu, low = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            q[i] = v[i] * by32;
            const unsigned u = __float_as_uint(q[i]);
            near = min(near, (u << 12) - 0x7fff8000u);           // (borders: the 20 bits that e4m3 has not are 0x80000)
            low = min(low, (u << 1) - 2u);
        }
        bool close = tiny || near <= 0x10000u;
        if (low < 0x79000000u - 2u) {                            // below 2^-6: steps of 2^-9, borders between them
#pragma unroll
            for (int i = 0; i < V; ++i)
                close |= fabsf(q[i]) < 0x1p-6f && fabsf(__builtin_amdgcn_fractf(fabsf(q[i]) * 512.f) - 0.5f) <= 0x1p-18f;
        }
        return close;
    };
    bool close = LOOP, close_in[ITERS];
    if constexpr (!LOOP) {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            close_in[k] = divide(p[k], p[k]);                    // (p becomes q)
            close |= close_in[k];
        }
    }
    // any lane of the row (and of the wave's other rows): then the row's maximum in float64 -- of the entries that share the
    // float32 maximum, as rounding keeps the order
    double by = 0.0;
    if (LANES > 64 ? __syncthreads_or(close) : (int)__any(close)) {
        unsigned long long exact = 0;
        if (own == most && own <= 0x7f800000u) {
            for (int c = lane * V; c < D; c += LANES * V) {
                float v[V], w[V];
                piece(c, v, false);
                norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (__float_as_uint(fabsf(v[i] * w[i])) == most)
                        exact = max(exact, (unsigned long long)__double_as_longlong(fabs((double)v[i] * (double)w[i])));
            }
        }
#pragma unroll
        for (int d = 1; d < (LANES < 64 ? LANES : 64); d <<= 1) exact = max(exact, (unsigned long long)__shfl_xor(exact, d, 64));
        if constexpr (LANES > 64) {
            if ((threadIdx.x & 63) == 0) s_exact[threadIdx.x >> 6] = exact;
            __syncthreads();
            exact = max(max(s_exact[0], s_exact[1]), max(s_exact[2], s_exact[3]));
        }
        by = most > 0x7f800000u ? (double)__builtin_nanf("") : zero ? (double)inv : 448.0 / __longlong_as_double(exact);
        if (tiny) scale = (float)(__longlong_as_double(exact) * (double)inv / 448.0);
    }
    if (in && lane == 0) a.scale[r] = scale;
    if (!in) return;
    auto finish = [&](int c, float (&q)[V], bool again) {
        if (again) {
            float h[V], w[V];
            piece(c, h, false);
            norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
            for (int i = 0; i < V; ++i) q[i] = norm_to_odd((double)h[i] * (double)w[i] * by);
        }
        uint8_t* out = a.q + r * a.ldq + c;
        if constexpr (V == 1) *out = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[0], 0, false);
        else {
            typedef unsigned word __attribute__((ext_vector_type(V / 4)));
            typedef unsigned any __attribute__((ext_vector_type(V / 4), aligned(1)));
            word o;
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
                o[i] = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], w, true);
            }
            if constexpr (!U) *(word*)out = o;
            else if (c + V <= D) *(any*)out = o;
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) if (c + i < D) out[i] = (uint8_t)(o[i / 4] >> (8 * (i & 3)));
            }
        }
    };
    if constexpr (LOOP) {
        for (int c = lane * V; c < D; c += LANES * V) {
            float v[V], w[V];
            piece(c, v, false);
            norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] *= w[i];
            const bool again = divide(v, v);
            finish(c, v, again);
        }
    } else {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) { const int c = (k * LANES + lane) * V; if (c < D) finish(c, p[k], close_in[k]); }
    }
}

// A workgroup goes over rows blockIdx.x, blockIdx.x + gridDim.x, ... (x PER rows at a time) and keeps its share of dw in
// registers (LOOP: in its own row of `part`).  1024 workgroups, 4 per CU: with the next row requested ahead that is enough
// loads in flight (188 us without the request, 173 with it), and dw's parts stay at 1024 rows.
template <typename T, int V, bool U, int LANES, int ITERS, bool LOOP>
__global__ __launch_bounds__(256) void k_norm_bwd(NormArgs a) {
    __shared__ __attribute__((aligned(16))) float s_red[2][8];
    __shared__ float s_dw[LANES < 256 ? 256 * V * ITERS : 1];
    constexpr int PER = 256 / LANES;
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES, D = a.channels;
    float dw[ITERS][V];
#pragma unroll
    for (int k = 0; k < ITERS; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    float* part = a.part + (int64_t)blockIdx.x * D;
    if constexpr (LOOP) {
        for (int c = lane * V; c < D; c += LANES * V)
#pragma unroll
            for (int i = 0; i < V; ++i) if (!U || c + i < D) part[c + i] = 0.f;
    }
    const int64_t step = (int64_t)gridDim.x * PER;
    // (a row's arrays are requested while the row in front is worked on; without that the sums over a row leave memory idle)
    typename SeqRaw<T, V>::type rh[ITERS], rg[ITERS], rs[ITERS];
    auto request = [&](int64_t r) {
        r = min(r, a.rows - 1);
        const T* hr = (const T*)a.sum + r * a.lds;
        const T* gr = (const T*)a.dy + r * a.lddy;
        const T* sr = a.dsum ? (const T*)a.dsum + r * a.ldds : hr;
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int c = (k * LANES + lane) * V;
            rh[k] = norm_raw<T, V, U>(hr, c, D); rg[k] = norm_raw<T, V, U>(gr, c, D); rs[k] = norm_raw<T, V, U>(sr, c, D);
        }
    };
    if (!LOOP && a.rows) request((int64_t)blockIdx.x * PER + sub);
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * PER; r0 < a.rows; r0 += step) {
        const bool in = r0 + sub < a.rows;
        const int64_t r = in ? r0 + sub : a.rows - 1;
        float h[ITERS][V], g[ITERS][V], ds[ITERS][V], ss = 0.f, eh = 0.f;
        auto fold = [&](int c, const float (&hv)[V], const float (&gv)[V]) {
            float w[V];
            norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
            for (int i = 0; i < V; ++i) { ss = fmaf(hv[i], hv[i], ss); eh = fmaf(gv[i] * w[i], hv[i], eh); }
        };
        const T* hr = (const T*)a.sum + r * a.lds;
        const T* gr = (const T*)a.dy + r * a.lddy;
        const T* sr = a.dsum ? (const T*)a.dsum + r * a.ldds : nullptr;
        if constexpr (LOOP) {
            for (int c = lane * V; c < D; c += LANES * V) { float hv[V], gv[V]; norm_load<T, V, U>(hr, c, D, hv); norm_load<T, V, U>(gr, c, D, gv); fold(c, hv, gv); }
        } else {
#pragma unroll
            for (int k = 0; k < ITERS; ++k) { seq_unpack<T, V>(rh[k], h[k]); seq_unpack<T, V>(rg[k], g[k]); seq_unpack<T, V>(rs[k], ds[k]); }
            request(r0 + step + sub);
#pragma unroll
            for (int k = 0; k < ITERS; ++k) { const int c = (k * LANES + lane) * V; if (c < D) fold(c, h[k], g[k]); }
        }
        row_sums<LANES>(ss, eh, s_red[turn]);
        turn ^= 1;
        const float inv = 1.f / sqrtf(ss / (float)D + a.eps), m = inv * inv * (eh / (float)D);
        if (!in) continue;
        auto finish = [&](int c, const float (&hv)[V], const float (&gv)[V], const float (&sv)[V], float (&acc)[V]) {
            float dh[V], w[V];
            norm_weights<V, U>(a.w, c, D, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dh[i] = fmaf(inv, fmaf(-hv[i], m, gv[i] * w[i]), sr ? sv[i] : 0.f);
                acc[i] = fmaf(gv[i] * inv, hv[i], acc[i]);
            }
            norm_store<T, V, U>((T*)a.dh + r * a.lddh, c, D, dh);
        };
        if constexpr (LOOP) {
            for (int c = lane * V; c < D; c += LANES * V) {
                float hv[V], gv[V], sv[V], acc[V];
                norm_load<T, V, U>(hr, c, D, hv); norm_load<T, V, U>(gr, c, D, gv);
                if (sr) norm_load<T, V, U>(sr, c, D, sv);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = !U || c + i < D ? part[c + i] : 0.f;
                finish(c, hv, gv, sv, acc);
#pragma unroll
                for (int i = 0; i < V; ++i) if (!U || c + i < D) part[c + i] = acc[i];
            }
        } else {
#pragma unroll
            for (int k = 0; k < ITERS; ++k) { const int c = (k * LANES + lane) * V; if (c < D) finish(c, h[k], g[k], ds[k], dw[k]); }
        }
    }
    if constexpr (!LOOP && LANES == 256) {
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int c = (k * LANES + lane) * V;
            if (c < D)
#pragma unroll
                for (int i = 0; i < V; ++i) if (!U || c + i < D) part[c + i] = dw[k][i];
        }
    } else if constexpr (!LOOP) {                                  // the workgroup's PER row groups, added in order
#pragma unroll
        for (int k = 0; k < ITERS; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s_dw[sub * (LANES * ITERS * V) + (k * LANES + lane) * V + i] = dw[k][i];
        __syncthreads();
        for (int c = threadIdx.x; c < D; c += 256) {
            float v = 0.f;
#pragma unroll
            for (int g = 0; g < PER; ++g) v += s_dw[g * (LANES * ITERS * V) + c];
            part[c] = v;
        }
    }
}

static int norm_groups(int64_t rows) { return (int)(rows < 1 ? 1 : rows < 1024 ? rows : 1024); }

template <int WHAT, typename T, int V, bool U, int LANES, int ITERS, bool LOOP> static int norm_launch3(const NormArgs& a, int groups, hipStream_t st) {
    constexpr int PER = 256 / LANES;
    const long long blocks = (a.rows + PER - 1) / PER;
    if (WHAT != 2 && blocks * 256 > SEQ_MOST_THREADS) return EVENTAD_ERR_TOO_LARGE;
    const dim3 grid((unsigned)blocks), block(256);
    if constexpr (WHAT == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_fwd<T, V, U, LANES, ITERS, LOOP>), grid, block, 0, st, a);
    if constexpr (WHAT == 1) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_fp8<T, V, U, LANES, ITERS, LOOP>), grid, block, 0, st, a);
    if constexpr (WHAT == 2) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_norm_bwd<T, V, U, LANES, ITERS, LOOP>), dim3(groups), block, 0, st, a);
    return evad_last_error();
}
// Short rows share a wave (400,000 x 256 bf16: 148 us, with a wave per row 173), and a row stays in one wave, without LDS, up to two
// pieces per lane (65,536 x 1024: 101 us, gradient 109; with four waves 103 and 175).  Up to four pieces the gradient, which
// keeps dw and the next row in registers too, still does better with a wave per row (65,536 x 1280: 153 us against 184), the
// forward forms with four waves (100,000 x 2048: 276 us against 302).  From there on four waves (16,384 x 4096: 103 us, a wave 117), up to
// eight pieces per lane (12,000 x 8192 f32: 288 us, with gradient 564, read again for every pass over the row 360 and 762; x 12,288 bf16
// 228 and 513 against 269 and 710).  The gradient's eight pieces of eight 16-bit elements take 390 registers, one wave per SIMD,
// and unaligned ones all 512 and scratch beside them; that is still the faster side (x 12,287 bf16 with gradient: 889 us against 1295).
template <int WHAT, typename T, int V, bool U> static int norm_launch2(const NormArgs& a, int groups, hipStream_t st) {
    const int pieces = (a.channels + V - 1) / V;
    if (pieces <= 16) return norm_launch3<WHAT, T, V, U, 16, 1, false>(a, groups, st);
    if (pieces <= 32) return norm_launch3<WHAT, T, V, U, 32, 1, false>(a, groups, st);
    if (pieces <= 64) return norm_launch3<WHAT, T, V, U, 64, 1, false>(a, groups, st);
    if (pieces <= 128) return norm_launch3<WHAT, T, V, U, 64, 2, false>(a, groups, st);
    if (pieces <= 256) return WHAT == 2 ? norm_launch3<WHAT, T, V, U, 64, 4, false>(a, groups, st) : norm_launch3<WHAT, T, V, U, 256, 1, false>(a, groups, st);
    if (pieces <= 512) return norm_launch3<WHAT, T, V, U, 256, 2, false>(a, groups, st);
    if (pieces <= 1024) return norm_launch3<WHAT, T, V, U, 256, 4, false>(a, groups, st);
    if (pieces <= 2048) return norm_launch3<WHAT, T, V, U, 256, 8, false>(a, groups, st);
    return norm_launch3<WHAT, T, V, U, 256, 1, true>(a, groups, st);
}
// Rows that are not whole aligned pieces: pieces all the same (12,000 x 8191 bf16: forward 196 us, with gradient 633, 8 bits 203; element
// by element 383, 1010 and 536), but few channels one to a lane, as most of the lanes would have none and one a tail
// (200,000 x 30 bf16: 25 and 59 us against 36 and 112; x 100 38 and 82 against 25 and 65).
template <int WHAT, typename T> static int norm_launch1(const NormArgs& a, bool vec, int groups, hipStream_t st) {
    constexpr int N = 16 / sizeof(T);
    if (vec && a.channels % N == 0) return norm_launch2<WHAT, T, N, false>(a, groups, st);
    if (a.channels >= 64) return norm_launch2<WHAT, T, N, true>(a, groups, st);
    if (a.channels <= 16) return norm_launch3<WHAT, T, 1, false, 16, 1, false>(a, groups, st);
    if (a.channels <= 32) return norm_launch3<WHAT, T, 1, false, 32, 1, false>(a, groups, st);
    return norm_launch3<WHAT, T, 1, false, 64, 1, false>(a, groups, st);
}
template <int WHAT> static int norm_launch(const NormArgs& a, int dtype, bool vec, int groups, hipStream_t st) {
    if (dtype == SEQ_F32) return norm_launch1<WHAT, float>(a, vec, groups, st);
    if (dtype == SEQ_BF16) return norm_launch1<WHAT, __bf16>(a, vec, groups, st);
    return norm_launch1<WHAT, _Float16>(a, vec, groups, st);
}
static bool norm_shape_ok(int64_t rows, int channels, int dtype) {
    return rows >= 0 && rows <= 0x7fffff00 && channels >= 1 && channels <= (1 << 24) && dtype >= 0 && dtype <= 2;
}

extern "C" int eventad_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* w, void* sum, int64_t lds,
                                    void* y, int64_t ldy, int64_t rows, int channels, float eps, int dtype, void* stream) {
    if (!norm_shape_ok(rows, channels, dtype) || !w || !(eps >= 0.f) ||
        (rows && (!x || !y || ldx < channels || ldy < channels || (residual && (!sum || ldr < channels || lds < channels))))) return EVAD_ERR_ARG;
    if (!rows) return EVAD_OK;
    NormArgs a = {};
    a.x = x; a.ldx = ldx; a.res = residual; a.ldr = ldr; a.w = w; a.sum = sum; a.lds = lds; a.y = y; a.ldy = ldy; a.rows = rows; a.channels = channels; a.eps = eps;
    const int e = dtype == SEQ_F32 ? 4 : 2;
    const bool vec = seq_aligned(x, ldx * e) && seq_aligned(y, ldy * e) && (!residual || (seq_aligned(residual, ldr * e) && seq_aligned(sum, lds * e)));
    return norm_launch<0>(a, dtype, vec, 0, (hipStream_t)stream);
}

extern "C" int eventad_rms_norm_fp8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const float* w, void* sum, int64_t lds,
                                    uint8_t* q, int64_t ldq, float* scale, int64_t rows, int channels, float eps, int dtype, void* stream) {
    if (!norm_shape_ok(rows, channels, dtype) || !w || !(eps >= 0.f) ||
        (rows && (!x || !q || !scale || ldx < channels || ldq < channels || (residual && (!sum || ldr < channels || lds < channels))))) return EVAD_ERR_ARG;
    if (!rows) return EVAD_OK;
    NormArgs a = {};
    a.x = x; a.ldx = ldx; a.res = residual; a.ldr = ldr; a.w = w; a.sum = sum; a.lds = lds; a.q = q; a.ldq = ldq; a.scale = scale;
    a.rows = rows; a.channels = channels; a.eps = eps;
    const int e = dtype == SEQ_F32 ? 4 : 2;
    const bool vec = seq_aligned(x, ldx * e) && (!residual || (seq_aligned(residual, ldr * e) && seq_aligned(sum, lds * e))) &&
                     ((((uintptr_t)q | (uintptr_t)ldq) & (16 / e - 1)) == 0);
    return norm_launch<1>(a, dtype, vec, 0, (hipStream_t)stream);
}

extern "C" int eventad_rms_norm_workspace(int64_t rows, int channels, int64_t* bytes) {
    if (!bytes || !norm_shape_ok(rows, channels, 0)) return EVAD_ERR_ARG;
    *bytes = ((int64_t)norm_groups(rows) + SEQ_SUM_PARTS) * channels * 4;
    return EVAD_OK;
}

extern "C" int eventad_rms_norm_bwd(const void* sum, int64_t lds, const float* w, const void* dy, int64_t lddy, const void* dsum, int64_t ldds,
                                    void* dh, int64_t lddh, float* dw, void* workspace, int64_t workspace_bytes, int64_t rows, int channels,
                                    float eps, int dtype, void* stream) {
    int64_t need = 0;
    if (!norm_shape_ok(rows, channels, dtype) || !w || !(eps >= 0.f) || !dw || eventad_rms_norm_workspace(rows, channels, &need) != EVAD_OK ||
        !workspace || workspace_bytes < need ||
        (rows && (!sum || !dy || !dh || lds < channels || lddy < channels || lddh < channels || (dsum && ldds < channels)))) return EVAD_ERR_ARG;
    NormArgs a = {};
    a.sum = (void*)sum; a.lds = lds; a.w = w; a.dy = dy; a.lddy = lddy; a.dsum = dsum; a.ldds = ldds; a.dh = dh; a.lddh = lddh;
    a.part = (float*)workspace; a.rows = rows; a.channels = channels; a.eps = eps;
    const int e = dtype == SEQ_F32 ? 4 : 2;
    const bool vec = seq_aligned(sum, lds * e) && seq_aligned(dy, lddy * e) && seq_aligned(dh, lddh * e) && (!dsum || seq_aligned(dsum, ldds * e));
    const int groups = norm_groups(rows);
    const int rc = norm_launch<2>(a, dtype, vec, groups, (hipStream_t)stream);
    if (rc) return rc;
    return seq_colsum(a.part, groups, channels, dw, a.part + (int64_t)groups * channels, (hipStream_t)stream);
}
