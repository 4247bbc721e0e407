// eventad_amd/csrc/seqscan.hip -- selective state-space scan over the rows of packed clips, its gradient and its
// single-token form.
//
// Per channel d with N states (A f32[channels, N] real, usually negative):
//   s_t = softplus(delta_t + bias)   (or delta_t + bias)
//   h_t[n] = exp(s_t A[n]) h_{t-1}[n] + s_t u_t B_t[n]
//   y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)
// h before a clip's first row is the clip's state or zero.  Gradient, with dy_t the gradient in front of the gate and
// g_t = dL/dh_t = C_t dy_t + exp(s_{t+1} A) g_{t+1}:
//   du_t = D dy_t + s_t sum_n g_t B_t        ds_t = u_t sum_n g_t B_t + sum_n A g_t exp(s_t A) h_{t-1}
//   dA = sum_t s_t g_t exp(s_t A) h_{t-1}    dB_t[n] = sum_d g_t s_t u_t     dC_t[n] = sum_d dy_t h_t
//
// Layout: LPC lanes share a channel and hold 4 of its states each in registers (LPC = 4 / 8 / 16 for N <= 16 / 32 / 64), so a
// wave has 64 / LPC channels and a 256-thread workgroup 256 / LPC.  Rows go by in tiles of 16: the four lanes of a quad form the
// step sizes of four different rows (softplus, gate and conversions once per row and channel, not once per lane) and hand
// them round with DPP; B and C of the tile stand in LDS as floats, read as one 16-byte access per lane and row.
//
// What bounds it is the vector ALU: per row, channel and state one v_exp_f32 and five other operations, against 8 bytes per
// row and channel in 16 bits.  A long row axis is therefore split into chunks only as far as the chip needs workgroups: the
// chunks' own end states come from a first pass (without C, gate or output), are joined by a short one, and the second
// pass starts every chunk from its true state.  The adjoint g is split the same way, from the end.
//
// Every sum over rows or channels is in float32 and in a fixed order (no atomics): results are reproducible bit for bit.
#include "seq.h"

#define SCAN_TILE 16
#define SCAN_MAX_STATE 64

struct ScanArgs {
    SeqClips clips;
    const void *u, *delta, *z, *B, *C;
    int64_t ldu, ldd, ldz, ldb, ldc;
    const float *A, *D, *bias, *state;
    float* final_state;
    void* y; int64_t ldy;
    float* ckpt;                                     // [tiles][channels][4 LPC]: the state in front of every 16th row
    float* carry; float* span; int* flag;            // per chunk: [channels][4 LPC] end state, [channels] sum of s, 1 = stands alone
    int rows, channels, n_state, chunk_rows, chunks, softplus;
    // gradient
    const void* dy; int64_t lddy;
    const float* dfinal; float* dstate;
    void *du, *ddelta, *dz; int64_t lddu, lddd, lddz;
    float* part_bc;                                  // [channel blocks][rows][2][4 LPC]
    float* part_p;                                   // [chunks][channels*N (dA) | channels (dD) | channels (dbias)]
};

template <int CTRL> __device__ __forceinline__ float seq_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// value of lane Q of the quad, in all four lanes
template <int Q> __device__ __forceinline__ float quad_bcast(float v) { return seq_dpp<Q * 0x55>(v); }
__device__ __forceinline__ float quad_bcast(float v, int q) {
    return q == 0 ? quad_bcast<0>(v) : q == 1 ? quad_bcast<1>(v) : q == 2 ? quad_bcast<2>(v) : quad_bcast<3>(v);
}
// sum over the LPC lanes of a channel, in all of them: xor 1, xor 2 (quad_perm), then the mirrored half and whole row of 16
template <int LPC> __device__ __forceinline__ float chan_sum(float v) {
    v += seq_dpp<0xB1>(v);
    v += seq_dpp<0x4E>(v);
    if constexpr (LPC >= 8) v += seq_dpp<0x141>(v);
    if constexpr (LPC >= 16) v += seq_dpp<0x140>(v);
    return v;
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], with log1p(e) = 2 artanh(r), r = e / (2 + e) <= 1/3, as its
// series to r^15 (next term 2 r^17 / 17 < 1e-9): relative accuracy for small e too, where log(1 + e) has none left.
__device__ __forceinline__ float scan_softplus(float x) {
    const float e = seq_exp2(-SEQ_LOG2E * fabsf(x));
    const float r = e * seq_rcp(2.f + e), q = r * r;
    float p = fmaf(q, 1.f / 15.f, 1.f / 13.f);
    p = fmaf(q, p, 1.f / 11.f);
    p = fmaf(q, p, 1.f / 9.f);
    p = fmaf(q, p, 1.f / 7.f);
    p = fmaf(q, p, 1.f / 5.f);
    p = fmaf(q, p, 1.f / 3.f);
    p = fmaf(q, p, 1.f);
    return fmaxf(x, 0.f) + 2.f * r * p;
}

// lane's place in its workgroup
template <int LPC> struct ScanLane {
    int d, j, q; bool in;                            // channel, lane of the channel, lane of the quad, channel exists
    __device__ __forceinline__ ScanLane(const ScanArgs& a) {
        d = blockIdx.x * (256 / LPC) + threadIdx.x / LPC;
        j = threadIdx.x % LPC; q = threadIdx.x & 3;
        in = d < a.channels;
        d = min(d, a.channels - 1);
    }
};
// a lane's four entries of a row of N floats
__device__ __forceinline__ void scan_load4(const float* __restrict__ row, int j, int N, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 4 * j + i < N ? row[4 * j + i] : 0.f;
}
__device__ __forceinline__ void scan_store4(float* __restrict__ row, int j, int N, const float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) if (4 * j + i < N) row[4 * j + i] = v[i];
}

// B and C of the 16 rows from t0 into LDS as floats, zero for rows outside [lo, hi) and states >= N
template <typename T, int LPC>
__device__ __forceinline__ void scan_stage(const ScanArgs& a, int t0, int lo, int hi, float* __restrict__ sB, float* __restrict__ sC) {
    constexpr int N4 = 4 * LPC;
#pragma unroll
    for (int e = threadIdx.x; e < SCAN_TILE * N4; e += 256) {
        const int r = t0 + e / N4, n = e % N4;
        float b = 0.f, c = 0.f;
        if (r >= lo && r < hi && n < a.n_state) {
            b = (float)((const T*)a.B)[(int64_t)r * a.ldb + n];
            if (sC) c = (float)((const T*)a.C)[(int64_t)r * a.ldc + n];
        }
        sB[e] = b;
        if (sC) sC[e] = c;
    }
}

// The walk over the clips' ends while rows go up (all values are the same in the whole workgroup).
struct ScanWalk { int s, next; };
__device__ __forceinline__ ScanWalk scan_walk(const SeqClips& c, int row) {
    ScanWalk w;
    w.s = __builtin_amdgcn_readfirstlane(seq_find(c, row));
    w.next = w.s < c.n ? __builtin_amdgcn_readfirstlane(seq_start(c, w.s + 1)) : 0x7fffffff;
    return w;
}

// WHAT 0: outputs.  WHAT 1: the chunk's end state for the chunks behind it.
template <typename T, int LPC, int WHAT>
__global__ __launch_bounds__(256) void k_scan_fwd(ScanArgs a) {
    constexpr int N4 = 4 * LPC;
    __shared__ __attribute__((aligned(16))) float sB[2][SCAN_TILE * N4], sC[2][SCAN_TILE * N4];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y;
    const int c0 = chunk * a.chunk_rows, c1 = min(a.rows, c0 + a.chunk_rows);
    const int lo = max(0, seq_start(a.clips, 0)), hi = min(a.rows, seq_start(a.clips, n));       // rows that belong to a clip
    float A2[4], h[4] = {0.f, 0.f, 0.f, 0.f};
    scan_load4(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] *= SEQ_LOG2E;
    const float bias = a.bias ? a.bias[L.d] : 0.f, Dd = a.D ? a.D[L.d] : 0.f;

    int from = c0;
    ScanWalk w;
    bool alone = false;
    if constexpr (WHAT == 1) {
        // only the rows since the last clip start of the chunk matter, and none if the next chunk starts a clip of its own
        w = scan_walk(a.clips, c1 - 1);
        const int first = w.s >= 0 ? seq_start(a.clips, w.s) : 0;
        alone = w.s < 0 || w.s >= n || w.next <= c1 || first >= c0;
        if (blockIdx.x == 0 && threadIdx.x == 0) a.flag[chunk] = alone ? 1 : 0;
        if (w.s < 0 || w.s >= n || w.next <= c1) {
            if (L.in) {
                const float zero[4] = {0.f, 0.f, 0.f, 0.f};
                scan_store4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, zero);
            }
            return;
        }
        if (first >= c0) {
            from = first;
            if (a.state) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
        }
        w.next = 0x7fffffff;
    } else {
        w = scan_walk(a.clips, c0);
        if (a.final_state && L.in) {                             // empty clips at the chunk's first row keep their state
            for (int e = w.s - 1; e >= 0 && seq_start(a.clips, e) == c0; --e) {
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (a.state) scan_load4(a.state + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
                scan_store4(a.final_state + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
            }
        }
        if (w.s >= 0 && w.s < n) {
            if (seq_start(a.clips, w.s) == c0) { if (a.state) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h); }
            else if (chunk > 0) scan_load4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, h);
        }
    }
    if (c1 <= c0) return;
    const int tile0 = from / SCAN_TILE * SCAN_TILE;
    float span = 0.f;
    T ru[4], rd[4], rz[4];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t r = min(t0 + 4 * k + L.q, a.rows - 1);
            ru[k] = ((const T*)a.u)[r * a.ldu + L.d];
            rd[k] = ((const T*)a.delta)[r * a.ldd + L.d];
            if (WHAT == 0 && a.z) rz[k] = ((const T*)a.z)[r * a.ldz + L.d];
        }
    };
    fetch(tile0);
    scan_stage<T, LPC>(a, tile0, max(lo, from), min(hi, c1), sB[0], WHAT == 0 ? sC[0] : nullptr);
    __syncthreads();
    int buf = 0;
    for (int t0 = tile0; t0 < c1; t0 += SCAN_TILE, buf ^= 1) {
        float st[4], x[4], u[4], gate[4], ys[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = t0 + 4 * k + L.q;
            const bool live = r >= max(lo, from) && r < min(hi, c1);
            u[k] = live ? (float)ru[k] : 0.f;
            const float raw = (float)rd[k] + bias;
            st[k] = live ? (a.softplus ? scan_softplus(raw) : raw) : 0.f;      // a row of no clip leaves the state as it is
            x[k] = st[k] * u[k];
            span += st[k];
            gate[k] = 1.f;
            if (WHAT == 0 && a.z) { const float z = (float)rz[k]; gate[k] = live ? z * seq_sigmoid(z) : 0.f; }
            ys[k] = 0.f;
        }
        const bool more = t0 + SCAN_TILE < c1;
        if (more) {
            fetch(t0 + SCAN_TILE);
            scan_stage<T, LPC>(a, t0 + SCAN_TILE, lo, min(hi, c1), sB[buf ^ 1], WHAT == 0 ? sC[buf ^ 1] : nullptr);
        }
        if (WHAT == 0 && a.ckpt && L.in) *(seq_f4*)(a.ckpt + ((size_t)(t0 / SCAN_TILE) * a.channels + L.d) * N4 + 4 * L.j) = seq_f4{h[0], h[1], h[2], h[3]};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i = 4 * k + q;
                if (WHAT == 0 && t0 + i >= w.next && w.s < n && t0 + i < c1) {     // a clip ended in front of this row
                    const int p = t0 + i;
                    if (a.final_state && w.s >= 0 && L.in) scan_store4(a.final_state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
                    ++w.s;
                    while (w.s < n && seq_start(a.clips, w.s + 1) <= p) {
                        if (a.final_state && L.in) {
                            float v[4] = {0.f, 0.f, 0.f, 0.f};
                            if (a.state) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, v);
                            scan_store4(a.final_state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, v);
                        }
                        ++w.s;
                    }
                    w.next = w.s < n ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, w.s + 1)) : 0x7fffffff;
#pragma unroll
                    for (int m = 0; m < 4; ++m) h[m] = 0.f;
                    if (a.state && w.s < n) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
                }
                const float sb = quad_bcast(st[k], q), xb = quad_bcast(x[k], q);
                const seq_f4 b4 = *(const seq_f4*)(sB[buf] + i * N4 + 4 * L.j);
                float acc = 0.f;
                if constexpr (WHAT == 0) {
                    const seq_f4 c4 = *(const seq_f4*)(sC[buf] + i * N4 + 4 * L.j);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        h[m] = fmaf(seq_exp2(sb * A2[m]), h[m], xb * b4[m]);
                        acc = fmaf(c4[m], h[m], acc);
                    }
                    acc = chan_sum<LPC>(acc);
                    ys[k] = L.q == q ? acc : ys[k];
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m) h[m] = fmaf(seq_exp2(sb * A2[m]), h[m], xb * b4[m]);
                }
            }
        }
        if constexpr (WHAT == 0) {
            if (L.in && L.j < 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = t0 + 4 * k + L.q;
                    if (r < c1) ((T*)a.y)[(int64_t)r * a.ldy + L.d] = (T)(r >= lo && r < hi ? fmaf(Dd, u[k], ys[k]) * gate[k] : 0.f);
                }
            }
        }
        __syncthreads();
    }
    if constexpr (WHAT == 1) {
        if (L.in) {
            scan_store4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, h);
            span += seq_dpp<0xB1>(span);
            span += seq_dpp<0x4E>(span);
            if (L.j == 0) a.span[(size_t)chunk * a.channels + L.d] = span;
        }
    } else if (a.final_state && L.in && w.next <= c1 && w.s < n) {                 // a clip ends with the chunk
        if (w.s >= 0) scan_store4(a.final_state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
        if (c1 == a.rows) {                                                        // empty clips behind the last row
            for (int e = w.s + 1; e < n; ++e) {
                float v[4] = {0.f, 0.f, 0.f, 0.f};
                if (a.state) scan_load4(a.state + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
                scan_store4(a.final_state + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
            }
        }
    }
}

// The chunks' true entry states: thread per (channel, state), chunk by chunk (REV: from the last).  carry[chunk] holds the
// chunk's own contribution on entry and what flows into the chunk on return.
template <int REV>
__global__ __launch_bounds__(256) void k_scan_join(ScanArgs a, int n4) {
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, width = (int64_t)a.channels * n4;
    if (at >= width) return;
    const int d = (int)(at / n4), i = (int)(at - (int64_t)d * n4);
    const float A2 = i < a.n_state ? a.A[(size_t)d * a.n_state + i] * SEQ_LOG2E : 0.f;
    float in = 0.f;
    for (int k0 = 0; k0 < a.chunks; k0 += 8) {
        float own[8], sp[8]; int fl[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = min(k0 + j, a.chunks - 1), c = REV ? a.chunks - 1 - k : k;
            own[j] = a.carry[c * width + at]; sp[j] = a.span[(size_t)c * a.channels + d]; fl[j] = a.flag[c];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (k0 + j >= a.chunks) break;
            const int c = REV ? a.chunks - 1 - (k0 + j) : k0 + j;
            a.carry[c * width + at] = in;
            in = fl[j] ? own[j] : fmaf(seq_exp2(sp[j] * A2), in, own[j]);
        }
    }
}

// The adjoint of a chunk by itself: what its rows contribute to dL/dh in front of its first row.
template <typename T, int LPC>
__global__ __launch_bounds__(256) void k_scan_adj(ScanArgs a) {
    constexpr int N4 = 4 * LPC;
    __shared__ __attribute__((aligned(16))) float sC[2][SCAN_TILE * N4];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y;
    const int c0 = chunk * a.chunk_rows, c1 = min(a.rows, c0 + a.chunk_rows);
    float A2[4], g[4] = {0.f, 0.f, 0.f, 0.f};
    scan_load4(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] *= SEQ_LOG2E;
    const float bias = a.bias ? a.bias[L.d] : 0.f;
    const ScanWalk w = scan_walk(a.clips, c0);
    const bool dead = w.s < 0 || w.s >= n || seq_start(a.clips, w.s) >= c0;        // nothing flows out of the chunk
    const bool ends = w.next <= c1;                                                // the clip ends in it: nothing flows through
    if (blockIdx.x == 0 && threadIdx.x == 0) a.flag[chunk] = dead || ends ? 1 : 0;
    if (dead) {
        if (L.in) scan_store4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
        return;
    }
    const int to = min(w.next, c1);                                                // rows [c0, to)
    if (ends && a.dfinal) scan_load4(a.dfinal + ((size_t)w.s * a.channels + L.d) * N, L.j, N, g);
    float span = 0.f;
    T rd[4], ry[4], rz[4];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t r = max(0, min(t0 + 4 * k + L.q, a.rows - 1));
            rd[k] = ((const T*)a.delta)[r * a.ldd + L.d];
            ry[k] = ((const T*)a.dy)[r * a.lddy + L.d];
            if (a.z) rz[k] = ((const T*)a.z)[r * a.ldz + L.d];
        }
    };
    auto stage = [&](int t0, float* s) {
        for (int e = threadIdx.x; e < SCAN_TILE * N4; e += 256) {
            const int r = t0 + e / N4, m = e % N4;
            s[e] = r < to && m < N ? (float)((const T*)a.C)[(int64_t)r * a.ldc + m] : 0.f;
        }
    };
    int t0 = (to - 1) / SCAN_TILE * SCAN_TILE, buf = 0;
    fetch(t0);
    stage(t0, sC[0]);
    __syncthreads();
    for (; t0 >= c0; t0 -= SCAN_TILE, buf ^= 1) {
        float st[4], dy[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool live = t0 + 4 * k + L.q < to;
            const float raw = (float)rd[k] + bias;
            st[k] = live ? (a.softplus ? scan_softplus(raw) : raw) : 0.f;
            dy[k] = live ? (float)ry[k] : 0.f;
            if (a.z && live) { const float z = (float)rz[k]; dy[k] *= z * seq_sigmoid(z); }
            span += st[k];
        }
        if (t0 - SCAN_TILE >= c0) { fetch(t0 - SCAN_TILE); stage(t0 - SCAN_TILE, sC[buf ^ 1]); }
#pragma unroll
        for (int k = 3; k >= 0; --k) {
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const float sb = quad_bcast(st[k], q), db = quad_bcast(dy[k], q);
                const seq_f4 c4 = *(const seq_f4*)(sC[buf] + (4 * k + q) * N4 + 4 * L.j);
#pragma unroll
                for (int m = 0; m < 4; ++m) g[m] = seq_exp2(sb * A2[m]) * fmaf(c4[m], db, g[m]);
            }
        }
        __syncthreads();
    }
    if (L.in) {
        scan_store4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
        span += seq_dpp<0xB1>(span);
        span += seq_dpp<0x4E>(span);
        if (L.j == 0) a.span[(size_t)chunk * a.channels + L.d] = span;
    }
}

// 8 values of every lane summed over the channels of the wave.  Two swap-and-add steps fold the halves of the wave and the
// halves of each half while they halve the number of values (a swap serves two values), then DPP rotations add up the
// channels inside a row of 16 lanes.  Returns, for row r of 16 lanes, v[0..1] = values 2 (r & 1) + {0, 1} of the first four
// (r < 2) or of the last four (r >= 2).
__device__ __forceinline__ void swap_add32(float& x, const float& y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(y), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
}
__device__ __forceinline__ void swap_add16(float& x, const float& y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(y), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
}
template <int LPC> __device__ __forceinline__ void wave_fold(float (&b)[4], const float (&c)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) swap_add32(b[i], c[i]);           // lanes 0..31: sums of b, lanes 32..63: sums of c
    swap_add16(b[0], b[2]);                                       // even rows of 16: entry 0, odd rows: entry 2
    swap_add16(b[1], b[3]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (LPC <= 8) b[i] += seq_dpp<0x128>(b[i]);     // row_ror:8
        if constexpr (LPC <= 4) b[i] += seq_dpp<0x124>(b[i]);     // row_ror:4
    }
}

template <typename T, int LPC>
__global__ __launch_bounds__(256) void k_scan_bwd(ScanArgs a) {
    constexpr int N4 = 4 * LPC, W = 2 * N4;
    __shared__ __attribute__((aligned(16))) float sB[2][SCAN_TILE * N4], sC[2][SCAN_TILE * N4], red[4][SCAN_TILE * W];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int c0 = chunk * a.chunk_rows, c1 = min(a.rows, c0 + a.chunk_rows);
    const int lo = max(0, seq_start(a.clips, 0)), hi = min(a.rows, seq_start(a.clips, n));
    float A2[4], g[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f}, dD = 0.f, dbias = 0.f;
    scan_load4(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] *= SEQ_LOG2E;
    const float bias = a.bias ? a.bias[L.d] : 0.f, Dd = a.D ? a.D[L.d] : 0.f;
    auto empty = [&](int e) {                                     // an empty clip passes the gradient of its state on
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.dfinal) scan_load4(a.dfinal + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
        scan_store4(a.dstate + ((size_t)e * a.channels + L.d) * N, L.j, N, v);
    };
    // rows go down: s = the clip of the current row, [first, next) its rows
    int s = __builtin_amdgcn_readfirstlane(seq_find(a.clips, c1 - 1));
    int first = s >= 0 ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, s)) : 0;
    if (a.dstate && L.in)                                         // empty clips between this chunk's last row and the next row
        for (int e = s + 1; e < n && seq_start(a.clips, e + 1) <= c1; ++e) empty(e);
    if (s >= 0 && s < n) {
        if (seq_start(a.clips, s + 1) <= c1) { if (a.dfinal) scan_load4(a.dfinal + ((size_t)s * a.channels + L.d) * N, L.j, N, g); }
        else if (a.chunks > 1) scan_load4(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
    }
    T ru[4], rd[4], rz[4], ry[4];
    auto fetch = [&](int t0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t r = max(0, min(t0 + 4 * k + L.q, a.rows - 1));
            ru[k] = ((const T*)a.u)[r * a.ldu + L.d];
            rd[k] = ((const T*)a.delta)[r * a.ldd + L.d];
            ry[k] = ((const T*)a.dy)[r * a.lddy + L.d];
            if (a.z) rz[k] = ((const T*)a.z)[r * a.ldz + L.d];
        }
    };
    int t0 = (c1 - 1) / SCAN_TILE * SCAN_TILE, buf = 0;
    if (c1 > c0) {
        fetch(t0);
        scan_stage<T, LPC>(a, t0, lo, min(hi, c1), sB[0], sC[0]);
    }
    __syncthreads();
    for (; c1 > c0 && t0 >= c0; t0 -= SCAN_TILE, buf ^= 1) {
        float st[4], x[4], u[4], dy[4], ys[4], sb_[4], sa_[4], hp[SCAN_TILE][4];
        T raw_d[4], raw_z[4], raw_y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = t0 + 4 * k + L.q;
            const bool live = r >= lo && r < min(hi, c1);
            raw_d[k] = rd[k]; raw_z[k] = rz[k]; raw_y[k] = ry[k];
            u[k] = live ? (float)ru[k] : 0.f;
            const float raw = (float)rd[k] + bias;
            st[k] = live ? (a.softplus ? scan_softplus(raw) : raw) : 0.f;
            x[k] = st[k] * u[k];
            dy[k] = live ? (float)ry[k] : 0.f;
            if (a.z && live) { const float z = (float)rz[k]; dy[k] *= z * seq_sigmoid(z); }
            ys[k] = 0.f; sb_[k] = 0.f; sa_[k] = 0.f;
        }
        float h[4];
        {
            const seq_f4 v = *(const seq_f4*)(a.ckpt + ((size_t)(t0 / SCAN_TILE) * a.channels + L.d) * N4 + 4 * L.j);
#pragma unroll
            for (int m = 0; m < 4; ++m) h[m] = v[m];
        }
        if (t0 - SCAN_TILE >= c0) {
            fetch(t0 - SCAN_TILE);
            scan_stage<T, LPC>(a, t0 - SCAN_TILE, lo, min(hi, c1), sB[buf ^ 1], sC[buf ^ 1]);
        }
        // forward through the tile again, keeping the state in front of every row
        {
            ScanWalk w = {s, 0x7fffffff};
            if (s >= 0 && first <= t0) { if (s < n) w.next = __builtin_amdgcn_readfirstlane(seq_start(a.clips, s + 1)); }
            else w = scan_walk(a.clips, t0);
            if (w.s >= 0 && w.s < n && seq_start(a.clips, w.s) == t0) {
#pragma unroll
                for (int m = 0; m < 4; ++m) h[m] = 0.f;
                if (a.state) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i = 4 * k + q, p = t0 + i;
                    if (p >= w.next && w.s < n && p < c1) {
                        ++w.s;
                        while (w.s < n && seq_start(a.clips, w.s + 1) <= p) ++w.s;
                        w.next = w.s < n ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, w.s + 1)) : 0x7fffffff;
#pragma unroll
                        for (int m = 0; m < 4; ++m) h[m] = 0.f;
                        if (a.state && w.s < n) scan_load4(a.state + ((size_t)w.s * a.channels + L.d) * N, L.j, N, h);
                    }
                    const float sb = quad_bcast(st[k], q), xb = quad_bcast(x[k], q);
                    const seq_f4 b4 = *(const seq_f4*)(sB[buf] + i * N4 + 4 * L.j);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        hp[i][m] = h[m];
                        h[m] = fmaf(seq_exp2(sb * A2[m]), h[m], xb * b4[m]);
                    }
                }
            }
        }
        // and back
#pragma unroll
        for (int k = 3; k >= 0; --k) {
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const int i = 4 * k + q, p = t0 + i;
                if (p < c1 && p < first) {                        // the row belongs to an earlier clip: its last row
                    const int was = s;
                    while (s >= 0 && seq_start(a.clips, s) > p) --s;
                    first = s >= 0 ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, s)) : -1;
                    if (a.dstate && L.in) for (int e = s + 1; e < was; ++e) empty(e);
#pragma unroll
                    for (int m = 0; m < 4; ++m) g[m] = 0.f;
                    if (a.dfinal && s >= 0) scan_load4(a.dfinal + ((size_t)s * a.channels + L.d) * N, L.j, N, g);
                }
                const float sb = quad_bcast(st[k], q), xb = quad_bcast(x[k], q), db = quad_bcast(dy[k], q);
                const seq_f4 b4 = *(const seq_f4*)(sB[buf] + i * N4 + 4 * L.j);
                const seq_f4 c4 = *(const seq_f4*)(sC[buf] + i * N4 + 4 * L.j);
                float y = 0.f, gb = 0.f, ga = 0.f, vb[4], vc[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const float e = seq_exp2(sb * A2[m]), ah = e * hp[i][m];
                    const float ht = fmaf(xb, b4[m], ah);
                    y = fmaf(c4[m], ht, y);
                    g[m] = fmaf(c4[m], db, g[m]);
                    vb[m] = g[m] * xb;
                    vc[m] = db * ht;
                    gb = fmaf(g[m], b4[m], gb);
                    const float f = g[m] * ah;
                    ga = fmaf(A2[m], f, ga);
                    dA[m] = fmaf(sb, f, dA[m]);
                    g[m] *= e;
                }
                if (a.dstate && p == first && p < c1 && s >= 0 && s < n && L.in)
                    scan_store4(a.dstate + ((size_t)s * a.channels + L.d) * N, L.j, N, g);
                y = chan_sum<LPC>(y); gb = chan_sum<LPC>(gb); ga = chan_sum<LPC>(ga);
                const bool mine = L.q == q;
                ys[k] = mine ? y : ys[k]; sb_[k] = mine ? gb : sb_[k]; sa_[k] = mine ? ga : sa_[k];
                if (!L.in) {
#pragma unroll
                    for (int m = 0; m < 4; ++m) { vb[m] = 0.f; vc[m] = 0.f; }
                }
                wave_fold<LPC>(vb, vc);
                if ((lane & 15) < LPC) {
                    float* w2 = red[wave] + i * W + (lane >> 5) * N4 + 4 * L.j + 2 * ((lane >> 4) & 1);
                    w2[0] = vb[0]; w2[1] = vb[1];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = t0 + 4 * k + L.q;
            const bool live = r >= lo && r < min(hi, c1);
            const float raw = (float)raw_d[k] + bias;
            const float slope = a.softplus ? seq_sigmoid(raw) : 1.f;
            const float du = fmaf(Dd, dy[k], st[k] * sb_[k]);
            const float dd = live ? fmaf(u[k], sb_[k], SEQ_LN2 * sa_[k]) * slope : 0.f;
            dbias += dd;
            dD = fmaf(dy[k], u[k], dD);
            if (r < c1 && L.in && L.j < 4) {
                ((T*)a.du)[(int64_t)r * a.lddu + L.d] = (T)du;
                ((T*)a.ddelta)[(int64_t)r * a.lddd + L.d] = (T)dd;
                if (a.z) {
                    const float z = (float)raw_z[k], sg = seq_sigmoid(z);
                    const float dz = (float)raw_y[k] * fmaf(Dd, u[k], ys[k]) * sg * fmaf(z, 1.f - sg, 1.f);
                    ((T*)a.dz)[(int64_t)r * a.lddz + L.d] = (T)(live ? dz : 0.f);
                }
            }
        }
        __syncthreads();                                          // red complete; sB / sC of the next tile staged
        for (int e = threadIdx.x; e < SCAN_TILE * W; e += 256) {
            const int r = t0 + e / W;
            if (r < c1) a.part_bc[((int64_t)blockIdx.x * a.rows + r) * W + e % W] = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
        }
        __syncthreads();                                          // red read
    }
    if (a.dstate && L.in && chunk == 0) {                         // empty clips in front of the first row
        const int s0 = seq_find(a.clips, 0);
        for (int e = 0; e < s0 && e < n; ++e) empty(e);
    }
    dD += seq_dpp<0xB1>(dD); dD += seq_dpp<0x4E>(dD);
    dbias += seq_dpp<0xB1>(dbias); dbias += seq_dpp<0x4E>(dbias);
    if (L.in) {
        float* part = a.part_p + (int64_t)chunk * a.channels * (N + 2);
        scan_store4(part + (size_t)L.d * N, L.j, N, dA);
        if (L.j == 0) { part[(size_t)a.channels * N + L.d] = dD; part[(size_t)a.channels * (N + 1) + L.d] = dbias; }
    }
}

// dB and dC: the channel blocks' sums, added in block order
template <typename T>
__global__ __launch_bounds__(256) void k_scan_bc(const float* __restrict__ part, int blocks, int rows, int n4, int N,
                                                 T* __restrict__ dB, int64_t lddb, T* __restrict__ dC, int64_t lddc) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, width = (int64_t)rows * 2 * n4;
    if (e >= width) return;
    const int64_t r = e / (2 * n4);
    const int m = (int)(e - r * 2 * n4), c = m >= n4, i = c ? m - n4 : m;
    if (i >= N) return;
    float s0 = 0.f, s1 = 0.f;
    int b = 0;
    for (; b + 1 < blocks; b += 2) { s0 += part[b * width + e]; s1 += part[(b + 1) * width + e]; }
    if (b < blocks) s0 += part[b * width + e];
    if (c) dC[r * lddc + i] = (T)(s0 + s1); else dB[r * lddb + i] = (T)(s0 + s1);
}

// One token per clip.  A lane owns four states of a channel: it reads 16 bytes of state and writes 16.  VEC: N is a multiple
// of 4 and both states are 16-byte aligned.  state_out may be the state itself.
template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPC;
    const int j = threadIdx.x % LPC, N = a.n_state;
    const int64_t total = (int64_t)a.rows * a.channels;
    const bool in = at < total;
    const int64_t cell = in ? at : total - 1;
    const int s = (int)(cell / a.channels), d = (int)(cell - (int64_t)s * a.channels);
    float h[4], A[4], b[4], c[4];
    const float* src = a.state + cell * N;
    const bool mine = 4 * j < N;
    if constexpr (VEC) {
        seq_f4 v = {0.f, 0.f, 0.f, 0.f}, w = {0.f, 0.f, 0.f, 0.f};
        if (mine) { v = *(const seq_f4*)(src + 4 * j); w = *(const seq_f4*)(a.A + (size_t)d * N + 4 * j); }
#pragma unroll
        for (int i = 0; i < 4; ++i) { h[i] = v[i]; A[i] = w[i]; }
    } else { scan_load4(src, j, N, h); scan_load4(a.A + (size_t)d * N, j, N, A); }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        b[i] = 4 * j + i < N ? (float)((const T*)a.B)[(int64_t)s * a.ldb + 4 * j + i] : 0.f;
        c[i] = 4 * j + i < N ? (float)((const T*)a.C)[(int64_t)s * a.ldc + 4 * j + i] : 0.f;
    }
    const float u = (float)((const T*)a.u)[(int64_t)s * a.ldu + d];
    const float raw = (float)((const T*)a.delta)[(int64_t)s * a.ldd + d] + (a.bias ? a.bias[d] : 0.f);
    const float st = a.softplus ? scan_softplus(raw) : raw, x = st * u;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = fmaf(seq_exp2(st * (A[i] * SEQ_LOG2E)), h[i], x * b[i]);
        acc = fmaf(c[i], h[i], acc);
    }
    acc = chan_sum<LPC>(acc);
    if (!in) return;
    float* dst = a.final_state + cell * N;
    if constexpr (VEC) { if (mine) *(seq_f4*)(dst + 4 * j) = seq_f4{h[0], h[1], h[2], h[3]}; }
    else scan_store4(dst, j, N, h);
    if (j == 0) {
        float y = fmaf(a.D ? a.D[d] : 0.f, u, acc);
        if (a.z) { const float z = (float)((const T*)a.z)[(int64_t)s * a.ldz + d]; y *= z * seq_sigmoid(z); }
        ((T*)a.y)[(int64_t)s * a.ldy + d] = (T)y;
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------
static int scan_lpc(int n_state) { return n_state <= 16 ? 4 : n_state <= 32 ? 8 : 16; }

// Rows of a chunk: as many chunks as bring the launch to `target` workgroups, none shorter than 64 rows.
static void scan_chunks(int64_t rows, int channels, int n_state, int backward, int* chunk_rows, int* chunks) {
    const int per = 256 / scan_lpc(n_state);
    const int64_t groups = (channels + per - 1) / per, target = backward ? 1024 : 1024;
    int64_t want = (target + groups - 1) / groups, most = (rows + 63) / 64;
    if (want > most) want = most;
    if (want < 1) want = 1;
    int64_t r = ((rows + want - 1) / want + SCAN_TILE - 1) / SCAN_TILE * SCAN_TILE;
    if (r < SCAN_TILE) r = SCAN_TILE;
    *chunk_rows = (int)r;
    *chunks = rows ? (int)((rows + r - 1) / r) : 1;
}

static bool scan_shape_ok(int64_t rows, int channels, int n_state, int dtype) {
    return rows >= 0 && rows <= 0x7fffff00 && channels >= 1 && channels <= (1 << 20) && n_state >= 1 && n_state <= SCAN_MAX_STATE &&
           dtype >= 0 && dtype <= 2;
}

static int64_t scan_carry_floats(int chunks, int channels, int n_state) {
    if (chunks <= 1) return 4;
    const int n4 = 4 * scan_lpc(n_state);
    return (int64_t)chunks * channels * n4 + (((int64_t)chunks * channels + 3) & ~3LL) + ((chunks + 3) & ~3);
}
static void scan_carry(ScanArgs& a, float* ws) {
    const int n4 = 4 * scan_lpc(a.n_state);
    a.carry = ws;
    a.span = ws + (int64_t)a.chunks * a.channels * n4;
    a.flag = (int*)(a.span + (((int64_t)a.chunks * a.channels + 3) & ~3LL));
}

template <int WHAT, typename T, int LPC> static int scan_launch2(const ScanArgs& a, hipStream_t st) {
    constexpr int per = 256 / LPC;
    const dim3 grid((a.channels + per - 1) / per, a.chunks), block(256);
    if constexpr (WHAT == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_fwd<T, LPC, 0>), grid, block, 0, st, a);
    if constexpr (WHAT == 1) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_fwd<T, LPC, 1>), grid, block, 0, st, a);
    if constexpr (WHAT == 2) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_adj<T, LPC>), grid, block, 0, st, a);
    if constexpr (WHAT == 3) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_bwd<T, LPC>), grid, block, 0, st, a);
    if constexpr (WHAT == 4) {
        const bool vec = a.n_state % 4 == 0 && seq_aligned(a.state, 0) && seq_aligned(a.final_state, 0) && seq_aligned(a.A, 0);
        const dim3 g(evad_blocks((long long)a.rows * a.channels * LPC, 256));
        if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<T, LPC, true>), g, block, 0, st, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<T, LPC, false>), g, block, 0, st, a);
    }
    return evad_last_error();
}
template <int WHAT, typename T> static int scan_launch1(const ScanArgs& a, hipStream_t st) {
    switch (scan_lpc(a.n_state)) {
        case 4: return scan_launch2<WHAT, T, 4>(a, st);
        case 8: return scan_launch2<WHAT, T, 8>(a, st);
        default: return scan_launch2<WHAT, T, 16>(a, st);
    }
}
template <int WHAT> static int scan_launch(const ScanArgs& a, int dtype, hipStream_t st) {
    if (dtype == SEQ_F32) return scan_launch1<WHAT, float>(a, st);
    if (dtype == SEQ_BF16) return scan_launch1<WHAT, __bf16>(a, st);
    return scan_launch1<WHAT, _Float16>(a, st);
}
template <int REV> static void scan_join(const ScanArgs& a, hipStream_t st) {
    const int n4 = 4 * scan_lpc(a.n_state);
    hipLaunchKernelGGL(k_scan_join<REV>, dim3(evad_blocks((long long)a.channels * n4, 256)), dim3(256), 0, st, a, n4);
}

extern "C" int eventad_selective_scan_workspace(int64_t rows, int channels, int n_state, int backward, int64_t* bytes) {
    if (!bytes || !scan_shape_ok(rows, channels, n_state, 0)) return EVAD_ERR_ARG;
    int cr, chunks;
    scan_chunks(rows, channels, n_state, backward, &cr, &chunks);
    int64_t f = scan_carry_floats(chunks, channels, n_state);
    if (backward) {
        const int per = 256 / scan_lpc(n_state), n4 = 4 * scan_lpc(n_state);
        const int64_t groups = (channels + per - 1) / per, cols = (int64_t)channels * (n_state + 2);
        f += groups * rows * 2 * n4 + (chunks + SEQ_SUM_PARTS) * cols;
    }
    *bytes = f * 4;
    return EVAD_OK;
}

extern "C" int eventad_selective_scan_checkpoint(int64_t rows, int channels, int n_state, int64_t* bytes) {
    if (!bytes || !scan_shape_ok(rows, channels, n_state, 0)) return EVAD_ERR_ARG;
    *bytes = (rows + SCAN_TILE - 1) / SCAN_TILE * channels * 16 * scan_lpc(n_state);
    return EVAD_OK;
}

static bool scan_common(ScanArgs& a, const void* u, int64_t ldu, const void* delta, int64_t ldd, const float* A, const void* B,
                        int64_t ldb, const void* C, int64_t ldc, const float* D, const void* z, int64_t ldz, const float* bias,
                        int64_t rows, int channels, int n_state, int softplus, int dtype) {
    if (!scan_shape_ok(rows, channels, n_state, dtype) || !A || softplus < 0 || softplus > 1) return false;
    if (rows && (!u || !delta || !B || !C || ldu < channels || ldd < channels || ldb < n_state || ldc < n_state || (z && ldz < channels))) return false;
    a.u = u; a.ldu = ldu; a.delta = delta; a.ldd = ldd; a.A = A; a.B = B; a.ldb = ldb; a.C = C; a.ldc = ldc; a.D = D;
    a.z = z; a.ldz = ldz; a.bias = bias; a.rows = (int)rows; a.channels = channels; a.n_state = n_state; a.softplus = softplus;
    return true;
}

extern "C" int eventad_selective_scan_fwd(const void* u, int64_t ldu, const void* delta, int64_t ldd, const float* A, const void* B,
                                          int64_t ldb, const void* C, int64_t ldc, const float* D, const void* z, int64_t ldz,
                                          const float* delta_bias, const int32_t* clip_start, int clips, const float* state,
                                          float* final_state, void* y, int64_t ldy, float* checkpoint, void* workspace,
                                          int64_t workspace_bytes, int64_t rows, int channels, int n_state, int softplus, int dtype,
                                          void* stream) {
    ScanArgs a = {};
    int64_t need = 0;
    if (!scan_common(a, u, ldu, delta, ldd, A, B, ldb, C, ldc, D, z, ldz, delta_bias, rows, channels, n_state, softplus, dtype) ||
        clips < 1 || (!clip_start && clips != 1) || (rows && (!y || ldy < channels)) || ((uintptr_t)checkpoint & 15) ||
        eventad_selective_scan_workspace(rows, channels, n_state, 0, &need) != EVAD_OK || !workspace || workspace_bytes < need ||
        ((uintptr_t)workspace & 15)) return EVAD_ERR_ARG;
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.state = state; a.final_state = final_state; a.y = y; a.ldy = ldy; a.ckpt = checkpoint;
    scan_chunks(rows, channels, n_state, 0, &a.chunk_rows, &a.chunks);
    if (!rows && !final_state) return EVAD_OK;
    scan_carry(a, (float*)workspace);
    hipStream_t st = (hipStream_t)stream;
    if (a.chunks > 1) {
        const int rc = scan_launch<1>(a, dtype, st);
        if (rc) return rc;
        scan_join<0>(a, st);
    }
    return scan_launch<0>(a, dtype, st);
}

extern "C" int eventad_selective_scan_bwd(const void* u, int64_t ldu, const void* delta, int64_t ldd, const float* A, const void* B,
                                          int64_t ldb, const void* C, int64_t ldc, const float* D, const void* z, int64_t ldz,
                                          const float* delta_bias, const int32_t* clip_start, int clips, const float* state,
                                          const float* checkpoint, const void* dy, int64_t lddy, const float* dfinal, void* du,
                                          int64_t lddu, void* ddelta, int64_t lddd, void* dB, int64_t lddb, void* dC, int64_t lddc,
                                          void* dz, int64_t lddz, float* dstate, float* dparams, void* workspace,
                                          int64_t workspace_bytes, int64_t rows, int channels, int n_state, int softplus, int dtype,
                                          void* stream) {
    ScanArgs a = {};
    int64_t need = 0;
    if (!scan_common(a, u, ldu, delta, ldd, A, B, ldb, C, ldc, D, z, ldz, delta_bias, rows, channels, n_state, softplus, dtype) ||
        clips < 1 || (!clip_start && clips != 1) || !dparams || ((uintptr_t)checkpoint & 15) ||
        (rows && (!dy || !du || !ddelta || !dB || !dC || !checkpoint || lddy < channels || lddu < channels || lddd < channels ||
                  lddb < n_state || lddc < n_state || (z && (!dz || lddz < channels)))) ||
        eventad_selective_scan_workspace(rows, channels, n_state, 1, &need) != EVAD_OK || !workspace || workspace_bytes < need ||
        ((uintptr_t)workspace & 15)) return EVAD_ERR_ARG;
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.state = state; a.ckpt = (float*)checkpoint; a.dy = dy; a.lddy = lddy; a.dfinal = dfinal; a.du = du; a.lddu = lddu;
    a.ddelta = ddelta; a.lddd = lddd; a.dz = dz; a.lddz = lddz; a.dstate = dstate;
    scan_chunks(rows, channels, n_state, 1, &a.chunk_rows, &a.chunks);
    float* ws = (float*)workspace;
    scan_carry(a, ws);
    const int per = 256 / scan_lpc(n_state), n4 = 4 * scan_lpc(n_state), groups = (channels + per - 1) / per;
    const int64_t cols = (int64_t)channels * (n_state + 2);
    a.part_bc = ws + scan_carry_floats(a.chunks, channels, n_state);
    a.part_p = a.part_bc + (int64_t)groups * rows * 2 * n4;
    hipStream_t st = (hipStream_t)stream;
    if (a.chunks > 1) {
        const int rc = scan_launch<2>(a, dtype, st);
        if (rc) return rc;
        scan_join<1>(a, st);
    }
    int rc = scan_launch<3>(a, dtype, st);
    if (rc) return rc;
    if (rows) {
        const dim3 grid(evad_blocks((long long)rows * 2 * n4, 256));
        if (dtype == SEQ_F32) hipLaunchKernelGGL(k_scan_bc<float>, grid, dim3(256), 0, st, a.part_bc, groups, (int)rows, n4, n_state, (float*)dB, lddb, (float*)dC, lddc);
        else if (dtype == SEQ_BF16) hipLaunchKernelGGL(k_scan_bc<__bf16>, grid, dim3(256), 0, st, a.part_bc, groups, (int)rows, n4, n_state, (__bf16*)dB, lddb, (__bf16*)dC, lddc);
        else hipLaunchKernelGGL(k_scan_bc<_Float16>, grid, dim3(256), 0, st, a.part_bc, groups, (int)rows, n4, n_state, (_Float16*)dB, lddb, (_Float16*)dC, lddc);
        rc = evad_last_error();
        if (rc) return rc;
    }
    return seq_colsum(a.part_p, a.chunks, cols, dparams, a.part_p + a.chunks * cols, st);
}

extern "C" int eventad_selective_scan_step(const void* u, int64_t ldu, const void* delta, int64_t ldd, const float* A, const void* B,
                                           int64_t ldb, const void* C, int64_t ldc, const float* D, const void* z, int64_t ldz,
                                           const float* delta_bias, const float* state, float* state_out, void* y, int64_t ldy,
                                           int clips, int channels, int n_state, int softplus, int dtype, void* stream) {
    ScanArgs a = {};
    if (!scan_common(a, u, ldu, delta, ldd, A, B, ldb, C, ldc, D, z, ldz, delta_bias, clips, channels, n_state, softplus, dtype) ||
        (clips && (!state || !state_out || !y || ldy < channels))) return EVAD_ERR_ARG;
    if (!clips) return EVAD_OK;
    a.state = state; a.final_state = state_out; a.y = y; a.ldy = ldy;
    return scan_launch<4>(a, dtype, (hipStream_t)stream);
}
