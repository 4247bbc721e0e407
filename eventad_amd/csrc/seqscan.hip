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
// Layout: LPC lanes share a channel and hold ST of its states each in registers (4 x 1 / 2 / 4 for N <= 4 / 8 / 16, 8 x 4 and 16 x 4
// for N <= 32 / 64), so a wave has 64 / LPC channels and a 256-thread workgroup 256 / LPC.  Rows go by in tiles of 16: the four lanes of a quad form the
// step sizes of four different rows (softplus, gate and conversions once per row and channel, not once per lane) and hand
// them round with DPP; B and C of the tile stand in LDS as floats, read as one 16-byte access per lane and row.
//
// What bounds it is the vector ALU: per row, channel and state one v_exp_f32 (17.5 T lane operations per second on this chip) and
// four others (50 T), in the gradient one and thirteen, against 8 bytes per row and channel in 16 bits.  A long row axis is
// therefore split into chunks only as far as the chip needs workgroups: the chunks' own end states come from a first pass
// (without C, gate or output), are joined by a short one, and the second pass starts every chunk from its true state.  The
// adjoint g is split the same way, from the end.
//
// Measured, 16 states: 16384 x 1024 bf16 62 us first pass + 7 join + 94 second pass; the operations above would take 37 for one
// pass.  500,000 x 64 f32 117 + 13 + 183 us (the second pass 575 MB, 3.1 TB/s).  Gradient of 16001 x 1024 bf16 67 us adjoint +
// 8 + 281 + 13 for the sums; the operations would take 85.  The passes keep the ALU about 75 % issuing; a layout with a channel's 16
// states in one lane (no broadcasts, sums over channels across the whole wave) takes the same time, more waves per SIMD spill.
//
// Every sum over rows or channels is in float32 and in a fixed order (no atomics): results are reproducible bit for bit.
#include "seq.h"

#define SCAN_TILE 16
#define SCAN_KEEP 8                  // rows per checkpoint: the backward pass holds that many rows in registers
#define SCAN_MAX_STATE 64

struct ScanArgs {
    SeqClips clips;
    const void *u, *delta, *z, *B, *C;
    int64_t ldu, ldd, ldz, ldb, ldc;
    const float *A, *D, *bias, *state;
    float* final_state;
    void* y; int64_t ldy;
    float* ckpt;                                     // [rows / 8][channels][ST LPC]: the state in front of every 8th row
    float* carry; float* span; int* flag;            // per chunk: [channels][ST LPC] end state, [channels] sum of s, 1 = stands alone
    int rows, channels, n_state, chunk_rows, chunks, softplus;
    // gradient
    const void* dy; int64_t lddy;
    const float* dfinal; float* dstate;
    void *du, *ddelta, *dz; int64_t lddu, lddd, lddz;
    float* part_bc;                                  // [channel blocks][rows][2][ST LPC]
    float* part_p;                                   // [chunks][channels*N (dA) | channels (dD) | channels (dbias)]
};

// value of lane Q of the quad, in all four lanes
template <int Q> __device__ __forceinline__ float quad_bcast(float v) { return seq_dpp<Q * 0x55>(v); }
// (as a register of its own: a multiplication with a DPP operand issues at 0.6 of the rate of a plain one -- 31 against 50 T
// lane operations per second -- and every broadcast value is used four times)
__device__ __forceinline__ float quad_bcast(float v, int q) {
    float b = q == 0 ? quad_bcast<0>(v) : q == 1 ? quad_bcast<1>(v) : q == 2 ? quad_bcast<2>(v) : quad_bcast<3>(v);
    asm("" : "+v"(b));
    return b;
}
// Four rows' partial sums v[0..3] in the LPC lanes of a channel -> the sum of row q in every lane with quad position q: the
// quads are folded first (mirrored half rows and rows: the lane order inside a quad does not matter to the sum), then a quad
// exchanges halves twice, which takes 9 operations for four rows instead of 12 for a sum in all lanes and a select.
template <int LPC> __device__ __forceinline__ float quad_rows(float (&v)[4], int q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (LPC >= 8) v[i] += seq_dpp<0x141>(v[i]);
        if constexpr (LPC >= 16) v[i] += seq_dpp<0x140>(v[i]);
    }
    const bool odd = q & 1, high = q & 2;
    const float a = (odd ? v[1] : v[0]) + seq_dpp<0xB1>(odd ? v[0] : v[1]);
    const float b = (odd ? v[3] : v[2]) + seq_dpp<0xB1>(odd ? v[2] : v[3]);
    return (high ? b : a) + seq_dpp<0x4E>(high ? a : b);
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], with log1p(e) = 2 artanh(r), r = e / (2 + e) <= 1/3: relative
// accuracy for small e too, where log(1 + e) has none left.  artanh(r) / r is a polynomial of degree 4 in r^2 fitted to
// [0, 1/9] (relative error 4e-9; its series needs r^14 for as much).
__device__ __forceinline__ float scan_softplus(float x) {
    const float e = seq_exp2(-SEQ_LOG2E * fabsf(x));
    const float r = e * seq_rcp(2.f + e), q = r * r;
    float p = fmaf(q, 0.14089167f, 0.13980302f);
    p = fmaf(q, p, 0.20012455f);
    p = fmaf(q, p, 0.33333158f);
    p = fmaf(q, p, 1.f);
    return fmaf(2.f * r, p, fmaxf(x, 0.f));
}

// A as the exponent of 2.  A step of 0 stands for a row that leaves the state as it is, also where A is -inf (a state that forgets
// at once): the lowest finite number takes its place, with which every step of 1e-36 or more still gives exp(s A) = 0.
__device__ __forceinline__ float scan_decay(float A) {
    const float e = A * SEQ_LOG2E;
    return e < -3.4028235e38f ? -3.4028235e38f : e;              // (NaN stays)
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
// a lane's ST entries of a row of N floats
template <int ST> __device__ __forceinline__ void scan_load(const float* __restrict__ row, int j, int N, float (&v)[ST]) {
#pragma unroll
    for (int i = 0; i < ST; ++i) v[i] = ST * j + i < N ? row[ST * j + i] : 0.f;
}
template <int ST> __device__ __forceinline__ void scan_store(float* __restrict__ row, int j, int N, const float (&v)[ST]) {
#pragma unroll
    for (int i = 0; i < ST; ++i) if (ST * j + i < N) row[ST * j + i] = v[i];
}
// the same as one access
template <int ST> using ScanVec = typename SeqVec<float, ST>::type;
template <int ST> __device__ __forceinline__ ScanVec<ST> scan_vec(const float (&v)[ST]) {
    ScanVec<ST> r;
#pragma unroll
    for (int i = 0; i < ST; ++i) r[i] = v[i];
    return r;
}

// The same number, which the compiler takes for a new one: what is read or computed from it is neither moved out of
// a loop nor turned into a pointer per access that the loop carries along (16 rows of B and C alone are 128 registers, the
// addresses of a tile's rows 60).
__device__ __forceinline__ int scan_again(int v) { asm volatile("" : "+v"(v)); return v; }

// A lane's element of four rows of a tile: rows 4 k + q, channel d.  p, the tile's first row, and step, four rows, are the same
// for the whole wave: one scalar base and one 32-bit offset per access, and no 64-bit arithmetic on the way.
template <typename T> struct ScanRows {
    char* p; unsigned step, at;
    __device__ __forceinline__ ScanRows(const void* base, int64_t ld, int t0, int q, int d)
        : p((char*)base + (int64_t)t0 * ld * (int)sizeof(T)), step(4 * (unsigned)ld * sizeof(T)), at((unsigned)(q * (int)ld + d) * sizeof(T)) {}
    __device__ __forceinline__ T& row(int k) const { return *(T*)(p + (scan_again(at) + k * step)); }
    __device__ __forceinline__ void fetch(T (&v)[4], bool full, int left) const {                // left: rows of the lane's
        if (full) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = row(k);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = (T)0.f; if (4 * k < left) v[k] = row(k); }
        }
    }
    template <int DIR> __device__ __forceinline__ void move(bool go) { const unsigned by = go ? 4u * step : 0u; p = DIR > 0 ? p + by : p - by; }
};

// B or C of a tile on their way to LDS as floats: requested a tile ahead, written when the rows in front are done.  A thread
// takes one state of every (256 / N4)th row; rows of no clip and states >= N become zero.
template <typename T, int N4> struct ScanStage {
    static constexpr int ALL = SCAN_TILE * N4, PER = (ALL + 255) / 256, STEP = 256 / N4;
    char* p; unsigned tile, at; bool in;             // tile: bytes from a tile to the next (2^30 at a row stride of 2^24)
    T v[PER];
    __device__ __forceinline__ ScanStage(const void* base, int64_t ld, int t0, int N)
        : p((char*)base + (int64_t)t0 * ld * (int)sizeof(T)), tile(SCAN_TILE * (unsigned)ld * sizeof(T)), in(threadIdx.x % N4 < N) {
        at = (unsigned)(threadIdx.x / N4 * (int)ld + min((int)threadIdx.x % N4, N - 1)) * sizeof(T);
    }
    __device__ __forceinline__ void load(bool full, int left) {                                  // left: rows of the tile
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            v[i] = (T)0.f;
            if ((full || (int)threadIdx.x / N4 + i * STEP < left) && (ALL >= 256 || (int)threadIdx.x < ALL)) v[i] = *(const T*)(p + (scan_again(at) + i * (tile / PER)));
        }
    }
    __device__ __forceinline__ void store(float* __restrict__ s, int t0, int lo, int hi) const {
        const bool clean = t0 >= lo && t0 + SCAN_TILE <= hi;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int r = t0 + threadIdx.x / N4 + i * STEP;
            if (ALL >= 256 || (int)threadIdx.x < ALL) s[threadIdx.x + 256 * i] = in && (clean || (r >= lo && r < hi)) ? (float)v[i] : 0.f;
        }
    }
    template <int DIR> __device__ __forceinline__ void move(bool go) {
        const unsigned by = go ? tile : 0u;
        p = DIR > 0 ? p + by : p - by;
    }
};

// B or C of a pair of rows, read from LDS a pair ahead (and, with a scheduling barrier behind the reads, not more: the
// registers would cost waves in flight)
template <int N4, int ST> struct ScanPair {
    const float* p; ScanVec<ST> v[2][2];
    __device__ __forceinline__ ScanPair(const float* at, int k = 0) : p(at) { read(k); }
    __device__ __forceinline__ void read(int k) {
        v[k & 1][0] = *(const ScanVec<ST>*)(p + 2 * k * N4);
        v[k & 1][1] = *(const ScanVec<ST>*)(p + (2 * k + 1) * N4);
    }
    __device__ __forceinline__ void ahead(int k) { if (k >= 0 && k < SCAN_TILE / 2) read(k); }
    __device__ __forceinline__ ScanVec<ST> row(int i) const { return v[(i >> 1) & 1][i & 1]; }
};

// Rows at .. end-1 of a staged tile, zeros in the place of the others.  A piece that shares its tile with another clip reads this
// copy: its own input and step of the other rows are zero, but a B or C that is infinite or no number there would get through.
template <int N4> __device__ __forceinline__ void scan_mask(float* dst, const float* src, int t0, int at, int end) {
#pragma unroll
    for (int e = threadIdx.x; e < SCAN_TILE * N4; e += 256) {
        const int r = t0 + e / N4;
        dst[e] = r >= at && r < end ? src[e] : 0.f;
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

// WHAT 0: outputs.  WHAT 1: the chunk's end state for the chunks behind it.  Four workgroups per CU; with 16 lanes per channel three,
// as their staging registers would be spilled at four (16384 x 1024 x 64 bf16: 690 us against 710).  With fewer lanes three cost more than
// the spills of the first pass (two registers with 4 lanes, six with 8): x 16 160 us against 153, x 24 315 against 307.
//
// A chunk is walked in pieces, the rows that a tile and a clip have in common.  A piece runs through all 16 rows of its
// tile as straight-line code, with step and input 0 for rows outside it, which leave the state as it is: the usual tile is one
// piece, a clip's end inside a tile costs one more, and there is no branch between two rows that would keep the reads
// of B and C from being requested ahead.
template <typename T, int LPC, int ST, int WHAT>
__global__ __launch_bounds__(256, LPC > 8 ? 3 : 4) void k_scan_fwd(ScanArgs a) {
    constexpr int N4 = ST * LPC;
    __shared__ __attribute__((aligned(16))) float sB[WHAT == 0 ? 3 : 2][SCAN_TILE * N4], sC[WHAT == 0 ? 3 : 1][SCAN_TILE * N4];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y;
    const int c0 = chunk * a.chunk_rows, c1 = c0 + min(a.chunk_rows, a.rows - c0);
    float A2[ST], h[ST];
#pragma unroll
    for (int m = 0; m < ST; ++m) h[m] = 0.f;
    scan_load(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < ST; ++i) A2[i] = scan_decay(A2[i]);
    const float bias = a.bias ? a.bias[L.d] : 0.f, Dd = WHAT == 0 && a.D ? a.D[L.d] : 0.f;
    auto entry = [&](int s) {                                    // the state in front of clip s
#pragma unroll
        for (int m = 0; m < ST; ++m) h[m] = 0.f;
        if (a.state && s >= 0 && s < n) scan_load(a.state + ((size_t)s * a.channels + L.d) * N, L.j, N, h);
    };
    auto leave = [&](int s) {                                    // h is the state behind clip s
        if (a.final_state && s >= 0 && s < n && L.in) scan_store(a.final_state + ((size_t)s * a.channels + L.d) * N, L.j, N, h);
    };

    ScanWalk w = scan_walk(a.clips, WHAT == 1 ? c1 - 1 : c0);
    const int first = w.s >= 0 ? seq_start(a.clips, w.s) : 0;
    int at = c0;                                                 // first row of the next piece
    if constexpr (WHAT == 1) {
        // only the rows since the last clip start of the chunk matter, and none if the next chunk starts with a clip of its own
        const bool none = w.s < 0 || w.s >= n || w.next <= c1;
        if (blockIdx.x == 0 && threadIdx.x == 0) a.flag[chunk] = none || first >= c0;
        if (none) {
            if (L.in) scan_store(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, h);
            return;
        }
        if (first >= c0) { at = first; entry(w.s); }
        w.next = 0x7fffffff;
    } else {
        if (a.final_state)                                       // empty clips at the chunk's first row keep their state
            for (int e = w.s - 1; e >= 0 && seq_start(a.clips, e) == c0; --e) { entry(e); leave(e); }
        if (w.s >= 0 && w.s < n && first < c0 && chunk > 0) scan_load(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, h);
        else entry(w.s);
    }
    if (c1 <= c0) return;
    // rows that belong to a clip (WHAT 1: to the one that matters)
    const int lo = WHAT == 1 ? at : seq_start(a.clips, 0), hi = min(c1, seq_start(a.clips, n));
    const bool gated = WHAT == 0 && a.z;
    int t0 = at / SCAN_TILE * SCAN_TILE, buf = 0;
    ScanRows<T> fu(a.u, a.ldu, t0, L.q, L.d), fd(a.delta, a.ldd, t0, L.q, L.d), fz(a.z, a.ldz, t0, L.q, L.d), oy(a.y, a.ldy, t0, L.q, L.d);
    float span = 0.f;
    T ru[4], rd[4], rz[4];
    ScanStage<T, N4> stB(a.B, a.ldb, t0, N), stC(a.C, a.ldc, t0, N);
    auto fetch = [&](int t) {
        const bool full = t + SCAN_TILE <= a.rows;
        const int left = a.rows - t;
        fu.fetch(ru, full, left - L.q);
        fd.fetch(rd, full, left - L.q);
        if (gated) fz.fetch(rz, full, left - L.q);
        stB.load(full, left);
        if (WHAT == 0) stC.load(full, left);
    };
    fetch(t0);
    stB.store(sB[0], t0, lo, hi);
    if constexpr (WHAT == 0) stC.store(sC[0], t0, lo, hi);
    __syncthreads();
    for (; t0 < c1; t0 += SCAN_TILE, buf ^= 1) {
        float st[4], u[4], gate[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u[k] = (float)ru[k];
            const float raw = (float)rd[k] + bias;
            st[k] = a.softplus ? scan_softplus(raw) : raw;
            gate[k] = 1.f;
            if (gated) { const float z = (float)rz[k]; gate[k] = z * seq_sigmoid(z); }
        }
        // (WHAT 1: the last tile requests itself again; without a branch here and at the store the rows stay one block of code)
        const bool more = t0 + SCAN_TILE < c1;
        const int t2 = more ? t0 + SCAN_TILE : t0;
        if (WHAT == 1 || more) {
            fu.template move<1>(more); fd.template move<1>(more); stB.template move<1>(more);
            if (WHAT == 0) { fz.template move<1>(true); stC.template move<1>(true); }
            fetch(t2);
        }
        auto keep = [&](int row) {                               // the state in front of the row, for the backward pass
            if (WHAT == 0 && a.ckpt && L.in) *(ScanVec<ST>*)(a.ckpt + ((size_t)(row / SCAN_KEEP) * a.channels + L.d) * N4 + ST * L.j) = scan_vec(h);
        };
        keep(t0);
        const int t1 = min(t0 + SCAN_TILE, c1);
        do {                                                     // the tile's pieces: rows at .. end-1
            const int end = min(t1, w.next);
            const bool whole = at == t0 && end == t0 + SCAN_TILE, live = at >= lo && at < hi;    // (of a clip, or of none)
            int use = buf;
            if (WHAT == 0 && !whole) {
                use = 2;
                __syncthreads();                                 // (the piece in front has read its copy)
                scan_mask<N4>(sB[use], sB[buf], t0, at, end);
                if constexpr (WHAT == 0) scan_mask<N4>(sC[use], sC[buf], t0, at, end);
                __syncthreads();
            }
            const float *tB = sB[use] + scan_again(ST * L.j), *tC = WHAT == 0 ? sC[use] + scan_again(ST * L.j) : tB;
            float s4[4], x4[4], ys[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { s4[k] = st[k]; x4[k] = st[k] * u[k]; }
            if (!whole || !live) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = t0 + 4 * k + L.q;
                    const bool mine = live && r >= at && r < end;
                    s4[k] = mine ? s4[k] : 0.f; x4[k] = mine ? x4[k] : 0.f;
                }
            }
            ScanPair<N4, ST> gB(tB), gC(WHAT == 0 ? tC : tB);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float acc[4];
                if constexpr (WHAT == 1) span += s4[k];
                if (k == 2 && at <= t0 + SCAN_KEEP && end > t0 + SCAN_KEEP) keep(t0 + SCAN_KEEP);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (q % 2 == 0) {
                        gB.ahead(2 * k + q / 2 + 1);
                        if constexpr (WHAT == 0) gC.ahead(2 * k + q / 2 + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    const float sb = quad_bcast(s4[k], q), xb = quad_bcast(x4[k], q);
                    const ScanVec<ST> b4 = gB.row(4 * k + q), c4 = gC.row(4 * k + q);
#pragma unroll
                    for (int m = 0; m < ST; ++m) {
                        h[m] = fmaf(seq_exp2(sb * A2[m]), h[m], xb * b4[m]);
                        if constexpr (WHAT == 0) acc[q] = m ? fmaf(c4[m], h[m], acc[q]) : c4[0] * h[0];
                    }
                }
                if constexpr (WHAT == 0) ys[k] = quad_rows<LPC>(acc, L.q);
            }
            if constexpr (WHAT == 0) {
                if (L.in && L.j < 4) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = t0 + 4 * k + L.q;
                        const float y = fmaf(Dd, u[k], ys[k]) * gate[k];
                        if (whole || (r >= at && r < end)) oy.row(k) = (T)(live ? y : 0.f);
                    }
                }
                if (end >= w.next && w.s < n) {                  // a clip ended with the piece
                    leave(w.s);
                    if (end < c1 || c1 == a.rows) {              // (clips that start with the next chunk are its own)
                        ++w.s;
                        while (w.s < n && seq_start(a.clips, w.s + 1) <= end) { entry(w.s); leave(w.s); ++w.s; }
                        w.next = w.s < n ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, w.s + 1)) : 0x7fffffff;
                        if (end < c1) entry(w.s);
                    }
                }
            }
            at = end;
        } while (at < t1);
        if (WHAT == 0) oy.template move<1>(true);
        if (WHAT == 1 || more) {
            stB.store(sB[buf ^ 1], t2, lo, hi);
            if constexpr (WHAT == 0) stC.store(sC[buf ^ 1], t2, lo, hi);
        }
        __syncthreads();
    }
    if constexpr (WHAT == 1) {
        if (L.in) {
            scan_store(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, h);
            span += seq_dpp<0xB1>(span);
            span += seq_dpp<0x4E>(span);
            if (L.j == 0) a.span[(size_t)chunk * a.channels + L.d] = span;
        }
    }
}

// The chunks' true entry states.  carry[chunk] holds the chunk's own contribution on entry and what flows into the chunk on
// return (REV: from the last chunk to the first).  A workgroup takes 16 (channel, state) columns; its G groups of 16 lanes read
// their share of the chunks at once and compose it, G lanes per column compose the shares, and each group goes over its share
// again, out of registers: one wait for memory.  64 groups beyond 256 chunks, 16 up to there: 1009 chunks of 64 channels x 16 13 us
// (16 groups that read twice 23, one thread per column 92), 63 chunks of 1024 channels 7.3 (64 groups 11).
#define JOIN_SHARE 16                // chunks of a group
// the state behind a stretch that passes on the factor `pass` (< 0: a clip starts in it) and adds `own`; a state of zero stays zero
// whatever the factor
__device__ __forceinline__ float join_past(float pass, float in, float own) { return pass < 0.f || in == 0.f ? own : fmaf(pass, in, own); }
template <int REV, int G>
__global__ __launch_bounds__(16 * G) void k_scan_join(ScanArgs a, int n4) {
    __shared__ float s_own[G][17], s_pass[G][17];
    const int col = threadIdx.x & 15, group = threadIdx.x >> 4, one = threadIdx.x / G, lane = threadIdx.x % G;
    const int64_t width = (int64_t)a.channels * n4, place = (int64_t)blockIdx.x * 16 + col, at = place < width ? place : width - 1;
    const int d = (int)(at / n4), i = (int)(at - (int64_t)d * n4);
    const float A2 = i < a.n_state ? scan_decay(a.A[(size_t)d * a.n_state + i]) : 0.f;
    const int share = (a.chunks + G - 1) / G, first = group * share, mine = min(share, a.chunks - first);
    float own[JOIN_SHARE], e[JOIN_SHARE], in = 0.f, pass = 1.f;
    int alone[JOIN_SHARE];
#pragma unroll
    for (int j = 0; j < JOIN_SHARE; ++j)
        if (j < share) {
            const int k = min(first + j, a.chunks - 1), c = REV ? a.chunks - 1 - k : k;
            own[j] = a.carry[c * width + at];
            e[j] = a.span[(size_t)c * a.channels + d];
            alone[j] = a.flag[c];
        }
#pragma unroll
    for (int j = 0; j < JOIN_SHARE; ++j)
        if (j < share && j < mine) {
            e[j] = alone[j] ? -1.f : seq_exp2(e[j] * A2);
            in = join_past(e[j], in, own[j]);
            pass = pass < 0.f || e[j] < 0.f ? -1.f : pass * e[j];
        }
    s_own[group][col] = in; s_pass[group][col] = pass;
    __syncthreads();
    float o = s_own[lane][one], p = s_pass[lane][one];
#pragma unroll
    for (int by = 1; by < G; by <<= 1) {
        const float o1 = __shfl_up(o, by, G), p1 = __shfl_up(p, by, G);
        if (lane >= by) {
            o = join_past(p, o1, o);
            p = p < 0.f || p1 < 0.f ? -1.f : p * p1;
        }
    }
    o = __shfl_up(o, 1, G);
    s_own[lane][one] = lane ? o : 0.f;
    __syncthreads();
    in = s_own[group][col];
#pragma unroll
    for (int j = 0; j < JOIN_SHARE; ++j)
        if (j < share && j < mine) {
            const int c = REV ? a.chunks - 1 - (first + j) : first + j;
            if (place < width) a.carry[c * width + at] = in;
            in = join_past(e[j], in, own[j]);
        }
}

// The adjoint of a chunk by itself: what its rows contribute to dL/dh in front of its first row.  The forward's first pass run
// backwards, without a gate's or u's part in it: 67 us for 16001 x 1024 x 16 bf16.  (More than four lanes per channel: three workgroups
// per CU, without spills, take 10 % less than four; the gradient behind it has two anyway.)
template <typename T, int LPC, int ST>
__global__ __launch_bounds__(256, LPC > 4 ? 3 : 4) void k_scan_adj(ScanArgs a) {
    constexpr int N4 = ST * LPC;
    __shared__ __attribute__((aligned(16))) float sC[2][SCAN_TILE * N4];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y;
    const int c0 = chunk * a.chunk_rows, c1 = c0 + min(a.chunk_rows, a.rows - c0);
    float A2[ST], g[ST];
#pragma unroll
    for (int m = 0; m < ST; ++m) g[m] = 0.f;
    scan_load(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < ST; ++i) A2[i] = scan_decay(A2[i]);
    const float bias = a.bias ? a.bias[L.d] : 0.f;
    const ScanWalk w = scan_walk(a.clips, c0);
    const bool dead = w.s < 0 || w.s >= n || seq_start(a.clips, w.s) >= c0;        // nothing flows out of the chunk
    const bool ends = w.next <= c1;                                                // the clip ends in it: nothing flows through
    if (blockIdx.x == 0 && threadIdx.x == 0) a.flag[chunk] = dead || ends ? 1 : 0;
    if (dead) {
        if (L.in) scan_store(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
        return;
    }
    const int to = min(w.next, c1);                                                // rows [c0, to)
    if (ends && a.dfinal) scan_load(a.dfinal + ((size_t)w.s * a.channels + L.d) * N, L.j, N, g);
    float span = 0.f;
    int t0 = (to - 1) / SCAN_TILE * SCAN_TILE, buf = 0;
    ScanRows<T> fd(a.delta, a.ldd, t0, L.q, L.d), fy(a.dy, a.lddy, t0, L.q, L.d), fz(a.z, a.ldz, t0, L.q, L.d);
    T rd[4], ry[4], rz[4];
    ScanStage<T, N4> stC(a.C, a.ldc, t0, N);
    auto fetch = [&](bool full) {
        const int left = a.rows - t0;
        fd.fetch(rd, full, left - L.q);
        fy.fetch(ry, full, left - L.q);
        if (a.z) fz.fetch(rz, full, left - L.q);
        stC.load(full, left);
    };
    fetch(t0 + SCAN_TILE <= a.rows);
    stC.store(sC[0], t0, c0, to);
    __syncthreads();
    for (; t0 >= c0; t0 -= SCAN_TILE, buf ^= 1) {
        float st[4], dy[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float raw = (float)rd[k] + bias;
            st[k] = a.softplus ? scan_softplus(raw) : raw;
            dy[k] = (float)ry[k];
            if (a.z) { const float z = (float)rz[k]; dy[k] *= z * seq_sigmoid(z); }
        }
        if (t0 + SCAN_TILE > to) {
#pragma unroll
            for (int k = 0; k < 4; ++k) { const bool live = t0 + 4 * k + L.q < to; st[k] = live ? st[k] : 0.f; dy[k] = live ? dy[k] : 0.f; }
        }
        // (the first tile requests itself again -- or, if it is a short last one of the array too, nothing anyone looks at)
        const int t2 = max(c0, t0 - SCAN_TILE);
        const bool down = t2 < t0;
        fd.template move<-1>(down); fy.template move<-1>(down); fz.template move<-1>(down); stC.template move<-1>(down);
        fetch(t2 + SCAN_TILE <= a.rows);
        ScanPair<N4, ST> gC(sC[buf] + ST * L.j, SCAN_TILE / 2 - 1);
#pragma unroll
        for (int k = 3; k >= 0; --k) {
            span += st[k];
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                if (q % 2 == 1) {
                    gC.ahead(2 * k + q / 2 - 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const float sb = quad_bcast(st[k], q), db = quad_bcast(dy[k], q);
                const ScanVec<ST> c4 = gC.row(4 * k + q);
#pragma unroll
                for (int m = 0; m < ST; ++m) g[m] = seq_exp2(sb * A2[m]) * fmaf(c4[m], db, g[m]);
            }
        }
        stC.store(sC[buf ^ 1], t2, c0, to);
        __syncthreads();
    }
    if (L.in) {
        scan_store(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
        span += seq_dpp<0xB1>(span);
        span += seq_dpp<0x4E>(span);
        if (L.j == 0) a.span[(size_t)chunk * a.channels + L.d] = span;
    }
}

// 2 ST values of every lane summed over the channels of the wave.  Swap-and-add steps fold the halves of the wave and the halves of
// each half while they halve the number of values (a swap serves two values), then DPP rotations add up the channels inside a
// row of 16 lanes.  Row r of 16 lanes returns sums of b (r < 2) or c in b[0 .. FOLD-1], of the states FOLD (r & 1) + 0 .. FOLD-1
// (ST = 1: of the one state, in both).
template <int LPC, int ST> __device__ __forceinline__ void wave_fold(float (&b)[ST], const float (&c)[ST]) {
    constexpr int FOLD = (ST + 1) / 2;
#pragma unroll
    for (int i = 0; i < ST; ++i) seq_swap32(b[i], c[i]);          // lanes 0..31: sums of b, lanes 32..63: sums of c
#pragma unroll
    for (int i = 0; i < FOLD; ++i) {
        seq_swap16(b[i], b[ST - FOLD + i]);                       // even rows of 16: entry i, odd rows: entry FOLD + i
        if constexpr (LPC <= 8) b[i] += seq_dpp<0x128>(b[i]);     // row_ror:8
        if constexpr (LPC <= 4) b[i] += seq_dpp<0x124>(b[i]);     // row_ror:4
    }
}

// The gradient of a chunk, from its last row to its first, in pieces like the forward's.  A piece takes its tile in halves: forward
// from the checkpoint, with e_t = exp(s_t A) and e_t h_{t-1} of the 8 rows kept in registers, then back with the adjoint.
// 227 registers, two waves per SIMD: 281 us for 16001 x 1024 x 16 bf16.  The sums over channels are a quarter of the operations;
// taking them through LDS halves those and leaves the time as it is (304 us against 305 in one run).
//
// What only the clips' borders need is read from the kernel's arguments where it is used (rare()): with all of them in scalar
// registers from the start, the loop moves a hundred scalars per tile in and out of vector registers.
typedef const __attribute__((address_space(4))) ScanArgs* ScanArgsPtr;
__device__ __forceinline__ ScanArgsPtr scan_rare() {
    ScanArgsPtr p = (ScanArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();                          // (the only argument)
    asm volatile("" : "+s"(p));
    return p;
}
__device__ __forceinline__ int seq_start(ScanArgsPtr p, int s) { const SeqClips c = {p->clips.start, p->clips.n, p->clips.rows}; return seq_start(c, s); }

template <typename T, int LPC, int ST>
__global__ __launch_bounds__(256, 2) void k_scan_bwd(ScanArgs a) {
    constexpr int N4 = ST * LPC, W = 2 * N4, FOLD = (ST + 1) / 2;
    __shared__ __attribute__((aligned(16))) float sB[3][SCAN_TILE * N4], sC[3][SCAN_TILE * N4], red[4][(SCAN_TILE + 1) * W];
    const ScanLane<LPC> L(a);
    const int N = a.n_state, n = a.clips.n, chunk = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int c0 = chunk * a.chunk_rows, c1 = c0 + min(a.chunk_rows, a.rows - c0);
    float A2[ST], g[ST], dA[ST], dD = 0.f, dbias = 0.f;
#pragma unroll
    for (int m = 0; m < ST; ++m) g[m] = dA[m] = 0.f;
    scan_load(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < ST; ++i) A2[i] = scan_decay(A2[i]);
    const float bias = a.bias ? a.bias[L.d] : 0.f, Dd = a.D ? a.D[L.d] : 0.f;
    auto entry = [&](int s) {                                     // the gradient of the state behind clip s
#pragma unroll
        for (int m = 0; m < ST; ++m) g[m] = 0.f;
        const ScanArgsPtr r = scan_rare();
        if (r->dfinal && s >= 0 && s < r->clips.n) scan_load(r->dfinal + ((size_t)s * r->channels + L.d) * N, L.j, N, g);
    };
    auto leave = [&](int s) {                                     // g is the gradient of the state in front of clip s
        const ScanArgsPtr r = scan_rare();
        if (r->dstate && s >= 0 && s < r->clips.n && L.in) scan_store(r->dstate + ((size_t)s * r->channels + L.d) * N, L.j, N, g);
    };
    // s = the clip of row end-1, first = its first row
    int s = __builtin_amdgcn_readfirstlane(seq_find(a.clips, c1 - 1));
    int first = s >= 0 ? __builtin_amdgcn_readfirstlane(seq_start(a.clips, s)) : 0;
    if (a.dstate)                                                 // empty clips between this chunk's last row and the next row
        for (int e = s + 1; e < n && seq_start(a.clips, e + 1) <= c1; ++e) { entry(e); leave(e); }
    if (s >= 0 && s < n && seq_start(a.clips, s + 1) > c1) {
        if (a.chunks > 1) scan_load(a.carry + ((size_t)chunk * a.channels + L.d) * N4, L.j, N4, g);
    } else entry(s);
    const int lo = seq_start(a.clips, 0), hi = min(c1, seq_start(a.clips, n));                    // rows that belong to a clip
    float* my_red = red[wave] + (lane >> 5) * N4 + ST * L.j + (ST > 1 ? FOLD * ((lane >> 4) & 1) : 0);               // (its last row takes what no row wants)
    const bool gated = a.z;
    int t0 = (c1 - 1) / SCAN_TILE * SCAN_TILE, buf = 0, end = c1;
    ScanRows<T> fu(a.u, a.ldu, t0, L.q, L.d), fd(a.delta, a.ldd, t0, L.q, L.d), fy(a.dy, a.lddy, t0, L.q, L.d), fz(a.z, a.ldz, t0, L.q, L.d);
    ScanRows<T> ou(a.du, a.lddu, t0, L.q, L.d), od(a.ddelta, a.lddd, t0, L.q, L.d), oz(a.dz, a.lddz, t0, L.q, L.d);
    T ru[4], rd[4], rz[4], ry[4];
    ScanVec<ST> kept[2];
    ScanStage<T, N4> stB(a.B, a.ldb, t0, N), stC(a.C, a.ldc, t0, N);
    const char* pk = (const char*)(a.ckpt + (size_t)(t0 / SCAN_KEEP) * a.channels * N4);
    const unsigned kept_step = (unsigned)a.channels * N4 * 4, kept_at = (unsigned)(L.d * N4 + ST * L.j) * 4;
    auto fetch = [&](bool full) {
        const int left = a.rows - t0;
        fu.fetch(ru, full, left - L.q);
        fd.fetch(rd, full, left - L.q);
        fy.fetch(ry, full, left - L.q);
        if (gated) fz.fetch(rz, full, left - L.q);
        stB.load(full, left);
        stC.load(full, left);
        kept[0] = *(const ScanVec<ST>*)(pk + scan_again(kept_at));
        kept[1] = ScanVec<ST>(0.f);
        if (full || left > SCAN_KEEP) kept[1] = *(const ScanVec<ST>*)(pk + kept_step + scan_again(kept_at));
    };
    if (c1 > c0) {
        fetch(t0 + SCAN_TILE <= a.rows);
        stB.store(sB[0], t0, lo, hi);
        stC.store(sC[0], t0, lo, hi);
    }
    __syncthreads();
    for (; c1 > c0 && t0 >= c0; t0 -= SCAN_TILE, buf ^= 1) {
        float st[4], u[4], dy[4];
        T raw_d[4], raw_z[4], raw_y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            raw_d[k] = rd[k]; raw_z[k] = rz[k]; raw_y[k] = ry[k];
            u[k] = (float)ru[k];
            const float raw = (float)rd[k] + bias;
            st[k] = a.softplus ? scan_softplus(raw) : raw;
            dy[k] = (float)ry[k];
            if (gated) { const float z = (float)rz[k]; dy[k] *= z * seq_sigmoid(z); }
        }
        const int t2 = max(c0, t0 - SCAN_TILE);
        const ScanVec<ST> k0 = kept[0], k1 = kept[1];
        do {                                                      // the tile's pieces: rows at .. end-1
            const int at = max(t0, first);
            const bool whole = at == t0 && end == t0 + SCAN_TILE, live = at >= lo && at < hi;     // (of a clip, or of none)
            int use = buf;
            if (!whole) {
                use = 2;
                __syncthreads();                                  // (the piece in front has read its copy)
                scan_mask<N4>(sB[2], sB[buf], t0, at, end);
                scan_mask<N4>(sC[2], sC[buf], t0, at, end);
                __syncthreads();
            }
            float s4[4], x4[4], d4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { s4[k] = st[k]; x4[k] = st[k] * u[k]; d4[k] = dy[k]; }
            if (!whole || !live || !L.in) {                       // (lanes past the last channel take part in the sums with zeros)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = t0 + 4 * k + L.q;
                    const bool mine = live && L.in && r >= at && r < end;
                    s4[k] = mine ? s4[k] : 0.f; x4[k] = mine ? x4[k] : 0.f; d4[k] = mine ? d4[k] : 0.f;
                }
            }
#pragma unroll
            for (int half = 1; half >= 0; --half) {
                const int h0 = t0 + half * SCAN_KEEP;
                if (at >= h0 + SCAN_KEEP || end <= h0) continue;
                const float* tB = sB[use] + scan_again(ST * L.j + half * SCAN_KEEP * N4);
                float h[ST], ex[SCAN_KEEP][ST], ah[SCAN_KEEP][ST];
#pragma unroll
                for (int m = 0; m < ST; ++m) h[m] = half ? k1[m] : k0[m];
                if (at == first && at >= h0) {                    // the clip starts here
#pragma unroll
                    for (int m = 0; m < ST; ++m) h[m] = 0.f;
                    const ScanArgsPtr r = scan_rare();
                    if (r->state && live) scan_load(r->state + ((size_t)s * r->channels + L.d) * N, L.j, N, h);
                }
#pragma unroll
                for (int i = 0; i < SCAN_KEEP; ++i) {
                    const int k = 2 * half + i / 4;
                    const float sb = quad_bcast(s4[k], i & 3), xb = quad_bcast(x4[k], i & 3);
                    const ScanVec<ST> b4 = *(const ScanVec<ST>*)(tB + i * N4);
#pragma unroll
                    for (int m = 0; m < ST; ++m) {
                        ex[i][m] = seq_exp2(sb * A2[m]);
                        ah[i][m] = ex[i][m] * h[m];
                        h[m] = fmaf(xb, b4[m], ah[i][m]);
                    }
                }
                if (half == 0 && at == t0) {                      // (the chunk's first tile requests itself again)
                    const bool down = t2 < t0;
                    fu.template move<-1>(down); fd.template move<-1>(down); fy.template move<-1>(down); fz.template move<-1>(down);
                    stB.template move<-1>(down); stC.template move<-1>(down);
                    pk -= down ? 2u * kept_step : 0u;
                    fetch(t2 + SCAN_TILE <= a.rows);
                }
                const float* tC = sC[use] + scan_again(ST * L.j + half * SCAN_KEEP * N4);
                tB = sB[use] + scan_again(ST * L.j + half * SCAN_KEEP * N4);       // (read again rather than kept in 32 registers)
#pragma unroll
                for (int kk = 1; kk >= 0; --kk) {
                    const int k = 2 * half + kk;
                    float ys[4], gbs[4], gas[4];
#pragma unroll
                    for (int q = 3; q >= 0; --q) {
                        const int i = 4 * kk + q;
                        const float sb = quad_bcast(s4[k], q), xb = quad_bcast(x4[k], q), db = quad_bcast(d4[k], q);
                        const ScanVec<ST> b4 = *(const ScanVec<ST>*)(tB + i * N4), c4 = *(const ScanVec<ST>*)(tC + i * N4);
                        float vb[ST], vc[ST];
#pragma unroll
                        for (int m = 0; m < ST; ++m) {
                            const float ht = fmaf(xb, b4[m], ah[i][m]);
                            ys[q] = m ? fmaf(c4[m], ht, ys[q]) : c4[0] * ht;
                            g[m] = fmaf(c4[m], db, g[m]);
                            vb[m] = g[m] * xb;
                            vc[m] = db * ht;
                            gbs[q] = m ? fmaf(g[m], b4[m], gbs[q]) : g[0] * b4[0];
                            const float f = g[m] * ah[i][m];
                            gas[q] = m ? fmaf(A2[m], f, gas[q]) : A2[0] * f;
                            dA[m] = fmaf(sb, f, dA[m]);
                            g[m] *= ex[i][m];
                        }
                        wave_fold<LPC, ST>(vb, vc);                   // (the lanes that hold one sum write it to one place)
                        const int p = h0 + i;
                        float* to = my_red + (p >= at && p < end ? (p - t0) * W : SCAN_TILE * W);
                        if constexpr (FOLD == 2) *(float2*)to = make_float2(vb[0], vb[1]); else *to = vb[0];
                    }
                    // the lane's row of these four
                    const float y = quad_rows<LPC>(ys, L.q), gb = quad_rows<LPC>(gbs, L.q), ga = quad_rows<LPC>(gas, L.q);
                    const int r = t0 + 4 * k + L.q;
                    const bool mine = L.in && (whole || (r >= at && r < end));
                    const float uk = live && mine ? u[k] : 0.f;
                    const float slope = a.softplus ? seq_sigmoid((float)raw_d[k] + bias) : 1.f;
                    const float dd = live && mine ? fmaf(uk, gb, SEQ_LN2 * ga) * slope : 0.f;
                    dbias += dd;
                    dD = fmaf(d4[k], uk, dD);
                    if (mine && L.j < 4) {
                        ou.row(k) = (T)(live ? fmaf(Dd, d4[k], s4[k] * gb) : 0.f);
                        od.row(k) = (T)dd;
                        if (gated) {
                            const float z = (float)raw_z[k], sg = seq_sigmoid(z);
                            const float dz = (float)raw_y[k] * fmaf(Dd, uk, y) * sg * fmaf(z, 1.f - sg, 1.f);
                            oz.row(k) = (T)(live ? dz : 0.f);
                        }
                    }
                }
            }
            end = at;
            if (at == first && s >= 0) {                          // the clip started with the piece: on to the one in front
                leave(s);
                if (at > c0) {
                    const int was = s;
                    const ScanArgsPtr r = scan_rare();
                    while (s >= 0 && seq_start(r, s) >= at) --s;
                    first = s >= 0 ? __builtin_amdgcn_readfirstlane(seq_start(r, s)) : 0;
                    if (r->dstate) for (int e = s + 1; e < was; ++e) { entry(e); leave(e); }
                    entry(s);
                }
            }
        } while (end > t0);
        stB.store(sB[buf ^ 1], t2, lo, hi);
        stC.store(sC[buf ^ 1], t2, lo, hi);
        ou.template move<-1>(true); od.template move<-1>(true); oz.template move<-1>(true);
        __syncthreads();                                          // red complete; B and C of the next tile in place
        const ScanArgsPtr r = scan_rare();
        float* part = r->part_bc + ((int64_t)blockIdx.x * r->rows + t0) * W;
        const int full = min(SCAN_TILE, c1 - t0) * W;
#pragma unroll
        for (int e = threadIdx.x; e < SCAN_TILE * W; e += 256)
            if (e < full) part[e] = (red[0][e] + red[1][e]) + (red[2][e] + red[3][e]);
        __syncthreads();                                          // red read
    }
    if (scan_rare()->dstate && chunk == 0) {                                 // empty clips in front of the first row
        const SeqClips c = {scan_rare()->clips.start, scan_rare()->clips.n, scan_rare()->clips.rows};
        const int s0 = seq_find(c, 0);
        for (int e = 0; e < s0 && e < c.n; ++e) { entry(e); leave(e); }
    }
    dD += seq_dpp<0xB1>(dD); dD += seq_dpp<0x4E>(dD);
    dbias += seq_dpp<0xB1>(dbias); dbias += seq_dpp<0x4E>(dbias);
    if (L.in) {
        const ScanArgsPtr r = scan_rare();
        float* part = r->part_p + (int64_t)chunk * r->channels * (N + 2);
        scan_store(part + (size_t)L.d * N, L.j, N, dA);
        if (L.j == 0) { part[(size_t)r->channels * N + L.d] = dD; part[(size_t)r->channels * (N + 1) + L.d] = dbias; }
    }
}

// dB and dC: the channel blocks' sums, added in block order (16001 rows, 16 blocks: 33 MB in 7.5 us)
template <typename T>
__global__ __launch_bounds__(256) void k_scan_bc(const float* __restrict__ part, int blocks, int rows, int n4, int N,
                                                 T* __restrict__ dB, int64_t lddb, T* __restrict__ dC, int64_t lddc) {
    const int64_t width = (int64_t)rows * 2 * n4;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < width; e += (int64_t)gridDim.x * 256) {
        const int64_t r = e / (2 * n4);
        const int m = (int)(e - r * 2 * n4), c = m >= n4, i = c ? m - n4 : m;
        if (i >= N) continue;
        float s0 = 0.f, s1 = 0.f;
        int b = 0;
        for (; b + 1 < blocks; b += 2) { s0 += part[b * width + e]; s1 += part[(b + 1) * width + e]; }
        if (b < blocks) s0 += part[b * width + e];
        if (c) dC[r * lddc + i] = (T)(s0 + s1); else dB[r * lddb + i] = (T)(s0 + s1);
    }
}

// One token per clip, bound by the bytes of the states: 4 N in and 4 N out per channel (2048 x 1024 x 16: 285 MB in 50 us,
// 5.7 TB/s; 6 x 256 x 16: 3.6 us).  A lane owns four states of a channel (16 bytes each way) and goes over four clips at a
// time, so that four states are requested before the first is used and the lanes of a quad form the step and the gate of one
// clip each (one clip at a time: 100 us).  VEC: rows of A, B, C and the states are whole and aligned groups of four; otherwise
// they are read entry by entry, the states too (2048 x 1024 x 16 with B and C off a border of four: 147 us instead of 55).
// state_out may be the state itself: a lane reads its entries before it writes them and nobody else needs them.
template <typename T, bool VEC> __device__ __forceinline__ void step_load4(const T* __restrict__ row, int j, int N, float (&v)[4]) {
    if constexpr (VEC) {
        typename SeqVec<T, 4>::type w = {};
        if (4 * j < N) w = *(const typename SeqVec<T, 4>::type*)(row + 4 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)w[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = 4 * j + i < N ? (float)row[4 * j + i] : 0.f;
    }
}

template <typename T, int LPC, bool VEC>
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a) {
    const ScanLane<LPC> L(a);
    const int N = a.n_state;
    float A2[4];
    step_load4<float, VEC>(a.A + (size_t)L.d * N, L.j, N, A2);
#pragma unroll
    for (int i = 0; i < 4; ++i) A2[i] = scan_decay(A2[i]);
    const float bias = a.bias ? a.bias[L.d] : 0.f, Dd = a.D ? a.D[L.d] : 0.f;
    for (int64_t s0 = blockIdx.y * 4; s0 < a.rows; s0 += gridDim.y * 4) {
        const int64_t mine = min(s0 + L.q, (int64_t)a.rows - 1);           // the clip whose step and output this lane forms
        float h[4][4], b[4][4], c[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t s = min(s0 + q, (int64_t)a.rows - 1);
            step_load4<float, VEC>(a.state + (s * a.channels + L.d) * N, L.j, N, h[q]);
            step_load4<T, VEC>((const T*)a.B + s * a.ldb, L.j, N, b[q]);
            step_load4<T, VEC>((const T*)a.C + s * a.ldc, L.j, N, c[q]);
        }
        const float u = (float)((const T*)a.u)[mine * a.ldu + L.d];
        const float raw = (float)((const T*)a.delta)[mine * a.ldd + L.d] + bias;
        const float z = a.z ? (float)((const T*)a.z)[mine * a.ldz + L.d] : 0.f;
        const float st = a.softplus ? scan_softplus(raw) : raw, x = st * u;
        float acc[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float sb = quad_bcast(st, q), xb = quad_bcast(x, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[q][i] = fmaf(seq_exp2(sb * A2[i]), h[q][i], xb * b[q][i]);
                acc[q] = i ? fmaf(c[q][i], h[q][i], acc[q]) : c[q][0] * h[q][0];
            }
        }
        const float y = fmaf(Dd, u, quad_rows<LPC>(acc, L.q)) * (a.z ? z * seq_sigmoid(z) : 1.f);
        if (!L.in) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (s0 + q >= a.rows) break;
            float* dst = a.final_state + ((s0 + q) * a.channels + L.d) * N;
            if constexpr (VEC) { if (4 * L.j < N) *(seq_f4*)(dst + 4 * L.j) = seq_f4{h[q][0], h[q][1], h[q][2], h[q][3]}; }
            else scan_store<4>(dst, L.j, N, h[q]);
        }
        if (L.j < 4 && s0 + L.q < a.rows) ((T*)a.y)[mine * a.ldy + L.d] = (T)y;
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------------
static int scan_lpc(int n_state) { return n_state <= 16 ? 4 : n_state <= 32 ? 8 : 16; }
static int scan_width(int n_state) { return n_state <= 4 ? 4 : n_state <= 8 ? 8 : 4 * scan_lpc(n_state); }  // floats of a state as kept here

// Rows of a chunk.  The chunks run side by side, so a short array is cut as short as the join of the chunks allows, and a long one
// into as many as the chip holds at once: 4 workgroups per CU in the forward passes (3 beyond 32 states), 2 in the gradient --
// one more would wait for a whole round (16 states, bf16; 17920 x 256: 560 workgroups 222 us, 500 of them 185).
//   forward: 1024 workgroups, chunks of 32 rows or more (1000 x 1024: 29 us, with 16 rows 31), of 16 while that makes no more
//     than 512 (256 x 256: 19 us, with 32 rows 22, with 64 29); no chunks up to 64 rows, where two launches fewer count (17 against 18).
//   gradient: 512 workgroups, chunks of 16 rows or more (256 x 256, forward and gradient: 44 us, with 32 rows 48, with 64 65);
//     1024 where that leaves 128 rows to a chunk, whose ends then level out better (12000 x 1024: 398 us against 408; with 64
//     rows left the second round costs more than that, 17920 x 256: 194 against 185).
static void scan_chunks(int64_t rows, int channels, int n_state, int backward, int* chunk_rows, int* chunks) {
    const int per = 256 / scan_lpc(n_state);
    const int64_t groups = (channels + per - 1) / per, by16 = (rows + 15) / 16, by32 = (rows + 31) / 32;
    int64_t want, most;
    if (backward) {
        want = (rows * groups >= 1024 * 128 ? 1024 : 512) / groups;
        most = by16;
    } else {
        want = rows <= 64 ? 1 : (n_state > 32 ? 768 : 1024) / groups;
        most = by16 * groups <= 512 ? by16 : by32 * groups > 512 ? by32 : 512 / groups;
    }
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

// a tile's rows are addressed by 32-bit offsets from its first
static bool scan_ld_ok(int64_t ld, int width) { return ld >= width && ld <= (1 << 24); }

static int64_t scan_carry_floats(int chunks, int channels, int n_state) {
    if (chunks <= 1) return 4;
    const int n4 = scan_width(n_state);
    return (int64_t)chunks * channels * n4 + (((int64_t)chunks * channels + 3) & ~3LL) + ((chunks + 3) & ~3);
}
static void scan_carry(ScanArgs& a, float* ws) {
    const int n4 = scan_width(a.n_state);
    a.carry = ws;
    a.span = ws + (int64_t)a.chunks * a.channels * n4;
    a.flag = (int*)(a.span + (((int64_t)a.chunks * a.channels + 3) & ~3LL));
}

template <int WHAT, typename T, int LPC, int ST> static int scan_launch2(const ScanArgs& a, hipStream_t st) {
    constexpr int per = 256 / LPC;
    const dim3 grid((a.channels + per - 1) / per, a.chunks), block(256);
    if constexpr (WHAT == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_fwd<T, LPC, ST, 0>), grid, block, 0, st, a);
    if constexpr (WHAT == 1) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_fwd<T, LPC, ST, 1>), grid, block, 0, st, a);
    if constexpr (WHAT == 2) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_adj<T, LPC, ST>), grid, block, 0, st, a);
    if constexpr (WHAT == 3) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_bwd<T, LPC, ST>), grid, block, 0, st, a);
    if constexpr (WHAT == 4) {
        const int bytes = 4 * sizeof(T);
        auto quads = [&](const void* p, int64_t ld) { return ((uintptr_t)p | (uintptr_t)(ld * (int64_t)sizeof(T))) % bytes == 0; };
        const bool vec = a.n_state % 4 == 0 && seq_aligned(a.state, 0) && seq_aligned(a.final_state, 0) && seq_aligned(a.A, 0) &&
                         quads(a.B, a.ldb) && quads(a.C, a.ldc);
        // enough workgroups to fill the chip (8 per CU); beyond that a workgroup goes over more clips with the same A
        const int64_t most = (2048 + grid.x - 1) / grid.x, fours = ((int64_t)a.rows + 3) / 4;
        const dim3 g(grid.x, (unsigned)(fours < most ? fours : most));
        if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<T, LPC, true>), g, block, 0, st, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_step<T, LPC, false>), g, block, 0, st, a);
    }
    return evad_last_error();
}
// Few states: one or two per lane instead of four of which most are none (16384 x 1024 bf16, forward / with gradient: 4 states 94 / 318 us,
// 8 states 113 / 381, 16 states 153 / 530, which all took before).
template <int WHAT, typename T> static int scan_launch1(const ScanArgs& a, hipStream_t st) {
    if (WHAT != 4) {                                             // (a single token is bound by the states' bytes)
        if (a.n_state <= 4) return scan_launch2<WHAT, T, 4, WHAT == 4 ? 4 : 1>(a, st);
        if (a.n_state <= 8) return scan_launch2<WHAT, T, 4, WHAT == 4 ? 4 : 2>(a, st);
    }
    switch (scan_lpc(a.n_state)) {
        case 4: return scan_launch2<WHAT, T, 4, 4>(a, st);
        case 8: return scan_launch2<WHAT, T, 8, 4>(a, st);
        default: return scan_launch2<WHAT, T, 16, 4>(a, st);
    }
}
template <int WHAT> static int scan_launch(const ScanArgs& a, int dtype, hipStream_t st) {
    if (dtype == SEQ_F32) return scan_launch1<WHAT, float>(a, st);
    if (dtype == SEQ_BF16) return scan_launch1<WHAT, __bf16>(a, st);
    return scan_launch1<WHAT, _Float16>(a, st);
}
template <int REV> static void scan_join(const ScanArgs& a, hipStream_t st) {
    const int n4 = scan_width(a.n_state);                        // (scan_chunks makes at most 1024)
    const dim3 grid((unsigned)(((int64_t)a.channels * n4 + 15) / 16));
    if (a.chunks > 16 * JOIN_SHARE) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<REV, 64>), grid, dim3(1024), 0, st, a, n4);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_scan_join<REV, 16>), grid, dim3(256), 0, st, a, n4);
}

extern "C" int eventad_selective_scan_workspace(int64_t rows, int channels, int n_state, int backward, int64_t* bytes) {
    if (!bytes || !scan_shape_ok(rows, channels, n_state, 0)) return EVAD_ERR_ARG;
    int cr, chunks;
    scan_chunks(rows, channels, n_state, backward, &cr, &chunks);
    int64_t f = scan_carry_floats(chunks, channels, n_state);
    if (backward) {
        const int per = 256 / scan_lpc(n_state), n4 = scan_width(n_state);
        const int64_t groups = (channels + per - 1) / per, cols = (int64_t)channels * (n_state + 2);
        f += groups * rows * 2 * n4 + (chunks + SEQ_SUM_PARTS) * cols;
    }
    *bytes = f * 4;
    return EVAD_OK;
}

extern "C" int eventad_selective_scan_checkpoint(int64_t rows, int channels, int n_state, int64_t* bytes) {
    if (!bytes || !scan_shape_ok(rows, channels, n_state, 0)) return EVAD_ERR_ARG;
    *bytes = (rows + SCAN_KEEP - 1) / SCAN_KEEP * channels * 4 * scan_width(n_state);
    return EVAD_OK;
}

static bool scan_common(ScanArgs& a, const void* u, int64_t ldu, const void* delta, int64_t ldd, const float* A, const void* B,
                        int64_t ldb, const void* C, int64_t ldc, const float* D, const void* z, int64_t ldz, const float* bias,
                        int64_t rows, int channels, int n_state, int softplus, int dtype) {
    if (!scan_shape_ok(rows, channels, n_state, dtype) || !A || softplus < 0 || softplus > 1) return false;
    if (rows && (!u || !delta || !B || !C || !scan_ld_ok(ldu, channels) || !scan_ld_ok(ldd, channels) || !scan_ld_ok(ldb, n_state) ||
                 !scan_ld_ok(ldc, n_state) || (z && !scan_ld_ok(ldz, channels)))) return false;
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
        clips < 1 || clips > SEQ_MOST_CLIPS || (!clip_start && clips != 1) || (rows && (!y || !scan_ld_ok(ldy, channels))) || ((uintptr_t)checkpoint & 15) ||
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
        clips < 1 || clips > SEQ_MOST_CLIPS || (!clip_start && clips != 1) || !dparams || ((uintptr_t)checkpoint & 15) ||
        (rows && (!dy || !du || !ddelta || !dB || !dC || !checkpoint || !scan_ld_ok(lddy, channels) || !scan_ld_ok(lddu, channels) ||
                  !scan_ld_ok(lddd, channels) || lddb < n_state || lddc < n_state || (z && (!dz || !scan_ld_ok(lddz, channels))))) ||
        eventad_selective_scan_workspace(rows, channels, n_state, 1, &need) != EVAD_OK || !workspace || workspace_bytes < need ||
        ((uintptr_t)workspace & 15)) return EVAD_ERR_ARG;
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.state = state; a.ckpt = (float*)checkpoint; a.dy = dy; a.lddy = lddy; a.dfinal = dfinal; a.du = du; a.lddu = lddu;
    a.ddelta = ddelta; a.lddd = lddd; a.dz = dz; a.lddz = lddz; a.dstate = dstate;
    scan_chunks(rows, channels, n_state, 1, &a.chunk_rows, &a.chunks);
    float* ws = (float*)workspace;
    scan_carry(a, ws);
    const int per = 256 / scan_lpc(n_state), n4 = scan_width(n_state), groups = (channels + per - 1) / per;
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
        const long long blocks = ((long long)rows * 2 * n4 + 255) / 256;
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
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
