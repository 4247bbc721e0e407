// eventad_amd/csrc/seqconv.hip -- short causal convolution over the rows of packed clips, its gradient and its
// single-token form.
//
//   pre_t = bias + sum_{k<K} w[:,k] x_{t-(K-1)+k},   y_t = act(pre_t),   K = 1 .. 8 taps, per channel
//
// x before a clip's first row is the clip's state (its last K-1 inputs of an earlier call) or zero.  Gradient, with
// d_t = dy_t act'(pre_t):  dx_t = sum_k w[:,k] d_{t+(K-1)-k} inside the clip,  dw[:,k] = sum_t d_t x_{t-(K-1)+k},
// dbias = sum_t d_t.
//
// Up to four taps it is bound by bytes (2K + 4 operations per element that is read and written once): K = 4, 400,000 x 256 f32 819 MB in
// 153 us (5.4 TB/s), its gradient 1229 MB in 280 us (4.4 TB/s; a copy of 4 GiB runs at 4.75), 17,920 x 1024 f16 73 MB in 19 us.  A thread owns four adjacent
// channels (one, where rows are not aligned to four) of a chunk of rows and slides down it with the K-1 inputs before the current
// row in registers, so a row is read once plus (K-1) / chunk for the chunk's start.  Rows go by in groups of four, requested
// a group ahead; a group that meets a clip's or the chunk's border goes row by row instead, reading again what it needs.
// Four channels and not the eight that 16 bytes of a 16-bit type hold: weights and windows of eight are 128 registers, and the
// waves that fit beside them do not cover the memory's latency.
// WAVE: with 64 columns or more a wave has one chunk, and the walk over the clips is scalar (17,920 x 1024 bf16 forward 22 us, without
// it 24; 400,000 x 256 with gradient 250 and 264); narrower arrays put several chunks into a wave.
#include "seq.h"

#define CONV_MAX_TAPS 8
#define CONV_GROUP 4
#define CONV_PAIR 2                  // the gradient's group: two arrays in, and collectors beside the window

struct ConvArgs {
    SeqClips clips;
    const void* x; int64_t ldx;
    const float* w; const float* bias;
    const void* state; void* final_state;            // [clips][taps-1][channels]
    void* y; int64_t ldy;
    int rows, channels, cols, chunk_rows, chunks, act, taps;
    // gradient
    const void* dy; int64_t lddy;
    const void* dfinal; void* dstate;
    void* dx; int64_t lddx;
    float* part;                                     // [chunks][channels*taps + channels]
};

// The kernels are built for K = 2, 3, 4 and 8 taps; K = 8 serves every other number: its first K - taps window entries are zero
// and stay out of the sums.  (17,920 x 1024 bf16, forward and with the gradient: four taps 18 and 60 us, by the kernels for eight 31 and
// 118; five 26 and 119, six 32 and 134, eight 41 and 158.  The gradient's 244 to 295 registers leave one or two waves per SIMD, and it
// reads seven rows behind every chunk.)
template <int K> __device__ __forceinline__ int conv_skip(const ConvArgs& a) { return K == 8 ? K - a.taps : 0; }

template <bool WAVE> __device__ __forceinline__ int conv_same(int v) { return WAVE ? __builtin_amdgcn_readfirstlane(v) : v; }

// A thread's place: its columns, its rows, its parameters.
template <typename T, int V, int K, bool WAVE> struct ConvLane {
    int c, r0, r1, chunk;                            // first channel; rows r0..r1-1
    float w[K][V], b[V];
    __device__ __forceinline__ bool place(const ConvArgs& a) {
        if constexpr (WAVE) {
            const unsigned wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), per = (a.cols + 63) / 64;
            chunk = wave / per;
            const int col = (int)(wave - chunk * per) * 64 + (threadIdx.x & 63);
            c = col * V;
            if (chunk >= a.chunks || col >= a.cols) return false;
        } else {
            const unsigned g = blockIdx.x * 256 + threadIdx.x;
            chunk = g / (unsigned)a.cols;
            c = (int)(g - (unsigned)chunk * a.cols) * V;
            if (chunk >= a.chunks) return false;
        }
        r0 = chunk * a.chunk_rows;
        r1 = r0 + min(a.chunk_rows, a.rows - r0);                // (the last chunk's end may not fit 32 bits)
        const int skip = conv_skip<K>(a);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            b[i] = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k) w[k][i] = k >= skip ? a.w[(size_t)(c + i) * a.taps + k - skip] : 0.f;
        }
        return true;
    }
    __device__ __forceinline__ void pre(const ConvArgs& a, const float (*win)[V], float (&out)[V]) const {   // win[0..K-1]
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = b[i];
        const int skip = conv_skip<K>(a);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k >= skip)
#pragma unroll
                for (int i = 0; i < V; ++i) out[i] = fmaf(w[k][i], win[k][i], out[i]);
    }
};

// the K-1 inputs in front of row p of clip s, which starts at `first`
template <typename T, int V, int K>
__device__ __forceinline__ void conv_window(const ConvArgs& a, int c, int s, int first, int p, float (*win)[V]) {
    const int skip = conv_skip<K>(a);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int q = p - (K - 1) + k;
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = 0.f;
        if (s < 0 || s >= a.clips.n || k < skip) continue;
        float v[V];
        if (q >= first) seq_load<T, V>((const T*)a.x + (int64_t)q * a.ldx + c, v);
        else if (a.state && q < first) seq_load<T, V>((const T*)a.state + ((int64_t)s * (a.taps - 1) + (K - 1 - skip + q - first)) * a.channels + c, v);
        else continue;
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = v[i];
    }
}

// rows of a state of clip s: `rows` of K - 1 window entries, or the same clip's rows of `in`, or zeros
template <typename T, int V, int K>
__device__ __forceinline__ void conv_store_state(const ConvArgs& a, int c, int s, const float (*win)[V], void* out) {
    const int skip = conv_skip<K>(a);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        if (k < skip) continue;
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = win[k][i];
        seq_store<T, V>((T*)out + ((int64_t)s * (a.taps - 1) + k - skip) * a.channels + c, v);
    }
}
template <typename T, int V>
__device__ __forceinline__ void conv_copy_state(const ConvArgs& a, int c, int s, const void* in, void* out) {
    for (int k = 0; k < a.taps - 1; ++k) {
        const int64_t at = ((int64_t)s * (a.taps - 1) + k) * a.channels + c;
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
        if (in) seq_load<T, V>((const T*)in + at, v);
        seq_store<T, V>((T*)out + at, v);
    }
}

template <typename T, int V, int K, bool WAVE>
__global__ __launch_bounds__(256) void k_conv_fwd(ConvArgs a) {
    ConvLane<T, V, K, WAVE> L;
    if (!L.place(a)) return;
    const int n = a.clips.n, c = L.c;
    int s = conv_same<WAVE>(seq_find(a.clips, L.r0));
    int next = s < n ? conv_same<WAVE>(seq_start(a.clips, s + 1)) : 0x7fffffff;       // where the clip ends
    float win[K - 1 + CONV_GROUP][V];
    const T* x = (const T*)a.x + (int64_t)L.r0 * a.ldx + c;
    typename SeqRaw<T, V>::type raw[CONV_GROUP];
    auto request = [&](int p0) {
#pragma unroll
        for (int j = 0; j < CONV_GROUP; ++j) raw[j] = seq_raw<T, V>(x + (int64_t)(min(p0 + j, L.r1 - 1) - L.r0) * a.ldx);
    };
    if (L.r1 > L.r0) request(L.r0);
    if (a.final_state)                                          // empty clips at the chunk's first row keep their state
        for (int e = s - 1; e >= 0 && seq_start(a.clips, e) == L.r0; --e) conv_copy_state<T, V>(a, c, e, a.state, a.final_state);
    conv_window<T, V, K>(a, c, s, s >= 0 ? seq_start(a.clips, s) : 0, L.r0, win);
    auto row = [&](int p, const float (*w)[V], bool live) {
        float y[V];
        L.pre(a, w, y);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (a.act) y[i] *= seq_sigmoid(y[i]);
            if (!live) y[i] = 0.f;
        }
        seq_store<T, V>((T*)a.y + (int64_t)p * a.ldy + c, y);
    };
    for (int p0 = L.r0; p0 < L.r1; p0 += CONV_GROUP) {
        float now[CONV_GROUP][V];
#pragma unroll
        for (int j = 0; j < CONV_GROUP; ++j) seq_unpack<T, V>(raw[j], now[j]);
        request(p0 + CONV_GROUP);
        if (s >= 0 && s < n && next >= p0 + CONV_GROUP && L.r1 >= p0 + CONV_GROUP) {
#pragma unroll
            for (int j = 0; j < CONV_GROUP; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i) win[K - 1 + j][i] = now[j][i];
#pragma unroll
            for (int j = 0; j < CONV_GROUP; ++j) row(p0 + j, win + j, true);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) win[k][i] = win[k + CONV_GROUP][i];
        } else {
#pragma unroll 1
            for (int p = p0; p < min(p0 + CONV_GROUP, L.r1); ++p) {
                if (p >= next && s < n) {                       // the clip ended in front of this row
                    if (a.final_state && s >= 0) conv_store_state<T, V, K>(a, c, s, win, a.final_state);
                    ++s;
                    while (s < n && seq_start(a.clips, s + 1) <= p) {
                        if (a.final_state) conv_copy_state<T, V>(a, c, s, a.state, a.final_state);
                        ++s;
                    }
                    next = s < n ? conv_same<WAVE>(seq_start(a.clips, s + 1)) : 0x7fffffff;
                    conv_window<T, V, K>(a, c, s, p, p, win);
                }
                float v[V];
                seq_load<T, V>((const T*)a.x + (int64_t)p * a.ldx + c, v);
#pragma unroll
                for (int i = 0; i < V; ++i) win[K - 1][i] = v[i];
                row(p, win, s >= 0 && s < n);
#pragma unroll
                for (int k = 0; k < K - 1; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
            }
        }
    }
    if (a.final_state && L.r1 > L.r0 && next <= L.r1 && s < n) { // a clip ends with the chunk
        if (s >= 0) conv_store_state<T, V, K>(a, c, s, win, a.final_state);
        if (L.r1 == a.rows)                                     // empty clips behind the last row
            for (++s; s < n; ++s) conv_copy_state<T, V>(a, c, s, a.state, a.final_state);
    }
}

// One pass down the chunk and the K-1 rows behind it: d_p is formed once per row, and a row's dx is complete K-1 rows later.
// acc[k] = what position p-(K-1)+k of the clip has collected when row p is reached.  (Three workgroups per CU: with four taps and fewer than
// 64 columns that spills 3 to 13 registers; 100,000 x 64 bf16 with the forward 44 us, where its bytes take 14.)
template <typename T, int V, int K, bool WAVE>
__global__ __launch_bounds__(256, K == 8 ? 1 : 3) void k_conv_bwd(ConvArgs a) {
    ConvLane<T, V, K, WAVE> L;
    if (!L.place(a)) return;
    const int n = a.clips.n, c = L.c, skip = conv_skip<K>(a);
    int s = conv_same<WAVE>(seq_find(a.clips, L.r0));
    int next = s < n ? conv_same<WAVE>(seq_start(a.clips, s + 1)) : 0x7fffffff;
    int first = s >= 0 ? conv_same<WAVE>(seq_start(a.clips, s)) : 0;
    float win[K - 1 + CONV_PAIR][V], acc[K - 1 + CONV_PAIR][V], dw[K][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
#pragma unroll
        for (int k = 0; k < K - 1 + CONV_PAIR; ++k) acc[k][i] = 0.f;
    }
    const int end = min(a.rows, L.r1 + K - 1);                  // (a position is given out K-1 rows behind it, fewer taps or not)
    const T* x = (const T*)a.x + (int64_t)L.r0 * a.ldx + c;
    const T* dy = (const T*)a.dy + (int64_t)L.r0 * a.lddy + c;
    typename SeqRaw<T, V>::type rawx[CONV_PAIR], rawg[CONV_PAIR];
    auto request = [&](int p0) {
#pragma unroll
        for (int j = 0; j < CONV_PAIR; ++j) {
            const int64_t r = min(p0 + j, end - 1) - L.r0;
            rawx[j] = seq_raw<T, V>(x + r * a.ldx);
            rawg[j] = seq_raw<T, V>(dy + r * a.lddy);
        }
    };
    if (end > L.r0) request(L.r0);
    if (a.dstate)
        for (int e = s - 1; e >= 0 && seq_start(a.clips, e) == L.r0; --e) conv_copy_state<T, V>(a, c, e, a.dfinal, a.dstate);
    conv_window<T, V, K>(a, c, s, first, L.r0, win);
    // row p with its window w and collectors to[0..K-1]
    auto row = [&](const float (*w)[V], float (*to)[V], const float (&g)[V], bool count) {
        float d[V], pre[V];
        if (a.act) {
            L.pre(a, w, pre);
#pragma unroll
            for (int i = 0; i < V; ++i) { const float sg = seq_sigmoid(pre[i]); d[i] = g[i] * (sg * fmaf(pre[i], 1.f - sg, 1.f)); }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = g[i];
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k >= skip)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (count) dw[k][i] = fmaf(d[i], w[k][i], dw[k][i]);
                    to[k][i] = fmaf(L.w[k][i], d[i], to[k][i]);
                }
        if (count)
#pragma unroll
            for (int i = 0; i < V; ++i) db[i] += d[i];
    };
    auto put = [&](int q, const float (*v)[V]) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = v[0][i];
        seq_store<T, V>((T*)a.dx + (int64_t)q * a.lddx + c, o);
    };
    // the gradient of position q of the current clip: a row of the chunk, or a row of the state of a clip that starts in it
    auto emit = [&](int q, const float (*v)[V]) {
        if (q >= first) { if (q >= L.r0 && q < L.r1) put(q, v); }
        else if (a.dstate && first >= L.r0 && first < L.r1 && q >= first - (a.taps - 1)) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = v[0][i];
            seq_store<T, V>((T*)a.dstate + ((int64_t)s * (a.taps - 1) + (a.taps - 1 + q - first)) * a.channels + c, o);
        }
    };
    // the clip ended in front of row p: what its last K-1 positions have collected, with the gradient of its final state
    auto flush = [&](int p) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            if (a.dfinal && k >= skip) {
                float f[V];
                seq_load<T, V>((const T*)a.dfinal + ((int64_t)s * (a.taps - 1) + k - skip) * a.channels + c, f);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[k][i] += f[i];
            }
            emit(p - (K - 1) + k, acc + k);
        }
    };
    bool done = false;
    for (int p0 = L.r0; p0 < end && !done; p0 += CONV_PAIR) {
        float g[CONV_PAIR][V], now[CONV_PAIR][V];
#pragma unroll
        for (int j = 0; j < CONV_PAIR; ++j) { seq_unpack<T, V>(rawx[j], now[j]); seq_unpack<T, V>(rawg[j], g[j]); }
        request(p0 + CONV_PAIR);
        if (s >= 0 && s < n && next >= p0 + CONV_PAIR && L.r1 >= p0 + CONV_PAIR && p0 - (K - 1) >= max(first, L.r0)) {
#pragma unroll
            for (int j = 0; j < CONV_PAIR; ++j) {
#pragma unroll
                for (int i = 0; i < V; ++i) win[K - 1 + j][i] = now[j][i];
                row(win + j, acc + j, g[j], true);
                put(p0 + j - (K - 1), acc + j);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k < K - 1; ++k) { win[k][i] = win[k + CONV_PAIR][i]; acc[k][i] = acc[k + CONV_PAIR][i]; }
#pragma unroll
                for (int k = K - 1; k < K - 1 + CONV_PAIR; ++k) acc[k][i] = 0.f;
            }
        } else {
#pragma unroll 1
            for (int p = p0; p < min(p0 + CONV_PAIR, end); ++p) {
                if (p >= next && s < n) {
                    if (s >= 0 && p > L.r0) flush(p);
                    if (p >= L.r1) { done = true; break; }      // the rows behind the chunk belong to another clip
                    ++s;
                    while (s < n && seq_start(a.clips, s + 1) <= p) {
                        if (a.dstate) conv_copy_state<T, V>(a, c, s, a.dfinal, a.dstate);
                        ++s;
                    }
                    next = s < n ? conv_same<WAVE>(seq_start(a.clips, s + 1)) : 0x7fffffff;
                    first = p;
                    conv_window<T, V, K>(a, c, s, p, p, win);
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i) acc[k][i] = 0.f;
                }
                if (s < 0 || s >= n) {                          // a row of no clip
                    if (p >= L.r1) { done = true; break; }
                    float zero[1][V];
#pragma unroll
                    for (int i = 0; i < V; ++i) zero[0][i] = 0.f;
                    put(p, zero);
                    continue;
                }
                float v[V], gr[V];
                seq_load<T, V>((const T*)a.x + (int64_t)p * a.ldx + c, v);
                seq_load<T, V>((const T*)a.dy + (int64_t)p * a.lddy + c, gr);
#pragma unroll
                for (int i = 0; i < V; ++i) win[K - 1][i] = v[i];
                row(win, acc, gr, p < L.r1);
                emit(p - (K - 1), acc);
#pragma unroll
                for (int i = 0; i < V; ++i) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) { win[k][i] = win[k + 1][i]; acc[k][i] = acc[k + 1][i]; }
                    acc[K - 1][i] = 0.f;
                }
            }
        }
    }
    if (!done && end > L.r0 && s >= 0 && s < n && next <= end) flush(end);
    if (a.dstate && L.r1 == a.rows && L.r1 > L.r0)              // empty clips behind the last row
        for (int e = n - 1; e >= 0 && seq_start(a.clips, e) == a.rows; --e) conv_copy_state<T, V>(a, c, e, a.dfinal, a.dstate);
    float* part = a.part + (int64_t)L.chunk * ((int64_t)a.channels * (a.taps + 1));
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) if (k >= skip) part[(size_t)(c + i) * a.taps + k - skip] = dw[k][i];
        part[(size_t)a.channels * a.taps + c + i] = db[i];
    }
}

// one token per clip (6 x 256: 2.1 us, all of it latency): reads the K-1 rows of state, writes them shifted (state_out may be the state itself: a thread reads
// all rows of its columns before it writes one)
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs a) {
    const unsigned g = blockIdx.x * 256 + threadIdx.x;
    const int s = g / (unsigned)a.cols, skip = conv_skip<K>(a);
    if (s >= a.rows) return;
    ConvLane<T, V, K, false> L;
    const int c = (int)(g - (unsigned)s * a.cols) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        L.b[i] = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) L.w[k][i] = k >= skip ? a.w[(size_t)(c + i) * a.taps + k - skip] : 0.f;
    }
    float win[K][V], y[V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = 0.f;
        if (k >= skip) seq_load<T, V>(k < K - 1 ? (const T*)a.state + ((int64_t)s * (a.taps - 1) + k - skip) * a.channels + c : (const T*)a.x + (int64_t)s * a.ldx + c, win[k]);
    }
    L.pre(a, win, y);
#pragma unroll
    for (int i = 0; i < V; ++i) if (a.act) y[i] *= seq_sigmoid(y[i]);
    seq_store<T, V>((T*)a.y + (int64_t)s * a.ldy + c, y);
    conv_store_state<T, V, K>(a, c, s, win + 1, a.final_state);
}

// ---- column sums (seq.h) -------------------------------------------------------------------------------------------------
// 64 columns x 4 row lanes per workgroup; gridDim.y workgroups share the rows of a column block (8334 rows of 1280 columns, 43 MB:
// 11 us, and 5 for the 64 parts).
__global__ __launch_bounds__(256) void k_seq_colsum(const float* __restrict__ in, int64_t rows, int64_t cols, float* __restrict__ out) {
    __shared__ float s[4][64];
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
    if (c < cols) {
        int64_t r = r0 + q;
        for (; r + 12 < r1; r += 16) {
            const float v0 = in[r * cols + c], v1 = in[(r + 4) * cols + c], v2 = in[(r + 8) * cols + c], v3 = in[(r + 12) * cols + c];
            a0 += v0; a1 += v1; a2 += v2; a3 += v3;
        }
        for (; r < r1; r += 4) a0 += in[r * cols + c];
    }
    s[q][lane] = (a0 + a1) + (a2 + a3);
    __syncthreads();
    if (q == 0 && c < cols) out[blockIdx.y * cols + c] = (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]);
}

int seq_colsum(const float* in, int64_t rows, int64_t cols, float* out, float* scratch, hipStream_t st) {
    // one launch while a workgroup has at most 64 rows to add; beyond that the rows are shared out so that ~2048 workgroups run
    // (gradients with such sums behind them, bf16: norm of 4096 x 256 18 us, in one launch 36; convolution of 100,000 x 64 45, 161)
    const int64_t blocks = (cols + 63) / 64;
    int64_t parts = rows <= 64 ? 1 : (rows + 31) / 32;
    const int64_t fill = (2048 + blocks - 1) / blocks;
    if (parts > fill) parts = fill;
    if (parts > SEQ_SUM_PARTS) parts = SEQ_SUM_PARTS;
    if (parts < 1) parts = 1;
    float* first = parts == 1 ? out : scratch;
    hipLaunchKernelGGL(k_seq_colsum, dim3((unsigned)blocks, (unsigned)parts), dim3(256), 0, st, in, rows, cols, first);
    if (parts > 1) hipLaunchKernelGGL(k_seq_colsum, dim3((unsigned)blocks, 1), dim3(256), 0, st, scratch, parts, cols, out);
    return evad_last_error();
}

// ---- entry points --------------------------------------------------------------------------------------------------------
template <int WHAT, typename T, int V, int K> static int conv_launch3(const ConvArgs& a, hipStream_t st) {
    const bool wave = WHAT != 2 && a.cols >= 64;
    const long long items = wave ? (long long)((a.cols + 63) / 64) * a.chunks * 64 : (long long)a.cols * (WHAT == 2 ? a.rows : a.chunks);
    if (items > SEQ_MOST_THREADS) return EVENTAD_ERR_TOO_LARGE;
    const dim3 grid(evad_blocks(items, 256)), block(256);
    if constexpr (WHAT == 2) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_step<T, V, K>), grid, block, 0, st, a);
    if constexpr (WHAT == 0) {
        if (wave) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_fwd<T, V, K, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_fwd<T, V, K, false>), grid, block, 0, st, a);
    }
    if constexpr (WHAT == 1) {
        if (wave) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_bwd<T, V, K, true>), grid, block, 0, st, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_bwd<T, V, K, false>), grid, block, 0, st, a);
    }
    return evad_last_error();
}
template <int WHAT, typename T, int V> static int conv_launch2(const ConvArgs& a, hipStream_t st) {
    switch (a.taps) {
        case 2: return conv_launch3<WHAT, T, V, 2>(a, st);
        case 3: return conv_launch3<WHAT, T, V, 3>(a, st);
        case 4: return conv_launch3<WHAT, T, V, 4>(a, st);
        default: return conv_launch3<WHAT, T, V, 8>(a, st);
    }
}
// Four channels to a thread where rows are whole aligned groups of four (17,920 x 1024 bf16 forward 21 us, with gradient 62), otherwise
// one (x 1023: 27 and 74; groups with a last one of three, element by element, 35 and 125).
template <int WHAT, typename T> static int conv_launch1(ConvArgs& a, bool vec, hipStream_t st) {
    const bool four = vec && a.channels % 4 == 0;
    a.cols = four ? a.channels / 4 : a.channels;
    return four ? conv_launch2<WHAT, T, 4>(a, st) : conv_launch2<WHAT, T, 1>(a, st);
}
template <int WHAT> static int conv_launch(ConvArgs& a, int dtype, bool vec, hipStream_t st) {
    if (dtype == SEQ_F32) return conv_launch1<WHAT, float>(a, vec, st);
    if (dtype == SEQ_BF16) return conv_launch1<WHAT, __bf16>(a, vec, st);
    return conv_launch1<WHAT, _Float16>(a, vec, st);
}
// rows of four elements start on a border of four elements
static bool conv_vec(const void* p, int64_t ld, int dtype) {
    const int e = dtype == SEQ_F32 ? 4 : 2;
    return (((uintptr_t)p | (uintptr_t)(ld * e)) & (4 * e - 1)) == 0;
}

// Rows of a chunk.  A long chunk wastes less on the K - 1 rows that it reads beside its own, and in the gradient on its part of dw;
// a short one gives the chip more threads.  Forward: 2^18 threads, 4 .. 32 rows (6000 x 2048 bf16: 17.4 us, with 2^19 20.0).
// Gradient, measured with the forward: 2^17 threads, 4 .. 48 rows (6000 x 2048: 50 us, with 2^16 55, with 2^19 88; 400,000 x 256 f32
// alone 280 us, with 64 rows 301, which leave the third round of workgroups almost empty), of at least 16 rows while 2^16 threads
// are left (100,000 x 64: 45 us, with 12 rows 49; 2240 x 256: 25 us with 4 rows, with 16 28).
static int conv_chunk_rows(int64_t rows, int channels, int backward) {
    const int64_t all = rows * ((channels + 3) / 4);
    int64_t r = backward ? all >> 17 : all >> 18;
    if (backward && r < 16) r = all >> 16 < 16 ? all >> 16 : 16;
    const int most = backward ? 48 : 32;
    return r < 4 ? 4 : r > most ? most : (int)r / 4 * 4;
}
static bool conv_shape_ok(int64_t rows, int channels, int taps, int dtype) {
    return rows >= 0 && rows <= 0x7ffffff0 && channels >= 1 && channels <= (1 << 20) && taps >= 1 && taps <= CONV_MAX_TAPS && dtype >= 0 && dtype <= 2;
}

extern "C" int eventad_causal_conv_workspace(int64_t rows, int channels, int taps, int64_t* bytes) {
    if (!bytes || !conv_shape_ok(rows, channels, taps, 0)) return EVAD_ERR_ARG;
    const int cr = conv_chunk_rows(rows, channels, 1);
    const int64_t chunks = rows ? (rows + cr - 1) / cr : 1;
    *bytes = (chunks + SEQ_SUM_PARTS) * (int64_t)channels * (taps + 1) * 4;
    return EVAD_OK;
}

extern "C" int eventad_causal_conv_fwd(const void* x, int64_t ldx, const float* w, const float* bias, const int32_t* clip_start,
                                       int clips, const void* state, void* final_state, void* y, int64_t ldy, int64_t rows,
                                       int channels, int taps, int act, int dtype, void* stream) {
    if (!conv_shape_ok(rows, channels, taps, dtype) || !w || clips < 1 || clips > SEQ_MOST_CLIPS || (!clip_start && clips != 1) || act < 0 || act > 1 ||
        (rows && (!x || !y || ldx < channels || ldy < channels))) return EVAD_ERR_ARG;
    ConvArgs a = {};
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.y = y; a.ldy = ldy; a.rows = (int)rows; a.channels = channels; a.act = act; a.taps = taps;
    if (taps > 1) { a.state = state; a.final_state = final_state; }
    a.chunk_rows = conv_chunk_rows(rows, channels, 0);
    a.chunks = rows ? (int)((rows + a.chunk_rows - 1) / a.chunk_rows) : 1;
    if (!rows && !a.final_state) return EVAD_OK;
    const bool vec = conv_vec(x, ldx, dtype) && conv_vec(y, ldy, dtype) && conv_vec(state, 0, dtype) && conv_vec(final_state, 0, dtype);
    return conv_launch<0>(a, dtype, vec, (hipStream_t)stream);
}

extern "C" int eventad_causal_conv_bwd(const void* x, int64_t ldx, const float* w, const float* bias, const int32_t* clip_start,
                                       int clips, const void* state, const void* dy, int64_t lddy, const void* dfinal, void* dx,
                                       int64_t lddx, void* dstate, float* dparams, void* workspace, int64_t workspace_bytes,
                                       int64_t rows, int channels, int taps, int act, int dtype, void* stream) {
    int64_t need = 0;
    if (eventad_causal_conv_workspace(rows, channels, taps, &need) != EVAD_OK) return EVAD_ERR_ARG;
    if (!conv_shape_ok(rows, channels, taps, dtype) || !w || clips < 1 || clips > SEQ_MOST_CLIPS || (!clip_start && clips != 1) || act < 0 || act > 1 ||
        !dparams || !workspace || workspace_bytes < need || (rows && (!x || !dy || !dx || ldx < channels || lddy < channels || lddx < channels)))
        return EVAD_ERR_ARG;
    ConvArgs a = {};
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.dy = dy; a.lddy = lddy; a.dx = dx; a.lddx = lddx;
    a.rows = (int)rows; a.channels = channels; a.act = act; a.taps = taps;
    if (taps > 1) { a.state = state; a.dfinal = dfinal; a.dstate = dstate; }
    a.chunk_rows = conv_chunk_rows(rows, channels, 1);
    a.chunks = rows ? (int)((rows + a.chunk_rows - 1) / a.chunk_rows) : 1;
    a.part = (float*)workspace;
    const bool vec = conv_vec(x, ldx, dtype) && conv_vec(dy, lddy, dtype) && conv_vec(dx, lddx, dtype) && conv_vec(state, 0, dtype) &&
                     conv_vec(dfinal, 0, dtype) && conv_vec(dstate, 0, dtype);
    const int rc = conv_launch<1>(a, dtype, vec, (hipStream_t)stream);
    if (rc) return rc;
    const int64_t cols = (int64_t)channels * (taps + 1);
    return seq_colsum(a.part, a.chunks, cols, dparams, a.part + a.chunks * cols, (hipStream_t)stream);
}

extern "C" int eventad_causal_conv_step(const void* x, int64_t ldx, const float* w, const float* bias, const void* state,
                                        void* state_out, void* y, int64_t ldy, int clips, int channels, int taps, int act,
                                        int dtype, void* stream) {
    if (!conv_shape_ok(clips, channels, taps, dtype) || !w || act < 0 || act > 1 ||
        (clips && (!x || !y || ldx < channels || ldy < channels || (taps > 1 && (!state || !state_out))))) return EVAD_ERR_ARG;
    if (!clips) return EVAD_OK;
    ConvArgs a = {};
    a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.state = state; a.final_state = state_out; a.y = y; a.ldy = ldy;
    a.rows = clips; a.channels = channels; a.act = act; a.taps = taps;
    const bool vec = conv_vec(x, ldx, dtype) && conv_vec(y, ldy, dtype) && conv_vec(state, 0, dtype) && conv_vec(state_out, 0, dtype);
    return conv_launch<2>(a, dtype, vec, (hipStream_t)stream);
}
