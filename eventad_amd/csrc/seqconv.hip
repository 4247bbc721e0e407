// eventad_amd/csrc/seqconv.hip -- short causal convolution over the rows of packed clips, its gradient and its
// single-token form.
//
//   pre_t = bias + sum_{k<K} w[:,k] x_{t-(K-1)+k},   y_t = act(pre_t),   K = 1 .. 8 taps, per channel
//
// x before a clip's first row is the clip's state (its last K-1 inputs of an earlier call) or zero.  Gradient, with
// d_t = dy_t act'(pre_t):  dx_t = sum_k w[:,k] d_{t+(K-1)-k} inside the clip,  dw[:,k] = sum_t d_t x_{t-(K-1)+k},
// dbias = sum_t d_t.
//
// All of it is bound by bytes (2K + 4 operations per element that is read and written once).  A thread owns one 16-byte
// column of a chunk of rows and slides down it with the K-1 inputs before the current row in registers, so a row is read
// once plus (K-1) / chunk for the chunk's start.
#include "seq.h"

#define CONV_MAX_TAPS 8
#define CONV_AHEAD 4                 // rows requested before the first of them is used

struct ConvArgs {
    SeqClips clips;
    const void* x; int64_t ldx;
    const float* w; const float* bias;
    const void* state; void* final_state;            // [clips][K-1][channels]
    void* y; int64_t ldy;
    int rows, channels, cols, chunk_rows, chunks, act;
    // gradient
    const void* dy; int64_t lddy;
    const void* dfinal; void* dstate;
    void* dx; int64_t lddx;
    float* part;                                     // [chunks][channels*K + channels]
};

// A thread's place: its columns, its rows, and the clip of its current row.
template <typename T, int V, int K> struct ConvLane {
    int c, r0, r1, s, next;                          // first channel; rows r0..r1-1; clip of the current row; where it ends
    float w[K][V], b[V];
};

template <typename T, int V, int K>
__device__ __forceinline__ bool conv_lane(const ConvArgs& a, ConvLane<T, V, K>& L) {
    const long long g = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int chunk = (int)(g / a.cols);
    if (chunk >= a.chunks) return false;
    L.c = (int)(g - (long long)chunk * a.cols) * V;
    L.r0 = chunk * a.chunk_rows;
    L.r1 = min(a.rows, L.r0 + a.chunk_rows);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        L.b[i] = a.bias ? a.bias[L.c + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) L.w[k][i] = a.w[(size_t)(L.c + i) * K + k];
    }
    L.s = seq_find(a.clips, L.r0);
    L.next = L.s < a.clips.n ? seq_start(a.clips, L.s + 1) : 0x7fffffff;
    return true;
}

// the K-1 inputs in front of row p of clip s, which starts at `first`
template <typename T, int V, int K>
__device__ __forceinline__ void conv_window(const ConvArgs& a, int c, int s, int first, int p, float (&win)[K][V]) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int q = p - (K - 1) + k;
#pragma unroll
        for (int i = 0; i < V; ++i) win[k][i] = 0.f;
        if (s < 0 || s >= a.clips.n) continue;
        if (q >= first) seq_load<T, V>((const T*)a.x + (int64_t)q * a.ldx + c, win[k]);
        else if (a.state) seq_load<T, V>((const T*)a.state + ((int64_t)s * (K - 1) + (K - 1 + q - first)) * a.channels + c, win[k]);
    }
}

// out rows (K-1) of clip s = in rows of the same clip, or zeros
template <typename T, int V, int K>
__device__ __forceinline__ void conv_copy_state(const ConvArgs& a, int c, int s, const void* in, void* out) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int64_t at = ((int64_t)s * (K - 1) + k) * a.channels + c;
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
        if (in) seq_load<T, V>((const T*)in + at, v);
        seq_store<T, V>((T*)out + at, v);
    }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void k_conv_fwd(ConvArgs a) {
    ConvLane<T, V, K> L;
    if (!conv_lane<T, V, K>(a, L)) return;
    const int n = a.clips.n, c = L.c;
    int s = L.s, next = L.next;
    float win[K][V];
    if (a.final_state)                                          // empty clips at the chunk's first row keep their state
        for (int e = s - 1; e >= 0 && seq_start(a.clips, e) == L.r0; --e) conv_copy_state<T, V, K>(a, c, e, a.state, a.final_state);
    conv_window<T, V, K>(a, c, s, s >= 0 ? seq_start(a.clips, s) : 0, L.r0, win);
    for (int p0 = L.r0; p0 < L.r1; p0 += CONV_AHEAD) {
        float x[CONV_AHEAD][V];
#pragma unroll
        for (int j = 0; j < CONV_AHEAD; ++j) seq_load<T, V>((const T*)a.x + (int64_t)min(p0 + j, L.r1 - 1) * a.ldx + c, x[j]);
#pragma unroll
        for (int j = 0; j < CONV_AHEAD; ++j) {
            const int p = p0 + j;
            if (p >= L.r1) break;
            if (p >= next && s < n) {                           // the clip ended in front of this row
                if (a.final_state && s >= 0 && p > L.r0) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) seq_store<T, V>((T*)a.final_state + ((int64_t)s * (K - 1) + k) * a.channels + c, win[k]);
                }
                ++s;
                while (s < n && seq_start(a.clips, s + 1) <= p) {
                    if (a.final_state) conv_copy_state<T, V, K>(a, c, s, a.state, a.final_state);
                    ++s;
                }
                next = s < n ? seq_start(a.clips, s + 1) : 0x7fffffff;
                conv_window<T, V, K>(a, c, s, p, p, win);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) win[K - 1][i] = x[j][i];
            float y[V];
            const bool live = s >= 0 && s < n;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float acc = L.b[i];
#pragma unroll
                for (int k = 0; k < K; ++k) acc = fmaf(L.w[k][i], win[k][i], acc);
                y[i] = live ? (a.act ? acc * seq_sigmoid(acc) : acc) : 0.f;
            }
            seq_store<T, V>((T*)a.y + (int64_t)p * a.ldy + c, y);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
        }
    }
    if (a.final_state && L.r1 > L.r0 && next <= L.r1 && s < n) { // a clip ends with the chunk
        if (s >= 0) {
#pragma unroll
            for (int k = 0; k < K - 1; ++k) seq_store<T, V>((T*)a.final_state + ((int64_t)s * (K - 1) + k) * a.channels + c, win[k]);
        }
        if (L.r1 == a.rows)                                     // empty clips behind the last row
            for (++s; s < n; ++s) conv_copy_state<T, V, K>(a, c, s, a.state, a.final_state);
    }
}

// One pass down the chunk: d_p is formed once per row (the chunk's K-1 rows behind its end included), and a row's dx is
// complete K-1 rows later.  acc[k] = what row p-(K-1)+k has collected.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void k_conv_bwd(ConvArgs a) {
    ConvLane<T, V, K> L;
    if (!conv_lane<T, V, K>(a, L)) return;
    const int n = a.clips.n, c = L.c;
    int s = L.s, next = L.next, first = s >= 0 ? seq_start(a.clips, s) : 0;
    float win[K][V], acc[K][V], dw[K][V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) { dw[k][i] = 0.f; acc[k][i] = 0.f; }
    }
    // the gradient of position q of the current clip: a row of the chunk, or a row of the state of a clip that starts in it
    auto emit = [&](int q, const float (&v)[V]) {
        if (q >= first) { if (q >= L.r0 && q < L.r1) seq_store<T, V>((T*)a.dx + (int64_t)q * a.lddx + c, v); }
        else if (a.dstate && first >= L.r0 && first < L.r1)
            seq_store<T, V>((T*)a.dstate + ((int64_t)s * (K - 1) + (K - 1 + q - first)) * a.channels + c, v);
    };
    // the clip ended in front of row p: what its last K-1 positions have collected, with the gradient of its final state
    auto flush = [&](int p) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            if (a.dfinal) {
                float f[V];
                seq_load<T, V>((const T*)a.dfinal + ((int64_t)s * (K - 1) + k) * a.channels + c, f);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[k][i] += f[i];
            }
            emit(p - (K - 1) + k, acc[k]);
        }
    };
    if (a.dstate)
        for (int e = s - 1; e >= 0 && seq_start(a.clips, e) == L.r0; --e) conv_copy_state<T, V, K>(a, c, e, a.dfinal, a.dstate);
    conv_window<T, V, K>(a, c, s, first, L.r0, win);
    const int end = min(a.rows, L.r1 + K - 1);
    bool done = false;
    for (int p0 = L.r0; p0 < end && !done; p0 += CONV_AHEAD) {
        float x[CONV_AHEAD][V], g[CONV_AHEAD][V];
#pragma unroll
        for (int j = 0; j < CONV_AHEAD; ++j) {
            const int64_t p = min(p0 + j, end - 1);
            seq_load<T, V>((const T*)a.x + p * a.ldx + c, x[j]);
            seq_load<T, V>((const T*)a.dy + p * a.lddy + c, g[j]);
        }
#pragma unroll
        for (int j = 0; j < CONV_AHEAD; ++j) {
            const int p = p0 + j;
            if (p >= end || done) break;
            if (p >= next && s < n) {
                if (s >= 0 && p > L.r0) flush(p);
                if (p >= L.r1) { done = true; break; }          // the rows behind the chunk belong to another clip
                ++s;
                while (s < n && seq_start(a.clips, s + 1) <= p) {
                    if (a.dstate) conv_copy_state<T, V, K>(a, c, s, a.dfinal, a.dstate);
                    ++s;
                }
                next = s < n ? seq_start(a.clips, s + 1) : 0x7fffffff;
                first = p;
                conv_window<T, V, K>(a, c, s, p, p, win);
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[k][i] = 0.f;
            }
            if (s < 0 || s >= n) {                              // a row of no clip
                if (p >= L.r1) { done = true; break; }
                float zero[V];
#pragma unroll
                for (int i = 0; i < V; ++i) zero[i] = 0.f;
                seq_store<T, V>((T*)a.dx + (int64_t)p * a.lddx + c, zero);
                continue;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                win[K - 1][i] = x[j][i];
                float d = g[j][i];
                if (a.act) {
                    float pre = L.b[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) pre = fmaf(L.w[k][i], win[k][i], pre);
                    const float sg = seq_sigmoid(pre);
                    d *= sg * fmaf(pre, 1.f - sg, 1.f);
                }
                if (p < L.r1) {
                    db[i] += d;
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k][i] = fmaf(d, win[k][i], dw[k][i]);
                }
#pragma unroll
                for (int k = 0; k < K; ++k) acc[k][i] = fmaf(L.w[k][i], d, acc[k][i]);
            }
            emit(p - (K - 1), acc[0]);
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) { win[k][i] = win[k + 1][i]; acc[k][i] = acc[k + 1][i]; }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[K - 1][i] = 0.f;
        }
    }
    if (!done && end > L.r0 && s >= 0 && s < n && next <= end) flush(end);
    if (a.dstate && L.r1 == a.rows && L.r1 > L.r0) {            // empty clips behind the last row
        for (int e = n - 1; e >= 0 && seq_start(a.clips, e) == a.rows; --e) conv_copy_state<T, V, K>(a, c, e, a.dfinal, a.dstate);
    }
    float* part = a.part + (int64_t)(L.r0 / a.chunk_rows) * ((int64_t)a.channels * (K + 1));
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) part[(size_t)(c + i) * K + k] = dw[k][i];
        part[(size_t)a.channels * K + c + i] = db[i];
    }
}

// one token per clip: reads the K-1 rows of state, writes them shifted (state_out may be the state itself: a thread reads
// all rows of its column before it writes one)
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void k_conv_step(ConvArgs a) {
    const long long g = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int s = (int)(g / a.cols);
    if (s >= a.rows) return;
    const int c = (int)(g - (long long)s * a.cols) * V;
    float win[K][V], y[V];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) seq_load<T, V>((const T*)a.state + ((int64_t)s * (K - 1) + k) * a.channels + c, win[k]);
    seq_load<T, V>((const T*)a.x + (int64_t)s * a.ldx + c, win[K - 1]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float acc = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) acc = fmaf(a.w[(size_t)(c + i) * K + k], win[k][i], acc);
        y[i] = a.act ? acc * seq_sigmoid(acc) : acc;
    }
    seq_store<T, V>((T*)a.y + (int64_t)s * a.ldy + c, y);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) seq_store<T, V>((T*)a.final_state + ((int64_t)s * (K - 1) + k) * a.channels + c, win[k + 1]);
}

// ---- column sums (seq.h) -------------------------------------------------------------------------------------------------
// 64 columns x 4 row lanes per workgroup; gridDim.y workgroups share the rows of a column block.
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
template <int WHAT, typename T, int V, int K> static void conv_launch3(const ConvArgs& a, hipStream_t st) {
    const long long items = (long long)a.cols * (WHAT == 2 ? a.rows : a.chunks);
    const dim3 grid(evad_blocks(items, 256)), block(256);
    if constexpr (WHAT == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_fwd<T, V, K>), grid, block, 0, st, a);
    else if constexpr (WHAT == 1) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_bwd<T, V, K>), grid, block, 0, st, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_conv_step<T, V, K>), grid, block, 0, st, a);
}
template <int WHAT, typename T, int V> static void conv_launch2(const ConvArgs& a, int K, hipStream_t st) {
    switch (K) {
        case 1: conv_launch3<WHAT, T, V, 1>(a, st); break;
        case 2: conv_launch3<WHAT, T, V, 2>(a, st); break;
        case 3: conv_launch3<WHAT, T, V, 3>(a, st); break;
        case 4: conv_launch3<WHAT, T, V, 4>(a, st); break;
        case 5: conv_launch3<WHAT, T, V, 5>(a, st); break;
        case 6: conv_launch3<WHAT, T, V, 6>(a, st); break;
        case 7: conv_launch3<WHAT, T, V, 7>(a, st); break;
        default: conv_launch3<WHAT, T, V, 8>(a, st); break;
    }
}
template <int WHAT, typename T> static void conv_launch1(ConvArgs& a, int K, bool vec, hipStream_t st) {
    constexpr int N = SeqVec<T>::n;
    if (vec && a.channels % N == 0) { a.cols = a.channels / N; conv_launch2<WHAT, T, N>(a, K, st); }
    else { a.cols = a.channels; conv_launch2<WHAT, T, 1>(a, K, st); }
}
template <int WHAT> static int conv_launch(ConvArgs& a, int K, int dtype, bool vec, hipStream_t st) {
    if (dtype == SEQ_F32) conv_launch1<WHAT, float>(a, K, vec, st);
    else if (dtype == SEQ_BF16) conv_launch1<WHAT, __bf16>(a, K, vec, st);
    else conv_launch1<WHAT, _Float16>(a, K, vec, st);
    return evad_last_error();
}

static int conv_chunk_rows(int64_t rows, int channels, int backward) {
    // long chunks waste fewer reads at their starts, short ones give the chip more threads
    return backward ? 64 : 32;
}
static bool conv_shape_ok(int64_t rows, int channels, int taps, int dtype) {
    return rows >= 0 && rows <= 0x7ffffff0 && channels >= 1 && channels <= (1 << 20) && taps >= 1 && taps <= CONV_MAX_TAPS && dtype >= 0 && dtype <= 2;
}
static int conv_elem(int dtype) { return dtype == SEQ_F32 ? 4 : 2; }

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
    if (!conv_shape_ok(rows, channels, taps, dtype) || !w || clips < 1 || (!clip_start && clips != 1) || act < 0 || act > 1 ||
        (rows && (!x || !y || ldx < channels || ldy < channels))) return EVAD_ERR_ARG;
    ConvArgs a = {};
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.y = y; a.ldy = ldy; a.rows = (int)rows; a.channels = channels; a.act = act;
    if (taps > 1) { a.state = state; a.final_state = final_state; }
    a.chunk_rows = conv_chunk_rows(rows, channels, 0);
    a.chunks = rows ? (int)((rows + a.chunk_rows - 1) / a.chunk_rows) : 1;
    if (!rows && !a.final_state) return EVAD_OK;
    const int e = conv_elem(dtype);
    const bool vec = seq_aligned(x, ldx * e) && seq_aligned(y, ldy * e) && seq_aligned(state, 0) && seq_aligned(final_state, 0);
    return conv_launch<0>(a, taps, dtype, vec, (hipStream_t)stream);
}

extern "C" int eventad_causal_conv_bwd(const void* x, int64_t ldx, const float* w, const float* bias, const int32_t* clip_start,
                                       int clips, const void* state, const void* dy, int64_t lddy, const void* dfinal, void* dx,
                                       int64_t lddx, void* dstate, float* dparams, void* workspace, int64_t workspace_bytes,
                                       int64_t rows, int channels, int taps, int act, int dtype, void* stream) {
    int64_t need = 0;
    if (eventad_causal_conv_workspace(rows, channels, taps, &need) != EVAD_OK) return EVAD_ERR_ARG;
    if (!conv_shape_ok(rows, channels, taps, dtype) || !w || clips < 1 || (!clip_start && clips != 1) || act < 0 || act > 1 ||
        !dparams || !workspace || workspace_bytes < need || (rows && (!x || !dy || !dx || ldx < channels || lddy < channels || lddx < channels)))
        return EVAD_ERR_ARG;
    ConvArgs a = {};
    a.clips = SeqClips{clip_start, clips, (int)rows};
    a.x = x; a.ldx = ldx; a.w = w; a.bias = bias; a.dy = dy; a.lddy = lddy; a.dx = dx; a.lddx = lddx;
    a.rows = (int)rows; a.channels = channels; a.act = act;
    if (taps > 1) { a.state = state; a.dfinal = dfinal; a.dstate = dstate; }
    a.chunk_rows = conv_chunk_rows(rows, channels, 1);
    a.chunks = rows ? (int)((rows + a.chunk_rows - 1) / a.chunk_rows) : 1;
    a.part = (float*)workspace;
    const int e = conv_elem(dtype);
    const bool vec = seq_aligned(x, ldx * e) && seq_aligned(dy, lddy * e) && seq_aligned(dx, lddx * e) && seq_aligned(state, 0) &&
                     seq_aligned(dfinal, 0) && seq_aligned(dstate, 0);
    const int rc = conv_launch<1>(a, taps, dtype, vec, (hipStream_t)stream);
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
    a.rows = clips; a.channels = channels; a.act = act;
    const int e = conv_elem(dtype);
    const bool vec = seq_aligned(x, ldx * e) && seq_aligned(y, ldy * e) && seq_aligned(state, 0) && seq_aligned(state_out, 0);
    return conv_launch<2>(a, taps, dtype, vec, (hipStream_t)stream);
}
