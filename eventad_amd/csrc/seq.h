// eventad_amd/csrc/seq.h -- shared by the sequence operators (seqconv.hip, seqscan.hip, rmsnorm.hip): element types, clip
// offsets, column sums.
//
// Rows of a [rows, channels] array are packed: clip s owns rows clip_start[s] .. clip_start[s+1]-1 (i32[clips+1], not
// decreasing, inside 0..rows); rows in front of the first and behind the last clip belong to none.  Without an array all
// rows are one clip.  The offsets are read on the device only, so no call waits for the GPU and every launch can be
// captured; whatever they hold, they are only compared with row numbers that the launch made itself: offsets outside 0..rows
// count as the nearer end, and ones that decrease give wrong numbers (and leave states of clips that no row leads to as they
// were), never an access outside an array.
#pragma once
#include "common.h"

#define SEQ_F32 0
#define SEQ_BF16 1
#define SEQ_F16 2

typedef float seq_f4 __attribute__((ext_vector_type(4)));

// V elements of a type as one access
template <typename T, int V> struct SeqVec { typedef T type __attribute__((ext_vector_type(V))); };

// V elements at p as floats / back, rounded to nearest even
template <typename T, int V> __device__ __forceinline__ void seq_load(const T* __restrict__ p, float (&out)[V]) {
    if constexpr (V == 1) out[0] = (float)*p;
    else {
        const typename SeqVec<T, V>::type v = *(const typename SeqVec<T, V>::type*)p;
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)v[i];
    }
}
template <typename T, int V> __device__ __forceinline__ void seq_store(T* __restrict__ p, const float (&in)[V]) {
    if constexpr (V == 1) *p = (T)in[0];
    else {
        typename SeqVec<T, V>::type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)in[i];
        *(typename SeqVec<T, V>::type*)p = v;
    }
}

// the same in two steps: request now, convert when it is there
template <typename T, int V> struct SeqRaw { typedef typename SeqVec<T, V>::type type; };
template <typename T> struct SeqRaw<T, 1> { typedef T type; };
template <typename T, int V> __device__ __forceinline__ typename SeqRaw<T, V>::type seq_raw(const T* __restrict__ p) {
    return *(const typename SeqRaw<T, V>::type*)p;
}
template <typename T, int V> __device__ __forceinline__ void seq_unpack(const typename SeqRaw<T, V>::type& v, float (&out)[V]) {
    if constexpr (V == 1) out[0] = (float)v;
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)v[i];
    }
}

#define SEQ_LOG2E 1.4426950408889634f
#define SEQ_LN2 0.6931471805599453f

__device__ __forceinline__ float seq_exp2(float x) { return __builtin_amdgcn_exp2f(x); }          // v_exp_f32, 1 ulp
__device__ __forceinline__ float seq_rcp(float x) { return __builtin_amdgcn_rcpf(x); }            // v_rcp_f32, 1 ulp
__device__ __forceinline__ float seq_sigmoid(float x) { return seq_rcp(1.f + seq_exp2(-SEQ_LOG2E * x)); }

template <int CTRL> __device__ __forceinline__ float seq_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ unsigned seq_dpp_bits(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// x = the sum over both halves of the wave: of x in lanes 0..31, of y in lanes 32..63
__device__ __forceinline__ void seq_swap32(float& x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(y), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
}
// x = the sum over each pair of rows of 16 lanes: of x in the even row, of y in the odd one
__device__ __forceinline__ void seq_swap16(float& x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(y), false, false);
    x = __int_as_float(r[0]) + __int_as_float(r[1]);
}
// sum over 16, 32 or 64 lanes, in all of them: xor 1, xor 2 (quad_perm), the mirrored half row and row, then the rows
template <int LANES> __device__ __forceinline__ float seq_lane_sum(float v) {
    v += seq_dpp<0xB1>(v);
    v += seq_dpp<0x4E>(v);
    v += seq_dpp<0x141>(v);
    v += seq_dpp<0x140>(v);
    if constexpr (LANES >= 32) seq_swap16(v, v);
    if constexpr (LANES >= 64) seq_swap32(v, v);
    return v;
}

struct SeqClips { const int* start; int n; int rows; };        // start == nullptr: one clip of all rows

__device__ __forceinline__ int seq_start(const SeqClips& c, int s) { return c.start ? min(max(c.start[s], 0), c.rows) : (s ? c.rows : 0); }

// the last s in 0..n with start[s] <= row, or -1: the clip of the row (n: behind the last clip), empty clips skipped
__device__ __forceinline__ int seq_find(const SeqClips& c, int row) {
    int lo = -1, hi = c.n + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (seq_start(c, mid) <= row) lo = mid; else hi = mid;
    }
    return lo;
}

#define SEQ_MOST_CLIPS ((1 << 30) - 1)         // (seq_find adds two of their numbers)
#define SEQ_MOST_THREADS 0xffffff00LL          // of one launch (threads are numbered in 32 bits)

static inline bool seq_aligned(const void* p, int64_t row_bytes) { return (((uintptr_t)p | (uintptr_t)row_bytes) & 15) == 0; }

// ---- column sums: out[c] = sum over rows of in[rows][cols], in a fixed order.  `scratch` holds SEQ_SUM_PARTS x cols floats.
#define SEQ_SUM_PARTS 64
int seq_colsum(const float* in, int64_t rows, int64_t cols, float* out, float* scratch, hipStream_t st);
