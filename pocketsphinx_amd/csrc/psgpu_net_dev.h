// psgpu_net_dev.h -- what the operators of an acoustic network (psgpu_proj.hip, psgpu_gnorm.hip, psgpu_netscr.hip) share: element
// types, wide accesses at any alignment, the utterance a packed row belongs to.
#pragma once
#include "psgpu_internal.h"

typedef _Float16 psg_half;
struct psg_bf16 { uint16_t bits; };

__device__ __forceinline__ float net_f32(float v) { return v; }
__device__ __forceinline__ float net_f32(psg_half v) { return (float)v; }
__device__ __forceinline__ float net_f32(psg_bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

// rounding to nearest, ties to even, infinities and NaN kept (NaN quiet)
template <typename T> __device__ __forceinline__ T net_cast(float v);
template <> __device__ __forceinline__ float net_cast<float>(float v) { return v; }
template <> __device__ __forceinline__ psg_half net_cast<psg_half>(float v) { return (psg_half)v; }
template <> __device__ __forceinline__ psg_bf16 net_cast<psg_bf16>(float v)
{
    const uint32_t u = __float_as_uint(v);
    psg_bf16 r;
    r.bits = (u & 0x7fffffffu) > 0x7f800000u ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
    return r;
}

// N consecutive elements that need no alignment beyond their own: the hardware serves wide loads and stores at any element address
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) net_pack { T v[N]; };

// The utterance of a packed row: the u with off[u] <= row < off[u + 1], or -1 (in front of the first, behind the last).  Empty
// utterances are stepped over.  Offsets that do not ascend give some u or -1, never an access outside off[0 .. n_utt].
__device__ __forceinline__ int net_utt_of_row(const int32_t *off, int n_utt, int row)
{
    int lo = 0, hi = n_utt;                         // first u in [0, n_utt] with off[u + 1] > row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (off[mid + 1] > row) hi = mid; else lo = mid + 1;
    }
    return lo < n_utt && off[lo] <= row ? lo : -1;
}

static inline size_t net_dtype_size(int32_t dtype) { return dtype == PSGPU_DT_F32 ? 4 : 2; }
static inline bool net_dtype_ok(int32_t dtype) { return dtype == PSGPU_DT_F32 || dtype == PSGPU_DT_F16 || dtype == PSGPU_DT_BF16; }
// bytes that rows of `width` elements at `stride` cover
static inline size_t net_span(int64_t rows, int64_t stride, int64_t width, size_t es) { return rows ? (size_t)((rows - 1) * stride + width) * es : 0; }
static inline bool net_disjoint(const void *a, size_t na, const void *b, size_t nb)
{
    return (uintptr_t)a + na <= (uintptr_t)b || (uintptr_t)b + nb <= (uintptr_t)a;
}
