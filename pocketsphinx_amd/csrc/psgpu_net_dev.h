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
template <> __device__ __forceinline__ psg_bf16 net_cast<psg_bf16>(float v) { return __builtin_bit_cast(psg_bf16, (__bf16)v); }

// N consecutive elements that need no alignment beyond their own: the hardware serves wide loads and stores at any element address
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) net_pack { T v[N]; };

// element e of 16 bytes in four registers (e a constant after unrolling)
typedef uint32_t net_u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ float net_elem(const net_u32x4 &v, int e)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(v[e]);
    else {
        const uint32_t w = v[e >> 1];
        if constexpr (__is_same(T, psg_bf16)) return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
        else return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w >> 16 : w));
    }
}

// The utterance of each of 64 packed rows, row0 + lane: the u with off[u] <= row < off[u + 1], or -1 (in front of the first, behind
// the last).  Empty utterances are stepped over.  Offsets that do not ascend give some u or -1, never an access outside
// off[0 .. n_utt].  All lanes of the wavefront call it.  64 offsets a step for the first row (two dependent loads for 4096 utterances;
// a binary search would wait for 12), then the 64 offsets behind it for the rest.
__device__ __forceinline__ int net_utt_of_rows(const int32_t *off, int n_utt, int row0)
{
    const int lane = (int)(threadIdx.x & 63), row = row0 + lane;
    int lo = 0, hi = n_utt;                         // the first u in [lo, hi] with off[u + 1] > row0 (hi: none)
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) >> 6, at = lo + lane * step;
        const uint64_t above = __ballot(at >= hi || off[min(at, n_utt - 1) + 1] > row0);
        const int f = above ? __builtin_ctzll(above) : 64;
        hi = min(hi, lo + f * step);
        lo = f ? min(hi, lo + (f - 1) * step + 1) : lo;
    }
    // off[lo + 1 + lane], the last of them standing for all behind it
    int v = lo + lane < n_utt ? off[lo + lane + 1] : 0x7fffffff;
    const uint64_t above = __ballot(lo + lane >= hi || v > row0);
    const int skip = above ? __builtin_ctzll(above) : 64;
    lo += skip;
    if (skip) v = lo + lane < n_utt ? off[lo + lane + 1] : 0x7fffffff;
    int pos = 0;                                    // how many of the 64 offsets are not above this lane's row
#pragma unroll
    for (int s = 32; s; s >>= 1)
        if (__shfl(v, pos + s - 1) <= row) pos += s;
    int u = lo + pos;
    if (pos == 63 && u < n_utt && off[u + 1] <= row) {      // more than 64 utterances end within these rows
        int a = u + 1, b = n_utt;
        while (a < b) {
            const int mid = (a + b) >> 1;
            if (off[mid + 1] > row) b = mid; else a = mid + 1;
        }
        u = a;
    }
    return u >= 0 && u < n_utt && off[u] <= row && off[u + 1] > row ? u : -1;
}

// A barrier in front of which this wavefront waits for all of its loads (and stores) but the N issued last, and for its LDS
// instructions.  Loads that go to LDS without a register need their own wait: a plain barrier's covers LDS instructions, not always these.
template <int N>
__device__ __forceinline__ void net_wait_barrier()
{
    static_assert(N >= 0 && N < 64, "a counter of six bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "i"(N) : "memory");
}

// Loads to LDS without a register: `bytes` (16 or 4) a lane from base + off (off the lane's, base all lanes'), to lds + lane * bytes.
// In assembly, so that the compiler does not know them: it would wait for all of them in front of every read of LDS, also of parts
// that they do not write (128 k rows of 1024 to 1024 outputs: 725 against 786 TFLOP/s).  net_wait_barrier() is the wait they need; they have
// no result in registers, and waits that the compiler places for its own loads only become longer by them.  (The idle cycles: a vector
// instruction may just have written `base`.)
template <int bytes>
__device__ __forceinline__ void net_load_lds(const void *base, uint32_t off, uint32_t lds)
{
    static_assert(bytes == 16 || bytes == 4, "a size that the instruction has");
    if constexpr (bytes == 16) asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dword %0, %1" :: "v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
// where an object in LDS begins
template <typename T> __device__ __forceinline__ uint32_t net_lds_at(T *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)p; }

// ---- matrix instructions ------------------------------------------------------------------------------------------------------------
// Products of 16 x 16 from 16 bytes a lane: lane l of the first operand holds row l & 15, of the second column l & 15, elements
// (l >> 4) * E .. + E - 1 of the reduced axis (E = 16 bytes of T; one instruction of 4 E elements for halves, four of 4 for floats, which
// take element j of every lane's chunk -- the same order on both sides, so the sum is the same set of products).  Lane l holds of the
// result column l & 15, rows (l >> 4) * 4 .. + 3.
typedef float net_f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 net_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 net_bf16x8 __attribute__((ext_vector_type(8)));
template <typename T> struct net_frag;
template <> struct net_frag<float> { typedef net_f32x4 type; };
template <> struct net_frag<psg_half> { typedef net_f16x8 type; };
template <> struct net_frag<psg_bf16> { typedef net_bf16x8 type; };

__device__ __forceinline__ net_f32x4 net_mfma(net_f32x4 a, net_f32x4 b, net_f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ net_f32x4 net_mfma(net_f16x8 a, net_f16x8 b, net_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ net_f32x4 net_mfma(net_bf16x8 a, net_bf16x8 b, net_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// E elements of a row from k on, zeros from d_in on; any alignment
template <typename T>
__device__ __forceinline__ typename net_frag<T>::type net_load_chunk(const T *row, int k, int d_in)
{
    constexpr int E = 16 / sizeof(T);
    net_pack<T, E> v;
    if (k + E <= d_in) v = *(const net_pack<T, E> *)(row + k);
    else {
        v = {};
        for (int e = 0; e < E; ++e)
            if (k + e < d_in) v.v[e] = row[k + e];
    }
    return __builtin_bit_cast(typename net_frag<T>::type, v);
}

static inline size_t net_dtype_size(int32_t dtype) { return dtype == PSGPU_DT_F32 ? 4 : 2; }
static inline bool net_dtype_ok(int32_t dtype) { return dtype == PSGPU_DT_F32 || dtype == PSGPU_DT_F16 || dtype == PSGPU_DT_BF16; }
// PSGPU_OK iff a gfx950 device is current, which one; asks the runtime about a device's kind once
int net_check_device(int *device);

// bytes that rows of `width` elements at `stride` cover
static inline size_t net_span(int64_t rows, int64_t stride, int64_t width, size_t es) { return rows ? (size_t)((rows - 1) * stride + width) * es : 0; }
static inline bool net_disjoint(const void *a, size_t na, const void *b, size_t nb)
{
    return (uintptr_t)a + na <= (uintptr_t)b || (uintptr_t)b + nb <= (uintptr_t)a;
}
