// psgpu_gnorm.hip -- group norm with an activation over packed utterances, channels last.
//
//   m, v     = mean and biased variance of x[t, c] over the utterance's frames t and the group's channels c
//   y[t, c]  = act((x[t, c] - m) / sqrt(v + eps) * weight[c] + bias[c])
//
// What cmn() with -varnorm is for cepstra (reference src/feat/cmn.c:166-233), per group of channels and with a learned scale.
// Sums run in 64 bits: sum x^2 - n m^2 is off by a few (m^2 / v) 2^-53 of it, which 32 bits do not show up to a mean of 10^4 spreads.
//
// Every kernel works on a slice of whole neighbouring groups of some rows: a work-item has one chunk of 16 bytes of the slice's
// channels and every nrl-th row, so a wavefront reads rows in one piece at any alignment.  Memory bounds them all.
#include "psgpu_net_dev.h"
#include <cmath>

struct gn_args {
    const void *x;
    int64_t xs;
    const int32_t *off;
    int32_t n_utt, total, n_chan, per, n_groups, gs;    // gs: groups a slice
    const float *weight, *bias;
    float eps;
    void *y;
    int64_t ys;
    double2 *part;                                      // [tiles + n_utt][n_groups] sums of a tile's rows of an utterance
    int32_t tile_rows;
};

struct gn_stat { float mhi, mlo, rstd; };               // the mean in two parts

// 1 - (the normal distribution's integral up to t >= 0) = exp(-t^2 / 2) s P(s), s = 1 / (1 + a t), the form of Hastings (Approximations for
// Digital Computers, 1955); P an own fit, whose relative error swings between equal extremes over 0 <= t <= 14, beyond which the result is 0
// in 32 bits: 1.6e-8 with a = 0.21 and degree 8; for results of 16 bits 8.7e-7 with a = 0.36 and degree 6, a 500th of float16's
// half-step.  erff() took three times the instructions and bound the kernel.
template <bool SHORT>
__device__ __forceinline__ float gn_upper_tail(float t)
{
    if constexpr (SHORT) {
        const float s = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, t, 1.0f));
        float p = 0.04705620851f;
        p = __builtin_fmaf(p, s, -0.1797644336f);
        p = __builtin_fmaf(p, s, 0.1809536743f);
        p = __builtin_fmaf(p, s, 0.02654954911f);
        p = __builtin_fmaf(p, s, 0.1397191875f);
        p = __builtin_fmaf(p, s, 0.1417724663f);
        p = __builtin_fmaf(p, s, 0.1437130447f);
        return __builtin_amdgcn_exp2f(t * t * -0.72134752044448170f) * (s * p);
    }
    const float s = __builtin_amdgcn_rcpf(__builtin_fmaf(0.21f, t, 1.0f));
    float p = -0.07165627723f;
    p = __builtin_fmaf(p, s, 0.2835884168f);
    p = __builtin_fmaf(p, s, -0.3302530846f);
    p = __builtin_fmaf(p, s, 0.3494006789f);
    p = __builtin_fmaf(p, s, -0.09392498913f);
    p = __builtin_fmaf(p, s, 0.1248726401f);
    p = __builtin_fmaf(p, s, 0.0691921909f);
    p = __builtin_fmaf(p, s, 0.08506885524f);
    p = __builtin_fmaf(p, s, 0.08371157581f);
    return __builtin_amdgcn_exp2f(t * t * -0.72134752044448170f) * (s * p);
}

// v / (1 + e^-v) through e^-|v| = 2^t, t = -|v| log2 e: for results of 32 bits with what rounding cost t (|v| 2^-24 of the result without it,
// 20 half-steps at v = -20; nothing that 16 bits show), and with e^v in the numerator below 0, where e^-v could leave float's range.
// From |v| = 200 on e^-|v| is 0 in any case; an infinity would make a NaN of the difference.
template <bool SHORT>
__device__ __forceinline__ float gn_silu(float v)
{
    if constexpr (SHORT) return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
    const float a = fminf(fabsf(v), 200.0f), t = a * -1.4426950408889634f;
    const float r = __builtin_fmaf(a, -1.925963033e-8f, __builtin_fmaf(a, -1.4426950408889634f, -t));
    const float e0 = __builtin_amdgcn_exp2f(t), e = __builtin_fmaf(e0, r * 0.69314718055994531f, e0);
    return (v < 0.0f ? v * e : v) * __builtin_amdgcn_rcpf(1.0f + e);
}

template <int ACT, bool SHORT>
__device__ __forceinline__ float gn_act(float v)
{
    switch (ACT) {
    case PSGPU_ACT_RELU: return v < 0.0f ? 0.0f : v;                              // (a NaN stays one)
    case PSGPU_ACT_SILU: return gn_silu<SHORT>(v);
    case PSGPU_ACT_GELU: {
        const float q = gn_upper_tail<SHORT>(fabsf(v));
        return v * (v < 0.0f ? q : 1.0f - q);
    }
    default: return v;
    }
}

// E channels of a row from c on, zeros from c1 on, as they lie in four registers
// (FULL: no chunk reaches beyond c1)
template <bool FULL, typename T>
__device__ __forceinline__ net_u32x4 gn_load(const T *row, int c, int c1)
{
    if constexpr (FULL) return __builtin_bit_cast(net_u32x4, *(const net_pack<T, 16 / sizeof(T)> *)(row + c));
    else return __builtin_bit_cast(net_u32x4, net_load_chunk(row, c, c1));
}

// K pairs of sums of a chunk: one for all its channels (they are of one group), or one a channel
template <typename T, int K>
__device__ __forceinline__ void gn_add(double (&sum)[K], double (&sq)[K], const net_u32x4 &v)
{
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); ++e) {
        const double d = (double)net_elem<T>(v, e);
        sum[K == 1 ? 0 : e] += d;
        sq[K == 1 ? 0 : e] = __builtin_fma(d, d, sq[K == 1 ? 0 : e]);
    }
}

// A slice's place: channels c0 .. c1 - 1 = groups g0 .. g0 + ng - 1; this work-item's row and chunk in it.  A slice of one group may
// be wider than the workgroup's chunks; its work-items then take it in strides of NT chunks.
template <typename T, int NT>
struct gn_place {
    int g0, ng, c0, c1, cw, nrl, rl, ck;
    __device__ __forceinline__ gn_place(const gn_args &a, int slice)
    {
        constexpr int E = 16 / sizeof(T);
        g0 = slice * a.gs;
        ng = min(a.gs, a.n_groups - g0);
        c0 = g0 * a.per;
        c1 = c0 + ng * a.per;
        cw = min((c1 - c0 + E - 1) / E, NT);
        nrl = NT / cw;
        rl = (int)threadIdx.x / cw;
        ck = (int)threadIdx.x - rl * cw;
        if (rl >= nrl) rl = 0x7fffffff;                  // no row is its own
    }
};

// sums over the lanes of `lanes` (a power of two) neighbours, to all of them
__device__ __forceinline__ void gn_sum_lanes(double &sum, double &sq, int lanes)
{
    for (int o = lanes >> 1; o; o >>= 1) { sum += __shfl_xor(sum, o); sq += __shfl_xor(sq, o); }
}

// the slice's groups: group tid / lanes (may be beyond ng) is summed by `lanes` neighbours
template <int NT>
__device__ __forceinline__ int gn_lanes(int ng)
{
    int l = 64;
    while (l > 1 && l * ng > NT) l >>= 1;
    return l;
}

// the work-items' sums joined by groups, in one order always.  s_red [NT * K]; every work-item calls it; lane 0 of a group's lanes has
// the result where its group is one (returns it, else -1)
template <typename T, int NT, int K>
__device__ __forceinline__ int gn_join(const gn_args &a, const gn_place<T, NT> &p, double (&sum)[K], double (&sq)[K], double2 *s_red, double2 &out)
{
    constexpr int E = 16 / sizeof(T);
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k) s_red[tid * K + k] = make_double2(sum[k], sq[k]);
    __syncthreads();
    const int lanes = gn_lanes<NT>(p.ng), g = tid / lanes, lane = tid & (lanes - 1);
    double s = 0.0, q = 0.0;
    if (g < p.ng) {
        const int n = K > 1 ? a.per : p.ng == 1 ? p.cw : a.per / E;             // a group's pairs in a row of work-items
        const int at = K > 1 ? g * a.per : g * n;
        if (p.nrl >= n) {
            for (int r = lane; r < p.nrl; r += lanes)
                for (int i = 0; i < n; ++i) {
                    const double2 v = s_red[r * p.cw * K + at + i];
                    s += v.x; q += v.y;
                }
        } else {
            for (int r = 0; r < p.nrl; ++r)
                for (int i = lane; i < n; i += lanes) {
                    const double2 v = s_red[r * p.cw * K + at + i];
                    s += v.x; q += v.y;
                }
        }
    }
    gn_sum_lanes(s, q, lanes);
    out = make_double2(s, q);
    return g < p.ng && lane == 0 ? g : -1;
}

__device__ __forceinline__ gn_stat gn_finish(double2 s, double n, float eps)
{
    const double mean = s.x / n;
    double var = s.y / n - mean * mean;
    if (var < 0.0) var = 0.0;                           // (a NaN stays one)
    gn_stat r;
    r.rstd = (float)(1.0 / sqrt(var + (double)eps));
    r.mhi = (float)mean;
    r.mlo = (float)(mean - (double)r.mhi);
    return r;
}

// what a chunk's channels are multiplied by and what is added
template <int E> struct gn_affine { float mhi[E], mlo[E], rw[E], b[E]; };

template <typename T, int NT, int K>
__device__ __forceinline__ void gn_affine_of(const gn_args &a, const gn_place<T, NT> &p, int c, const gn_stat *s_stat, gn_affine<16 / sizeof(T)> &f)
{
    constexpr int E = 16 / sizeof(T);
    const int g1 = min((c - p.c0) / a.per, p.ng - 1);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int ce = min(c + e, p.c1 - 1);
        const gn_stat s = s_stat[K == 1 || p.ng == 1 ? g1 : (ce - p.c0) / a.per];
        f.mhi[e] = s.mhi;
        f.mlo[e] = s.mlo;
        f.rw[e] = a.weight ? s.rstd * a.weight[ce] : s.rstd;
        f.b[e] = a.bias ? a.bias[ce] : 0.0f;
    }
}

template <typename T, int ACT, bool FULL>
__device__ __forceinline__ void gn_store(const net_u32x4 &v, const gn_affine<16 / sizeof(T)> &f, T *row, int c, int c1)
{
    constexpr int E = 16 / sizeof(T);
    net_pack<T, E> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = net_cast<T>(gn_act<ACT, sizeof(T) == 2>(__builtin_fmaf((net_elem<T>(v, e) - f.mhi[e]) - f.mlo[e], f.rw[e], f.b[e])));
    if (FULL || c + E <= c1) *(net_pack<T, E> *)(row + c) = o;
    else
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c + e < c1) row[c + e] = o.v[e];
}

// ---- an utterance's slice a workgroup ----------------------------------------------------------------------------------------------
// The first NCH chunks of a work-item stay in registers from the sums to the result: what fits there is read once.  512 utterances of
// 10 frames of 1024: 11 us, one trip to memory, the sums' join and the stores.
template <typename T, int NT, int NCH, int K, bool FULL, int ACT>
__global__ __launch_bounds__(NT, 4)
void gnorm_held_kernel(gn_args a)
{
    constexpr int E = 16 / sizeof(T);
    __shared__ double2 s_red[NT * K];
    __shared__ gn_stat s_stat[NT];
    const int u = blockIdx.y;
    const int t0 = max(a.off[u], 0), t1 = min(a.off[u + 1], a.total);
    if (t1 <= t0) return;
    const gn_place<T, NT> p(a, blockIdx.x);
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const int len = t1 - t0, c = p.c0 + p.ck * E;
    // rows rl + i nrl, i < mine; at 32-bit offsets from the utterance's first (the host sees to that)
    const int mine = p.rl < len ? (len - 1 - p.rl) / p.nrl + 1 : 0;
    const char *xu = (const char *)(x + t0 * a.xs);
    const uint32_t x0 = mine ? (uint32_t)(p.rl * (int)a.xs) * sizeof(T) : 0, x_step = (uint32_t)(p.nrl * (int)a.xs) * sizeof(T);
    net_u32x4 held[NCH];
    double sum[K] = {}, sq[K] = {};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        held[i] = {};
        if (i < mine) held[i] = gn_load<FULL>((const T *)(xu + (x0 + i * x_step)), c, p.c1);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        gn_add<T, K>(sum, sq, held[i]);
        __builtin_amdgcn_sched_barrier(0);              // (or all chunks are widened to 64 bits before the first sum)
    }
    const bool wide = c + NT * E < p.c1 && p.nrl == 1;          // one group, wider than the workgroup
    const int64_t behind = (int64_t)p.rl + (int64_t)NCH * p.nrl;
    for (int64_t r = behind; r < len; r += p.nrl) gn_add<T, K>(sum, sq, gn_load<FULL>(x + (t0 + r) * a.xs, c, p.c1));
    if (wide)
        for (int64_t r = p.rl; r < len; ++r)
            for (int cc = c + NT * E; cc < p.c1; cc += NT * E) gn_add<T, K>(sum, sq, gn_load<FULL>(x + (t0 + r) * a.xs, cc, p.c1));
    double2 tot;
    const int g = gn_join<T, NT, K>(a, p, sum, sq, s_red, tot);
    if (g >= 0) s_stat[g] = gn_finish(tot, (double)len * a.per, a.eps);
    __syncthreads();
    if (p.rl >= len || c >= p.c1) return;
    gn_affine<E> f;
    gn_affine_of<T, NT, K>(a, p, c, s_stat, f);
    // kept as they lie in memory: without this the compiler keeps every element unpacked from the sums on
#pragma unroll
    for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(held[i]));
    char *yu = (char *)(y + t0 * a.ys);
    const uint32_t y0 = (uint32_t)(p.rl * (int)a.ys) * sizeof(T), y_step = (uint32_t)(p.nrl * (int)a.ys) * sizeof(T);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i < mine) gn_store<T, ACT, FULL>(held[i], f, (T *)(yu + (y0 + i * y_step)), c, p.c1);
    for (int64_t r = behind; r < len; r += p.nrl) gn_store<T, ACT, FULL>(gn_load<FULL>(x + (t0 + r) * a.xs, c, p.c1), f, y + (t0 + r) * a.ys, c, p.c1);
    if (wide)
        for (int cc = c + NT * E; cc < p.c1; cc += NT * E) {
            gn_affine_of<T, NT, K>(a, p, cc, s_stat, f);
            for (int64_t r = p.rl; r < len; ++r) gn_store<T, ACT, FULL>(gn_load<FULL>(x + (t0 + r) * a.xs, cc, p.c1), f, y + (t0 + r) * a.ys, cc, p.c1);
        }
}

// As above, one group a slice, for slices that fill the registers: workgroups go from one (utterance, group) to the next, and while one's
// results leave the next one's rows come into the registers that they free.  (Without that a compute unit's two workgroups load,
// compute and store in step: 634 us for 384 k rows of 1024 in 32 groups.)  Neighbouring groups, which share lines of memory, run on
// one die (workgroups are dealt to the 8 dies in turn; 577 -> 534 us).  384 k rows of 1024 in 32 groups with GELU: 505 us, 3.1 TB/s; 280
// us of it are vector instructions, 28 a value, which the memory's time comes on top of: all 16 wavefronts are in one phase.
template <typename T, int NT, int NCH, int ACT>
__global__ __launch_bounds__(NT, 4)
void gnorm_stream_kernel(gn_args a)
{
    constexpr int E = 16 / sizeof(T);
    __shared__ double2 s_red[NT];
    __shared__ gn_stat s_stat[1];
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const int64_t items = (int64_t)a.n_utt * a.n_groups;
    const int cw = a.per / E, nrl = NT / cw, rl = (int)threadIdx.x / cw, ck = (int)threadIdx.x - rl * cw;
    const uint32_t x_step = (uint32_t)(nrl * (int)a.xs) * sizeof(T), y_step = (uint32_t)(nrl * (int)a.ys) * sizeof(T);
    const uint32_t x0 = (uint32_t)((rl < nrl ? rl : 0) * (int)a.xs + ck * E) * sizeof(T), y0 = (uint32_t)((rl < nrl ? rl : 0) * (int)a.ys + ck * E) * sizeof(T);
    // the next item that has rows, from `item` on
    auto next_of = [&](int64_t item, int &t0, int &len) {
        for (; item < items; item += gridDim.x) {
            const int u = (int)(item / a.n_groups);
            t0 = max(a.off[u], 0);
            len = min(a.off[u + 1], a.total) - t0;
            if (len > 0) break;
        }
        return item;
    };
    int t0 = 0, len = 0;
    int64_t item = next_of((gridDim.x & 7) == 0 ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x, t0, len);
    if (item >= items) return;
    net_u32x4 held[NCH];
    int mine = rl < nrl && rl < len ? (len - 1 - rl) / nrl + 1 : 0;
    const char *xu = (const char *)(x + t0 * a.xs + (item % a.n_groups) * a.per);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        held[i] = {};
        if (i < mine) held[i] = __builtin_bit_cast(net_u32x4, *(const net_pack<T, E> *)(xu + (x0 + i * x_step)));
    }
    while (item < items) {
        const int c = (int)(item % a.n_groups) * a.per + ck * E;
        double sum[1] = {}, sq[1] = {};
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            gn_add<T, 1>(sum, sq, held[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        // rows beyond the registers
#pragma unroll 1
        for (int i = NCH; i < mine; ++i) gn_add<T, 1>(sum, sq, __builtin_bit_cast(net_u32x4, *(const net_pack<T, E> *)(x + ((int64_t)t0 + rl + (int64_t)i * nrl) * a.xs + c)));
        double s = sum[0], q = sq[0];
        gn_sum_lanes(s, q, 64);
        if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = make_double2(s, q);
        __syncthreads();
        if (threadIdx.x < 64) {
            const double2 v = threadIdx.x < NT / 64 ? s_red[threadIdx.x] : make_double2(0.0, 0.0);
            s = v.x; q = v.y;
            gn_sum_lanes(s, q, NT / 64);
            if (threadIdx.x == 0) s_stat[0] = gn_finish(make_double2(s, q), (double)len * a.per, a.eps);
        }
        __syncthreads();
        const gn_stat st = s_stat[0];
        gn_affine<E> f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            f.mhi[e] = st.mhi;
            f.mlo[e] = st.mlo;
            f.rw[e] = a.weight ? st.rstd * a.weight[c + e] : st.rstd;
            f.b[e] = a.bias ? a.bias[c + e] : 0.0f;
        }
        const int was = mine, t_was = t0;
        char *yu = (char *)(y + t0 * a.ys + (c - ck * E));
        item = next_of(item + gridDim.x, t0, len);
        mine = item < items && rl < nrl && rl < len ? (len - 1 - rl) / nrl + 1 : 0;
        if (item < items) xu = (const char *)(x + t0 * a.xs + (item % a.n_groups) * a.per);
#pragma unroll
        for (int i = 0; i < NCH; ++i) asm volatile("" : "+v"(held[i]));
        uint32_t xo = x0, yo = y0;
        asm volatile("" : "+v"(xo), "+v"(yo));          // (or all 2 NCH offsets are kept in registers from item to item)
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if (i < was) gn_store<T, ACT, true>(held[i], f, (T *)(yu + yo), 0, E);
            held[i] = {};
            if (i < mine) held[i] = __builtin_bit_cast(net_u32x4, *(const net_pack<T, E> *)(xu + xo));
            xo += x_step;
            yo += y_step;
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll 1
        for (int i = NCH; i < was; ++i) {
            const int64_t r = (int64_t)t_was + rl + (int64_t)i * nrl;
            gn_store<T, ACT, true>(__builtin_bit_cast(net_u32x4, *(const net_pack<T, E> *)(x + r * a.xs + c)), f, y + r * a.ys, c, c + E);
        }
    }
}

// ---- tiles of rows, in two passes: 102 k rows of 429 floats in 47 + 94 us, 3.7 TB/s ------------------------------------------------------
// Every tile of the second pass sums all of its utterance's tiles anew, which is nothing for 30 s of audio (188 tiles: 24 us in all for one
// utterance) but grows with the square of its length: 65536 frames of 1024 in bfloat16 take 964 us, where a copy takes 38.
// Rows row .. tile_end - 1 begin in which utterance, and how far it reaches; false: no more utterances in the tile.  Partial sums lie
// at tile + utterance: along the rows one of the two grows from piece to piece, so every piece has a place of its own.
__device__ __forceinline__ bool gn_next(const gn_args &a, int &row, int tile_end, int &u, int &end)
{
    while (row < tile_end) {
        u = __builtin_amdgcn_readfirstlane(net_utt_of_rows(a.off, a.n_utt, row));
        if (u >= 0) {
            end = min(a.off[u + 1], tile_end);
            return true;
        }
        const int first = a.off[0];
        if (first <= row) return false;
        row = first;
    }
    return false;
}

template <typename T, int NT, int K, bool FULL>
__global__ __launch_bounds__(NT)
void gnorm_sums_kernel(gn_args a)
{
    constexpr int E = 16 / sizeof(T);
    __shared__ double2 s_red[NT * K];
    const gn_place<T, NT> p(a, blockIdx.x);
    const int tile = blockIdx.y;
    const int tile_end = (int)min(((int64_t)tile + 1) * a.tile_rows, (int64_t)a.total);
    int row = tile * a.tile_rows, u, end;
    const T *x = (const T *)a.x;
    while (gn_next(a, row, tile_end, u, end)) {
        double sum[K] = {}, sq[K] = {};
        for (int c = p.c0 + p.ck * E; c < p.c1; c += NT * E) {
            int64_t r = (int64_t)row + p.rl;
            for (; r + 3 * p.nrl < end; r += 4 * p.nrl) {
                net_u32x4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = gn_load<FULL>(x + (r + i * p.nrl) * a.xs, c, p.c1);
#pragma unroll
                for (int i = 0; i < 4; ++i) gn_add<T, K>(sum, sq, v[i]);
            }
            for (; r < end; r += p.nrl) gn_add<T, K>(sum, sq, gn_load<FULL>(x + r * a.xs, c, p.c1));
        }
        double2 tot;
        const int g = gn_join<T, NT, K>(a, p, sum, sq, s_red, tot);
        if (g >= 0) a.part[((size_t)tile + u) * a.n_groups + p.g0 + g] = tot;
        __syncthreads();
        row = end;
    }
}

template <typename T, int NT, int K, bool FULL, int ACT>
__global__ __launch_bounds__(NT, 4)
void gnorm_apply_kernel(gn_args a)
{
    constexpr int E = 16 / sizeof(T);
    __shared__ gn_stat s_stat[NT];
    const gn_place<T, NT> p(a, blockIdx.x);
    // the last tiles of the first pass are the first here: the caches may still hold them
    const int tile = gridDim.y - 1 - blockIdx.y;
    const int tile_end = (int)min(((int64_t)tile + 1) * a.tile_rows, (int64_t)a.total);
    int row = tile * a.tile_rows, u, end;
    const T *x = (const T *)a.x;
    T *y = (T *)a.y;
    const int lanes = gn_lanes<NT>(p.ng), g = (int)threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
    while (gn_next(a, row, tile_end, u, end)) {
        const int t0 = max(a.off[u], 0), t1 = min(a.off[u + 1], a.total);
        const int i0 = t0 / a.tile_rows, i1 = (t1 - 1) / a.tile_rows;
        double s = 0.0, q = 0.0;
        if (g < p.ng)
            for (int i = i0 + lane; i <= i1; i += lanes) {
                const double2 v = a.part[((size_t)i + u) * a.n_groups + p.g0 + g];
                s += v.x; q += v.y;
            }
        gn_sum_lanes(s, q, lanes);
        if (g < p.ng && lane == 0) s_stat[g] = gn_finish(make_double2(s, q), (double)(t1 - t0) * a.per, a.eps);
        __syncthreads();
        for (int c = p.c0 + p.ck * E; c < p.c1 && p.rl < end - row; c += NT * E) {
            gn_affine<E> f;
            gn_affine_of<T, NT, K>(a, p, c, s_stat, f);
            int64_t r = (int64_t)row + p.rl;
            for (; r + 3 * p.nrl < end; r += 4 * p.nrl) {
                net_u32x4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = gn_load<FULL>(x + (r + i * p.nrl) * a.xs, c, p.c1);
#pragma unroll
                for (int i = 0; i < 4; ++i) gn_store<T, ACT, FULL>(v[i], f, y + (r + i * p.nrl) * a.ys, c, p.c1);
            }
            for (; r < end; r += p.nrl) gn_store<T, ACT, FULL>(gn_load<FULL>(x + r * a.xs, c, p.c1), f, y + r * a.ys, c, p.c1);
        }
        __syncthreads();
        row = end;
    }
}

// ---- which way ---------------------------------------------------------------------------------------------------------------------
// At most so many tiles.  102 k rows of 429 in 11 groups, 1024 / 2048 / 4096 / 8192 of them: float32 145 / 151 / 142 / 149 us, bfloat16 109 / 125 /
// 143 / 188; 12800 rows: the same within 1 %.
constexpr int kGnTiles = 4096;

// rows of a tile: about kGnTiles tiles, of 16 rows or more
static inline int32_t gn_tile_rows(int32_t total) { const int32_t r = (int32_t)(((int64_t)total + kGnTiles - 1) / kGnTiles); return r < 16 ? 16 : (r + 15) / 16 * 16; }

extern "C" size_t psgpu_group_norm_work_bytes(int32_t n_utt, int32_t total_frames, int32_t n_groups)
{
    if (n_utt <= 0 || total_frames <= 0 || n_groups <= 0) return 0;
    const int32_t rows = gn_tile_rows(total_frames);
    return ((size_t)((total_frames - 1) / rows + 1) + (size_t)n_utt) * (size_t)n_groups * sizeof(double2);
}

// the groups a slice may have so that its chunks are at most nt, and (one statistic a work-item to keep) its groups at most nt
static int32_t gn_slice(int32_t n_groups, int32_t per, int e, int nt)
{
    int64_t gs = (int64_t)nt * e / per;
    if (gs > nt) gs = nt;
    if (gs > n_groups) gs = n_groups;
    return gs < 1 ? 1 : (int32_t)gs;
}

template <typename T, int ACT>
static void gn_run(gn_args a, hipStream_t st)
{
    constexpr int E = 16 / sizeof(T);
    const int64_t mean_len = ((int64_t)a.total + a.n_utt - 1) / a.n_utt;
    const bool one = a.per % E == 0;                    // a chunk lies in one group
    int64_t gs = gn_slice(a.n_groups, a.per, E, 256);
    auto chunks = [&](int64_t g) { return mean_len * ((g * a.per + E - 1) / E); };      // of an utterance's slice of g groups
    auto slices = [&](int64_t g) { return (a.n_groups + g - 1) / g; };
    // One launch where an utterance's group fits a workgroup's registers on average and there are enough of them: 256 work-items hold
    // 8 chunks each, 1024 hold 12.  1024 channels in 32 groups of bfloat16, held / stream / tiles, us (a replayed graph, 15 us of which are
    // the replay): 1 utterance of 64 frames 16.4 / - / 17.1, of 256 16.1 / - / 17.4; 4 of 500 17.8 / 18.7 / 23.6, 8 of 500 18.5 / 18.3 / 24.2, 16 of
    // 500 19.4 / 25.2 / 31.0; 64 of 256 23.2 / 69.5 / 33.6, of 512 41.6 / 73.3 / 53.0, of 1024 90.0 / 89.1 / 94.4.  Stream / tiles: 4 of 2000
    // 24.2 / 27.9, 16 of 2000 39.9 / 61.5, 32 of 2000 67 / 105, 64 of 2048 187 / 180, of 4096 356 / 322; float32 64 of 1024 143 / 168, of 2048 271 / 308.
    // The mean length decides, for the offsets are on the device: one long utterance among many short ones is one workgroup's a group, row
    // by row behind its registers (30 s among 511 single frames: 1330 us).
    const bool near_rows = a.xs < 1 << 16 && a.ys < 1 << 16;       // 1024 x 12 rows of them lie within 2^32 bytes
    if (near_rows && chunks(1) <= 256 * 8 && ((int64_t)a.total * a.n_chan <= 1 << 17 || (int64_t)a.n_utt * a.n_groups >= 256)) {
        while (gs > 1 && (chunks(gs) > 256 * 8 || a.n_utt * slices(gs) < 512)) gs = (gs + 1) / 2;
        a.gs = (int32_t)gs;
        const dim3 grid((uint32_t)slices(gs), (uint32_t)a.n_utt);
        if (one) gnorm_held_kernel<T, 256, 8, 1, true, ACT><<<grid, 256, 0, st>>>(a);
        else if (gs == 1) gnorm_held_kernel<T, 256, 8, 1, false, ACT><<<grid, 256, 0, st>>>(a);
        else gnorm_held_kernel<T, 256, 8, E, false, ACT><<<grid, 256, 0, st>>>(a);
        return;
    }
    if (near_rows && one && a.per <= 1024 * E && chunks(1) <= 1024 * 12 && (int64_t)a.n_utt * a.n_groups >= 512) {
        a.gs = 1;
        gnorm_stream_kernel<T, 1024, 12, ACT><<<256, 1024, 0, st>>>(a);              // one workgroup a compute unit
        return;
    }
    a.gs = (int32_t)gs;
    a.tile_rows = gn_tile_rows(a.total);
    const dim3 grid((uint32_t)slices(gs), (uint32_t)((a.total - 1) / a.tile_rows + 1));
    if (one) {
        gnorm_sums_kernel<T, 256, 1, true><<<grid, 256, 0, st>>>(a);
        gnorm_apply_kernel<T, 256, 1, true, ACT><<<grid, 256, 0, st>>>(a);
    } else if (gs == 1) {
        gnorm_sums_kernel<T, 256, 1, false><<<grid, 256, 0, st>>>(a);
        gnorm_apply_kernel<T, 256, 1, false, ACT><<<grid, 256, 0, st>>>(a);
    } else {
        gnorm_sums_kernel<T, 256, E, false><<<grid, 256, 0, st>>>(a);
        gnorm_apply_kernel<T, 256, E, false, ACT><<<grid, 256, 0, st>>>(a);
    }
}

template <typename T>
static void gn_run_act(const gn_args &a, int32_t act, hipStream_t st)
{
    switch (act) {
    case PSGPU_ACT_RELU: gn_run<T, PSGPU_ACT_RELU>(a, st); break;
    case PSGPU_ACT_SILU: gn_run<T, PSGPU_ACT_SILU>(a, st); break;
    case PSGPU_ACT_GELU: gn_run<T, PSGPU_ACT_GELU>(a, st); break;
    default: gn_run<T, PSGPU_ACT_NONE>(a, st);
    }
}

extern "C" int psgpu_group_norm_dev(int32_t dtype, const void *x_dev, int64_t x_stride, const int32_t *utt_off_dev, int32_t n_utt,
                                    int32_t total_frames, int32_t n_chan, int32_t n_groups, const float *weight_dev,
                                    const float *bias_dev, float eps, int32_t act, void *y_dev, int64_t y_stride, void *work_dev,
                                    size_t work_bytes, void *stream)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(net_dtype_ok(dtype), "psgpu_group_norm_dev: dtype %d", dtype);
    PSGPU_REQUIRE(n_utt >= 0 && n_utt <= 65535 && total_frames >= 0, "psgpu_group_norm_dev: %d frames of %d utterances (at most 65535)", total_frames, n_utt);
    PSGPU_REQUIRE(n_chan >= 1 && n_chan <= (1 << 30) && n_groups >= 1 && n_chan % n_groups == 0, "psgpu_group_norm_dev: %d channels in %d groups", n_chan, n_groups);
    PSGPU_REQUIRE(x_stride >= n_chan && y_stride >= n_chan, "psgpu_group_norm_dev: a row stride is below %d", n_chan);
    PSGPU_REQUIRE(act >= PSGPU_ACT_NONE && act <= PSGPU_ACT_GELU, "psgpu_group_norm_dev: activation %d", act);
    PSGPU_REQUIRE(std::isfinite(eps) && eps >= 0.0f, "psgpu_group_norm_dev: eps %g", (double)eps);
    if (total_frames == 0 || n_utt == 0) return PSGPU_OK;
    PSGPU_REQUIRE(x_dev && y_dev && utt_off_dev, "psgpu_group_norm_dev: NULL device buffer");
    const size_t es = net_dtype_size(dtype), need = psgpu_group_norm_work_bytes(n_utt, total_frames, n_groups);
    const size_t nx = net_span(total_frames, x_stride, n_chan, es), ny = net_span(total_frames, y_stride, n_chan, es);
    PSGPU_REQUIRE((x_dev == y_dev && x_stride == y_stride) || net_disjoint(x_dev, nx, y_dev, ny),
                  "psgpu_group_norm_dev: the output overlaps the input without being it");
    PSGPU_REQUIRE(work_bytes >= need && work_dev, "psgpu_group_norm_dev: %zu bytes of workspace, psgpu_group_norm_work_bytes asks for %zu", work_bytes, need);
    PSGPU_REQUIRE(((uintptr_t)work_dev & 15) == 0, "psgpu_group_norm_dev: the workspace is not aligned to 16 bytes");
    PSGPU_REQUIRE(net_disjoint(x_dev, nx, work_dev, need) && net_disjoint(y_dev, ny, work_dev, need), "psgpu_group_norm_dev: the workspace overlaps the input or the output");
    const int rc = net_check_device(nullptr);
    if (rc != PSGPU_OK) return rc;
    gn_args a = {};
    a.x = x_dev; a.xs = x_stride; a.off = utt_off_dev; a.n_utt = n_utt; a.total = total_frames; a.n_chan = n_chan; a.per = n_chan / n_groups;
    a.n_groups = n_groups; a.weight = weight_dev; a.bias = bias_dev; a.eps = eps; a.y = y_dev; a.ys = y_stride; a.part = (double2 *)work_dev;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == PSGPU_DT_F32) gn_run_act<float>(a, act, st);
    else if (dtype == PSGPU_DT_F16) gn_run_act<psg_half>(a, act, st);
    else gn_run_act<psg_bf16>(a, act, st);
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
