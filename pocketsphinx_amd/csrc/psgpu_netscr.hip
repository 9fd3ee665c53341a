// psgpu_netscr.hip -- senone scores of an acoustic network's outputs: what ps_decode_senscr() / acmod_set_insenfh() read from a file
// (reference src/pocketsphinx.c:1199-1218), made on the device in the searches' format.
//
//   l[t,s]      = z[t,s] - log_prior[s]
//   senscr[t,s] = min(32767, floor((max_s' l[t,s'] - l[t,s]) * scale / (1024 ln(logbase)) + 1/2))
//   best[t]     = max_s l[t,s] - log sum_s exp z[t,s]
//
// The logarithm of the softmax's sum is the same for every senone of a frame and leaves with the frame's best, as
// ptm_mgau_senone_eval's normalisation does (ptm_mgau.c:398-400); it stays in best[] alone.  Differences are taken in 64 bits: a score
// next to a rounding border is decided by their last bits, and the reference's scores are whole numbers that a search compares.
#include "psgpu_net_dev.h"
#include <atomic>
#include <cmath>

// Memory bounds it: a row is read once, kept in registers, and its scores are written; 64-bit arithmetic is spent on few elements.
constexpr int kScrThreads = 256;

// one score in 64 bits
__device__ __forceinline__ int scr_exact(double l, double top, double unit)
{
    if (l == top && l != -INFINITY) return 0;
    if (l != l) return 32767;
    const double d = floor((top - l) * unit + 0.5);
    return d < 32767.0 ? (int)d : 32767;
}

typedef short scr_short2 __attribute__((ext_vector_type(2)));
template <int N> struct __attribute__((packed, aligned(2))) scr_pack { int16_t v[N]; };

// rows longer than the registers: read three times
template <typename T>
__global__ __launch_bounds__(kScrThreads)
void netscr_long_kernel(const T *__restrict__ z, int64_t z_stride, int32_t n_sen, const float *__restrict__ prior, double unit,
                        int16_t *__restrict__ out, int64_t out_stride, float *__restrict__ best)
{
    __shared__ double s_l[kScrThreads / 64];
    __shared__ float s_z[kScrThreads / 64];
    __shared__ double s_sum[kScrThreads / 64];
    const size_t t = blockIdx.x;
    const int tid = threadIdx.x;
    const T *row = z + t * z_stride;
    auto like = [&](int s) { return (double)net_f32(row[s]) - (prior ? (double)prior[s] : 0.0); };
    double ml = -INFINITY;
    float mz = -INFINITY;
    bool nan = false;
    for (int s = tid; s < n_sen; s += kScrThreads) {
        ml = fmax(ml, like(s));                    // (fmax steps over a NaN)
        const float v = net_f32(row[s]);
        mz = fmaxf(mz, v);
        nan |= v != v;
    }
    for (int o = 32; o; o >>= 1) { ml = fmax(ml, __shfl_xor(ml, o)); mz = fmaxf(mz, __shfl_xor(mz, o)); }
    if ((tid & 63) == 0) { s_l[tid >> 6] = ml; s_z[tid >> 6] = mz; }
    nan = __syncthreads_or(nan);
    for (int w = 0; w < kScrThreads / 64; ++w) { ml = fmax(ml, s_l[w]); mz = fmaxf(mz, s_z[w]); }
    double sum = 0.0;
    for (int s = tid; s < n_sen; s += kScrThreads) {
        out[t * out_stride + s] = (int16_t)scr_exact(like(s), ml, unit);
        sum += (double)expf(net_f32(row[s]) - mz);
    }
    if (!best) return;
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
        for (int w = 0; w < kScrThreads / 64; ++w) sum += s_sum[w];
        best[t] = nan ? NAN : (mz == -INFINITY ? -INFINITY : (float)(ml - ((double)mz + log(sum))));
    }
}

// numbers in the order of unsigned integers; not for NaN
__device__ __forceinline__ unsigned long long scr_key(double v)
{
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double scr_value(unsigned long long k) { return __longlong_as_double((long long)(k >> 63 ? k ^ 1ull << 63 : ~k)); }

// A row a workgroup, NCH chunks of 16 bytes a work-item, in registers, the next row on its way; the priors are fetched once for all of
// a workgroup's rows.  96 k rows of 5126 in bfloat16: 533 us, 3.7 TB/s; vector instructions, 29 a value, are 360 us of it.
//
// l in 32 bits, lf = fl(z - prior), keeps the order: the best l is among those whose lf is the greatest, and only those are taken in 64
// bits.  A score's q = (top - l) unit + 1/2 in 32 bits is off by at most c + 6 q 2^-23, c = (2 |top| unit + 4) 2^-23: the three
// differences round by 2^-24 of |top|, |l| <= |top| + (top - l) and top - l, the products and sums by 2^-24 of q each, and twice all that is
// allowed.  Where q less that and q plus that have one whole part it is the score's; else the score is taken in 64 bits (2 in 10000
// of a network's outputs).  The conversion to 16 bits ends at 32767, where a NaN and a masked senone are taken too (a minimum steps
// over a NaN).  `plain` says that unit is not so far from 1 that these steps leave float's range; without it, or with a best that is
// not finite, all scores are taken in 64 bits.
//
// The softmax's sum: exp(z - m) = 2^(z a - m a) in one fused step, a = log2(e) in 32 bits; m a rounded is b, which all terms share, and
// the logarithm gets b - m a back in 64 bits.  b - m a is up to half of b's last place, and 2 to it a factor of all terms: for m up to 1e6 one
// of 2^(1/16), beyond 1e10 one that leaves float's range.  A row whose m is beyond 1e6 (masked as a whole by a low finite value, say)
// takes 2^((z - m) a) instead, from memory.
template <typename T, int NT, int NCH>
__global__ __launch_bounds__(NT, 4)
void netscr_row_kernel(const T *__restrict__ z, int64_t z_stride, int32_t rows, int32_t n_sen, const float *__restrict__ prior, double unit,
                       int plain, int16_t *__restrict__ out, int64_t out_stride, float *__restrict__ best)
{
    constexpr int E = 16 / sizeof(T), W = NT / 64;
    constexpr uint32_t kMask = sizeof(T) == 4 ? 0xff800000u : __is_same(T, psg_half) ? 0xfc00fc00u : 0xff80ff80u;      // minus infinity
    __shared__ float s_l[2][W], s_z[2][W];
    __shared__ double s_sum[2][W];
    __shared__ unsigned long long s_top[2];
    const int tid = threadIdx.x, wave = tid >> 6;
    const float unitf = (float)unit;
    float pr[NCH][E];
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int s = (i * NT + tid) * E + e;
            pr[i][e] = prior && s < n_sen ? prior[s] : 0.0f;
        }
    net_u32x4 v[NCH], next[NCH];                            // the row, and the one behind it on its way
    auto fetch = [&](const T *row) {
        int n = n_sen, me = tid;                            // (not to be turned into a dozen values that live through the rows' loop)
        asm volatile("" : "+s"(n), "+v"(me));
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int s = (i * NT + me) * E;
            next[i] = net_u32x4{kMask, kMask, kMask, kMask};
            if (s + E <= n) next[i] = __builtin_bit_cast(net_u32x4, *(const net_pack<T, E> *)((const char *)row + (uint32_t)(i * NT + me) * 16));
            else if (s < n) {                               // the row's last E, moved down; the places behind its end are masked
                const int by = (s + E - n) * (int)sizeof(T) * 8;
                const unsigned __int128 w = __builtin_bit_cast(unsigned __int128, *(const net_pack<T, E> *)(row + (n - E)));
                next[i] = __builtin_bit_cast(net_u32x4, w >> by | __builtin_bit_cast(unsigned __int128, next[i]) << (128 - by));
            }
        }
    };
    fetch(z + (int64_t)blockIdx.x * z_stride);
    int par = 0;
    for (int64_t t = blockIdx.x; t < rows; t += gridDim.x, par ^= 1) {
        const T *row = z + t * z_stride;
#pragma unroll
        for (int i = 0; i < NCH; ++i) v[i] = next[i];
        if (tid == 0) s_top[par] = scr_key(-INFINITY);
        float ml = -INFINITY, mz = -INFINITY;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            asm volatile("" : "+v"(v[i]));                  // (kept as they lie in memory, unpacked where they are used)
            if ((i * NT + wave * 64) * E >= n_sen) break;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float ze = net_elem<T>(v[i], e);
                ml = fmaxf(ml, ze - pr[i][e]);              // (fmaxf steps over a NaN)
                mz = fmaxf(mz, ze);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        const float own = ml;
        for (int o = 32; o; o >>= 1) { ml = fmaxf(ml, __shfl_xor(ml, o)); mz = fmaxf(mz, __shfl_xor(mz, o)); }
        if ((tid & 63) == 0) { s_l[par][wave] = ml; s_z[par][wave] = mz; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) { ml = fmaxf(ml, s_l[par][w]); mz = fmaxf(mz, s_z[par][w]); }
        if (t + gridDim.x < rows) fetch(row + gridDim.x * z_stride);
        if (own == ml) {                                    // the best may be here
            double mine = -INFINITY;
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float ze = net_elem<T>(v[i], e), p = pr[i][e];
                    if (ze - p == ml) {
                        asm volatile("" : "+v"(ze), "+v"(p));       // (or every prior is widened to 64 bits beforehand)
                        mine = fmax(mine, (double)ze - (double)p);
                    }
                }
            atomicMax(&s_top[par], scr_key(mine));
        }
        const float a = 1.4426950408889634f;
        const bool huge = !(fabsf(mz) < 1e6f);
        const float b = huge ? 0.0f : mz * a;
        double total = 0.0;
        if (best) {
            float sum = 0.0f;
            if (!huge) {
#pragma unroll
                for (int i = 0; i < NCH; ++i) {
                    asm volatile("" : "+v"(v[i]));
                    if ((i * NT + wave * 64) * E >= n_sen) break;
#pragma unroll
                    for (int e = 0; e < E; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(net_elem<T>(v[i], e), a, -b));
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll 1
                for (int s = tid; s < n_sen; s += NT) {
                    const float ze = net_f32(row[s]);
                    sum += ze == mz ? 1.0f : __builtin_amdgcn_exp2f((ze - mz) * a);       // (also for two infinities)
                }
            }
            total = sum;
            for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o);
            if ((tid & 63) == 0) s_sum[par][wave] = total;
        }
        __syncthreads();
        const double top = scr_value(s_top[par]);
        if (best && tid == 0) {
            total = 0.0;
            for (int w = 0; w < W; ++w) total += s_sum[par][w];
            if (mz > -INFINITY)                             // (a NaN among the outputs is one in the sum)
                best[t] = (float)(top - ((double)mz + ((double)logf((float)total) + (huge ? 0.0 : (double)b - (double)mz * (double)a) * 0.69314718055994531)));
            else {
                bool nan = false;
                for (int s = 0; s < n_sen; ++s) { const float ze = net_f32(row[s]); nan |= ze != ze; }
                best[t] = nan ? NAN : -INFINITY;
            }
        }
        const float topf = ml, c = __builtin_fmaf(fabsf(topf) * 2.0f, unitf, 4.0f) * 0x1p-23f;
        const bool far = !plain || !(fabsf(topf) < INFINITY);       // then the two are 0 and -5: unlike everywhere
        const float unit0 = far ? 0.0f : unitf * (1.0f - 6 * 0x1p-23f), unit1 = far ? 0.0f : unitf * (1.0f + 6 * 0x1p-23f);
        const float half0 = far ? 0.0f : 0.5f - c, half1 = far ? -5.0f : 0.5f + c;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            int me = tid;
            asm volatile("" : "+v"(v[i]), "+v"(me));
            __builtin_amdgcn_sched_barrier(0);
            const int s = (i * NT + me) * E;
            if (s >= n_sen) break;
            struct { scr_short2 v[E / 2]; } lo_;
            auto &lo = lo_.v;
            bool unsure[E / 2], any = false;
#pragma unroll
            for (int e = 0; e < E; e += 2) {
                const float d0 = fminf(topf - (net_elem<T>(v[i], e) - pr[i][e]), 3e38f), d1 = fminf(topf - (net_elem<T>(v[i], e + 1) - pr[i][e + 1]), 3e38f);
                lo[e / 2] = __builtin_amdgcn_cvt_pk_i16((int)__builtin_fmaf(d0, unit0, half0), (int)__builtin_fmaf(d1, unit0, half0));
                const scr_short2 hi = __builtin_amdgcn_cvt_pk_i16((int)__builtin_fmaf(d0, unit1, half1), (int)__builtin_fmaf(d1, unit1, half1));
                unsure[e / 2] = __builtin_bit_cast(uint32_t, lo[e / 2]) != __builtin_bit_cast(uint32_t, hi);
                any |= unsure[e / 2];
            }
            int16_t *to = out + t * out_stride + s;
            if (s + E <= n_sen) *(scr_pack<E> *)to = __builtin_bit_cast(scr_pack<E>, lo_);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (s + e < n_sen) to[e] = lo[e / 2][e & 1];
            if (any) {
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < E; e += 2) m |= unsure[e / 2] ? 3u << e : 0u;
                while (m) {
                    const int e = __builtin_ctz(m);
                    m &= m - 1;
                    if (s + e < n_sen) to[e] = (int16_t)scr_exact((double)net_f32(row[s + e]) - (prior ? (double)prior[s + e] : 0.0), top, unit);
                }
            }
        }
    }
}

template <typename T>
static void scr_run(const void *z, int64_t zs, int32_t rows, int32_t n_sen, const float *prior, double unit, int16_t *out, int64_t os, float *best, hipStream_t st)
{
    constexpr int E = 16 / sizeof(T);
    const int plain = unit >= 1e-6 && unit <= 1e6;
    const int64_t chunks = ((int64_t)n_sen + E - 1) / E;
    // Workgroups that run at once (4 a compute unit), or twice as many where a row more or less in some does not count.  Rows of 5126 in
    // bfloat16, 1024 / 2048 workgroups, us: 4096 rows 38.7 / 43.5, 16384 rows 109 / 111, 32768 rows 199 / 200, 96 k rows 542 / 535; float32: 58.0 / 62.7,
    // 213 / 217, 413 / 416, 1193 / 1197.  Few rows: all of a compute unit's wavefronts on each.  256 / 1024 work-items a row: 512 rows 16.3 / 17.6, 1024
    // rows 21.3 / 27.5, 2048 rows 27.7 / 37.6; float32 16.9 / 18.9, 23.8 / 23.9, 35.3 / 35.4; 256 rows and fewer the same.
    const int32_t most = rows < 16384 ? 1024 : 2048;
#define ROWS(NT, NCH) netscr_row_kernel<T, NT, NCH><<<(uint32_t)(rows < most ? rows : most), NT, 0, st>>>((const T *)z, zs, rows, n_sen, prior, unit, plain, out, os, best)
    if (n_sen < E) netscr_long_kernel<T><<<(uint32_t)rows, kScrThreads, 0, st>>>((const T *)z, zs, n_sen, prior, unit, out, os, best);
    else if (rows > 512 && chunks <= 256 * 4) {
        if (chunks <= 256) ROWS(256, 1);
        else if (chunks <= 256 * 2) ROWS(256, 2);
        else if (chunks <= 256 * 3) ROWS(256, 3);
        else ROWS(256, 4);
    } else if (chunks <= 1024) ROWS(1024, 1);
    else if (chunks <= 1024 * 2) ROWS(1024, 2);
    else if (chunks <= 1024 * 3) ROWS(1024, 3);
    else if (chunks <= 1024 * 5) ROWS(1024, 5);
    else netscr_long_kernel<T><<<(uint32_t)rows, kScrThreads, 0, st>>>((const T *)z, zs, n_sen, prior, unit, out, os, best);
#undef ROWS
}

// hipGetDeviceProperties costs more than a launch: its answer for a device is kept
int net_check_device(int *device)
{
    static std::atomic<uint8_t> good[64];
    int d = -1;
    if (hipGetDevice(&d) == hipSuccess && d >= 0 && d < 64 && good[d].load(std::memory_order_relaxed)) {
        if (device) *device = d;
        return PSGPU_OK;
    }
    const int rc = psgpu_check_device();
    if (rc != PSGPU_OK) return rc;
    if (d >= 0 && d < 64) good[d].store(1, std::memory_order_relaxed);
    if (device) *device = d;
    return PSGPU_OK;
}

extern "C" int psgpu_senone_scores_dev(int32_t dtype, const void *logits_dev, int64_t logits_stride, int32_t total_frames, int32_t n_sen,
                                       const float *log_prior_dev, double scale, double logbase, int16_t *senscr_dev,
                                       int64_t senscr_stride, float *best_dev, void *stream)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(net_dtype_ok(dtype), "psgpu_senone_scores_dev: dtype %d", dtype);
    PSGPU_REQUIRE(total_frames >= 0 && n_sen >= 1, "psgpu_senone_scores_dev: %d frames of %d senones", total_frames, n_sen);
    PSGPU_REQUIRE(logits_stride >= n_sen && senscr_stride >= n_sen, "psgpu_senone_scores_dev: a row stride is below %d", n_sen);
    PSGPU_REQUIRE(std::isfinite(scale) && scale > 0.0, "psgpu_senone_scores_dev: scale %g", scale);
    PSGPU_REQUIRE(std::isfinite(logbase) && logbase > 1.0, "psgpu_senone_scores_dev: logbase %g", logbase);
    if (total_frames == 0) return PSGPU_OK;
    PSGPU_REQUIRE(logits_dev && senscr_dev, "psgpu_senone_scores_dev: NULL device buffer");
    PSGPU_REQUIRE(net_disjoint(logits_dev, net_span(total_frames, logits_stride, n_sen, net_dtype_size(dtype)), senscr_dev,
                               net_span(total_frames, senscr_stride, n_sen, 2)), "psgpu_senone_scores_dev: the scores overlap the logits");
    const int rc = net_check_device(nullptr);
    if (rc != PSGPU_OK) return rc;
    const double unit = scale / (std::log(logbase) * (double)(1 << kSenscrShift));
    const hipStream_t st = (hipStream_t)stream;
#define RUN(T) scr_run<T>(logits_dev, logits_stride, total_frames, n_sen, log_prior_dev, unit, senscr_dev, senscr_stride, best_dev, st)
    if (dtype == PSGPU_DT_F32) RUN(float);
    else if (dtype == PSGPU_DT_F16) RUN(psg_half);
    else RUN(psg_bf16);
#undef RUN
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
