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

constexpr int kScrThreads = 256;

template <typename T>
__global__ __launch_bounds__(kScrThreads)
void netscr_row_kernel(const T *__restrict__ z, int64_t z_stride, int32_t n_sen, const float *__restrict__ prior, double unit,
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
        const double l = like(s);
        int q = 32767;
        if (l == ml && l != -INFINITY) q = 0;
        else if (l == l) {
            const double d = floor((ml - l) * unit + 0.5);
            if (d < 32767.0) q = (int)d;
        }
        out[t * out_stride + s] = (int16_t)q;
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
    const dim3 grid((uint32_t)total_frames);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == PSGPU_DT_F32)
        netscr_row_kernel<float><<<grid, kScrThreads, 0, st>>>((const float *)logits_dev, logits_stride, n_sen, log_prior_dev, unit, senscr_dev, senscr_stride, best_dev);
    else if (dtype == PSGPU_DT_F16)
        netscr_row_kernel<psg_half><<<grid, kScrThreads, 0, st>>>((const psg_half *)logits_dev, logits_stride, n_sen, log_prior_dev, unit, senscr_dev, senscr_stride, best_dev);
    else
        netscr_row_kernel<psg_bf16><<<grid, kScrThreads, 0, st>>>((const psg_bf16 *)logits_dev, logits_stride, n_sen, log_prior_dev, unit, senscr_dev, senscr_stride, best_dev);
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
