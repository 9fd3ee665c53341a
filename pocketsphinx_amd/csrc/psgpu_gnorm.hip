// psgpu_gnorm.hip -- group norm with an activation over packed utterances, channels last.
//
//   m, v     = mean and biased variance of x[t, c] over the utterance's frames t and the group's channels c
//   y[t, c]  = act((x[t, c] - m) / sqrt(v + eps) * weight[c] + bias[c])
//
// What cmn() with -varnorm is for cepstra (reference src/feat/cmn.c:166-233), per group of channels and with a learned scale.
// Sums run in 64 bits: sum x^2 - n m^2 then keeps its digits for groups whose mean is far above their spread.
#include "psgpu_net_dev.h"
#include <cmath>

constexpr int kGnThreads = 256;

__device__ __forceinline__ float gn_act(int act, float v)
{
    switch (act) {
    case PSGPU_ACT_RELU: return v < 0.0f ? 0.0f : v;                              // (a NaN stays one)
    case PSGPU_ACT_SILU: return v / (1.0f + expf(-v));
    case PSGPU_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    default: return v;
    }
}

template <typename T>
__global__ __launch_bounds__(kGnThreads)
void gnorm_group_kernel(const T *x, int64_t x_stride, const int32_t *__restrict__ utt_off, int32_t total, int32_t n_chan, int32_t per,
                        const float *__restrict__ weight, const float *__restrict__ bias, float eps, int act, T *y, int64_t y_stride)
{
    __shared__ double s_sum[kGnThreads / 64], s_sq[kGnThreads / 64];
    const int u = blockIdx.y, c0 = blockIdx.x * per, tid = threadIdx.x;
    const int t0 = max(utt_off[u], 0), t1 = min(utt_off[u + 1], total);
    if (t1 <= t0) return;
    const int64_t n = (int64_t)(t1 - t0) * per;
    double sum = 0.0, sq = 0.0;
    for (int64_t i = tid; i < n; i += kGnThreads) {
        const double v = (double)net_f32(x[(t0 + i / per) * x_stride + c0 + i % per]);
        sum += v;
        sq += v * v;
    }
    for (int o = 32; o; o >>= 1) { sum += __shfl_xor(sum, o); sq += __shfl_xor(sq, o); }
    if ((tid & 63) == 0) { s_sum[tid >> 6] = sum; s_sq[tid >> 6] = sq; }
    __syncthreads();
    sum = sq = 0.0;
    for (int w = 0; w < kGnThreads / 64; ++w) { sum += s_sum[w]; sq += s_sq[w]; }
    const double mean = sum / (double)n;
    double var = sq / (double)n - mean * mean;
    if (var < 0.0) var = 0.0;                       // (a NaN stays one)
    const float rstd = (float)(1.0 / sqrt(var + (double)eps)), mhi = (float)mean, mlo = (float)(mean - (double)mhi);
    for (int64_t i = tid; i < n; i += kGnThreads) {
        const int64_t t = t0 + i / per;
        const int c = c0 + (int)(i % per);
        float v = ((net_f32(x[t * x_stride + c]) - mhi) - mlo) * rstd;
        v = v * (weight ? weight[c] : 1.0f) + (bias ? bias[c] : 0.0f);
        y[t * y_stride + c] = net_cast<T>(gn_act(act, v));
    }
}

extern "C" size_t psgpu_group_norm_work_bytes(int32_t n_utt, int32_t total_frames, int32_t n_groups)
{
    return 0;
}

extern "C" int psgpu_group_norm_dev(int32_t dtype, const void *x_dev, int64_t x_stride, const int32_t *utt_off_dev, int32_t n_utt,
                                    int32_t total_frames, int32_t n_chan, int32_t n_groups, const float *weight_dev,
                                    const float *bias_dev, float eps, int32_t act, void *y_dev, int64_t y_stride, void *work_dev,
                                    size_t work_bytes, void *stream)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(net_dtype_ok(dtype), "psgpu_group_norm_dev: dtype %d", dtype);
    PSGPU_REQUIRE(n_utt >= 0 && n_utt <= 65535 && total_frames >= 0, "psgpu_group_norm_dev: %d frames of %d utterances (at most 65535)", total_frames, n_utt);
    PSGPU_REQUIRE(n_chan >= 1 && n_groups >= 1 && n_chan % n_groups == 0, "psgpu_group_norm_dev: %d channels in %d groups", n_chan, n_groups);
    PSGPU_REQUIRE(x_stride >= n_chan && y_stride >= n_chan, "psgpu_group_norm_dev: a row stride is below %d", n_chan);
    PSGPU_REQUIRE(act >= PSGPU_ACT_NONE && act <= PSGPU_ACT_GELU, "psgpu_group_norm_dev: activation %d", act);
    PSGPU_REQUIRE(std::isfinite(eps) && eps >= 0.0f, "psgpu_group_norm_dev: eps %g", (double)eps);
    if (total_frames == 0 || n_utt == 0) return PSGPU_OK;
    PSGPU_REQUIRE(x_dev && y_dev && utt_off_dev, "psgpu_group_norm_dev: NULL device buffer");
    const size_t es = net_dtype_size(dtype);
    PSGPU_REQUIRE((x_dev == y_dev && x_stride == y_stride)
                  || net_disjoint(x_dev, net_span(total_frames, x_stride, n_chan, es), y_dev, net_span(total_frames, y_stride, n_chan, es)),
                  "psgpu_group_norm_dev: the output overlaps the input without being it");
    PSGPU_REQUIRE(work_bytes >= psgpu_group_norm_work_bytes(n_utt, total_frames, n_groups) && (work_dev || !psgpu_group_norm_work_bytes(n_utt, total_frames, n_groups)),
                  "psgpu_group_norm_dev: %zu bytes of workspace, psgpu_group_norm_work_bytes asks for %zu", work_bytes,
                  psgpu_group_norm_work_bytes(n_utt, total_frames, n_groups));
    const int rc = net_check_device(nullptr);
    if (rc != PSGPU_OK) return rc;
    const dim3 grid((uint32_t)n_groups, (uint32_t)n_utt);
    const hipStream_t st = (hipStream_t)stream;
    const int per = n_chan / n_groups;
    if (dtype == PSGPU_DT_F32)
        gnorm_group_kernel<float><<<grid, kGnThreads, 0, st>>>((const float *)x_dev, x_stride, utt_off_dev, total_frames, n_chan, per, weight_dev, bias_dev, eps, act, (float *)y_dev, y_stride);
    else if (dtype == PSGPU_DT_F16)
        gnorm_group_kernel<psg_half><<<grid, kGnThreads, 0, st>>>((const psg_half *)x_dev, x_stride, utt_off_dev, total_frames, n_chan, per, weight_dev, bias_dev, eps, act, (psg_half *)y_dev, y_stride);
    else
        gnorm_group_kernel<psg_bf16><<<grid, kGnThreads, 0, st>>>((const psg_bf16 *)x_dev, x_stride, utt_off_dev, total_frames, n_chan, per, weight_dev, bias_dev, eps, act, (psg_bf16 *)y_dev, y_stride);
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
