// psgpu_proj.hip -- a shared projection of packed rows with low-rank adapters of many utterances.
//
//   y[t, o] = bias[o] + sum_k W[o, k] x[t, k] + s_a sum_r B_a[o, r] h[t, r],   h[t, r] = sum_k A_a[r, k] x[t, k]
//
// a = the adapter of the utterance row t belongs to: the speaker's correction of a transform that all share (what -lda is for the
// features, reference src/feat/lda.c:139-159, and -mllr for the means of one decoder's speaker, src/ps_mllr.c).  Products of the inputs'
// type, sums in 32 bits, one rounding at the end.
//
// psgpu_proj_t keeps the weights and every loaded adapter on the device, laid out once:
//   W  [Np][Kp], A per slot [Rp][Kp], B per slot [Np][Rp], zeros in the padding.
#include "psgpu_net_dev.h"
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

struct psgpu_proj_s {
    int device = 0;
    int32_t dtype = 0, d_in = 0, d_out = 0, max_adapters = 0, max_rank = 0;
    int32_t kp = 0, np = 0, rp = 0;                 // padded d_in, d_out, max_rank
    char *w = nullptr;
    float *bias = nullptr;                          // [np], zeros where there is none
    char *a = nullptr, *b = nullptr;                // [max_adapters] slots
    int32_t *rank = nullptr;                        // [max_adapters], 0: nothing loaded
    float *scale = nullptr;
};

constexpr int kProjNoRow = -2;                      // rows of no utterance: left as they are

// ---- one wavefront a row: which adapter it has, and h ------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(64)
void proj_shrink_kernel(const T *__restrict__ x, int64_t x_stride, int32_t d_in, int32_t kp, const T *__restrict__ a, int32_t rp,
                        const int32_t *__restrict__ rank, const float *__restrict__ scale, int32_t max_adapters,
                        const int32_t *__restrict__ utt_off, const int32_t *__restrict__ adapter, int32_t n_utt,
                        int32_t *__restrict__ row_slot, float *__restrict__ h)
{
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x;
    const int u = net_utt_of_row(utt_off, n_utt, (int)t);
    int slot = u < 0 ? kProjNoRow : (adapter ? adapter[u] : -1);
    if (slot >= 0 && (slot >= max_adapters || rank[slot] == 0)) slot = -1;
    if (slot < 0 && u >= 0) slot = -1;
    if (lane == 0) row_slot[t] = slot;
    if (slot < 0) return;
    const T *ar = a + (size_t)slot * rp * kp;
    const int r_n = rank[slot];
    for (int r = 0; r < r_n; ++r) {
        float s = 0.0f;
        for (int k = lane; k < d_in; k += 64) s += net_f32(x[t * x_stride + k]) * net_f32(ar[(size_t)r * kp + k]);
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) h[t * rp + r] = s * scale[slot];
    }
}

// ---- a 32 x 32 tile of y a workgroup ----------------------------------------------------------------------------------------------
constexpr int kTile = 32;
template <typename T, typename Y>
__global__ __launch_bounds__(256)
void proj_tile_kernel(const T *__restrict__ x, int64_t x_stride, int32_t rows, int32_t d_in, int32_t kp, const T *__restrict__ w,
                      const float *__restrict__ bias, int32_t d_out, const T *__restrict__ b, int32_t np, int32_t rp,
                      const int32_t *__restrict__ rank, const int32_t *__restrict__ row_slot, const float *__restrict__ h,
                      Y *__restrict__ y, int64_t y_stride)
{
    __shared__ float s_x[kTile][kTile + 1], s_w[kTile][kTile + 1];
    const int r0 = blockIdx.y * kTile, o0 = blockIdx.x * kTile, tid = threadIdx.x;
    const int o = tid & 31, r = tid >> 5;           // this work-item's column and its rows r, r + 8, r + 16, r + 24
    float acc[4] = {0, 0, 0, 0};
    for (int k0 = 0; k0 < d_in; k0 += kTile) {
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + r + 8 * i;
            s_x[r + 8 * i][o] = row < rows && k0 + o < d_in ? net_f32(x[(size_t)row * x_stride + k0 + o]) : 0.0f;
            s_w[r + 8 * i][o] = net_f32(w[(size_t)(o0 + r + 8 * i) * kp + k0 + o]);
        }
        __syncthreads();
        for (int k = 0; k < kTile; ++k)
            for (int i = 0; i < 4; ++i) acc[i] += s_x[r + 8 * i][k] * s_w[o][k];
        __syncthreads();
    }
    if (o0 + o >= d_out) return;
    for (int i = 0; i < 4; ++i) {
        const int row = r0 + r + 8 * i;
        if (row >= rows) continue;
        const int slot = row_slot ? row_slot[row] : -1;
        if (slot == kProjNoRow) continue;
        float v = acc[i] + bias[o0 + o];
        if (slot >= 0)
            for (int j = 0; j < rank[slot]; ++j) v += h[(size_t)row * rp + j] * net_f32(b[((size_t)slot * np + o0 + o) * rp + j]);
        y[(size_t)row * y_stride + o0 + o] = net_cast<Y>(v);
    }
}

static inline int32_t round_up(int32_t v, int32_t m) { return (v + m - 1) / m * m; }

extern "C" void psgpu_proj_free(psgpu_proj_t *p)
{
    if (!p) return;
    int cur = -1;
    (void)hipGetDevice(&cur);
    if (cur != p->device) (void)hipSetDevice(p->device);
    (void)hipFree(p->w); (void)hipFree(p->bias); (void)hipFree(p->a); (void)hipFree(p->b); (void)hipFree(p->rank); (void)hipFree(p->scale);
    if (cur >= 0 && cur != p->device) (void)hipSetDevice(cur);
    delete p;
}

// rows x cols elements of es bytes -> [rows_p][cols_p], zeros behind
static void pad_rows(std::vector<char> &dst, const void *src, size_t rows, size_t cols, size_t rows_p, size_t cols_p, size_t es)
{
    dst.assign(rows_p * cols_p * es, 0);
    for (size_t r = 0; r < rows; ++r) memcpy(dst.data() + r * cols_p * es, (const char *)src + r * cols * es, cols * es);
}

static int proj_fill(psgpu_proj_t *p, const void *weight, const float *bias)
{
    const size_t es = net_dtype_size(p->dtype), na = (size_t)p->max_adapters;
    std::vector<char> buf;
    pad_rows(buf, weight, p->d_out, p->d_in, p->np, p->kp, es);
    PSGPU_HIP(hipMalloc((void **)&p->w, buf.size()));
    PSGPU_HIP(hipMemcpy(p->w, buf.data(), buf.size(), hipMemcpyHostToDevice));
    buf.assign((size_t)p->np * 4, 0);
    if (bias) memcpy(buf.data(), bias, (size_t)p->d_out * 4);
    PSGPU_HIP(hipMalloc((void **)&p->bias, buf.size()));
    PSGPU_HIP(hipMemcpy(p->bias, buf.data(), buf.size(), hipMemcpyHostToDevice));
    if (!na) return PSGPU_OK;
    PSGPU_HIP(hipMalloc((void **)&p->a, na * p->rp * p->kp * es));
    PSGPU_HIP(hipMalloc((void **)&p->b, na * p->np * p->rp * es));
    PSGPU_HIP(hipMalloc((void **)&p->rank, na * 4));
    PSGPU_HIP(hipMalloc((void **)&p->scale, na * 4));
    buf.assign(na * 4, 0);
    PSGPU_HIP(hipMemcpy(p->rank, buf.data(), na * 4, hipMemcpyHostToDevice));
    PSGPU_HIP(hipMemcpy(p->scale, buf.data(), na * 4, hipMemcpyHostToDevice));
    return PSGPU_OK;
}

extern "C" int psgpu_proj_create(psgpu_proj_t **out, int32_t dtype, int32_t d_in, int32_t d_out, const void *weight, const float *bias,
                                 int32_t max_adapters, int32_t max_rank)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(out && weight, "psgpu_proj_create: NULL argument");
    *out = nullptr;
    PSGPU_REQUIRE(net_dtype_ok(dtype), "psgpu_proj_create: dtype %d", dtype);
    PSGPU_REQUIRE(d_in >= 1 && d_in <= (1 << 20) && d_out >= 1 && d_out <= (1 << 20), "psgpu_proj_create: %d inputs, %d outputs (1..2^20)", d_in, d_out);
    PSGPU_REQUIRE(max_adapters >= 0 && max_adapters <= 65536, "psgpu_proj_create: %d adapters (0..65536)", max_adapters);
    PSGPU_REQUIRE(max_adapters == 0 || (max_rank >= 1 && max_rank <= PSGPU_PROJ_MAX_RANK), "psgpu_proj_create: rank %d (1..%d)", max_rank, PSGPU_PROJ_MAX_RANK);
    int rc = psgpu_check_device();
    if (rc != PSGPU_OK) return rc;
    psgpu_proj_t *p = new (std::nothrow) psgpu_proj_t;
    if (!p) { psgpu_set_error("psgpu_proj_create: out of memory"); return PSGPU_ENOMEM; }
    p->device = psgpu_get_device();
    p->dtype = dtype; p->d_in = d_in; p->d_out = d_out; p->max_adapters = max_adapters; p->max_rank = max_adapters ? max_rank : 0;
    p->kp = round_up(d_in, 64); p->np = round_up(d_out, 256); p->rp = round_up(p->max_rank, 16);
    try { rc = proj_fill(p, weight, bias); }
    catch (const std::bad_alloc &) { psgpu_set_error("psgpu_proj_create: out of memory"); rc = PSGPU_ENOMEM; }
    if (rc != PSGPU_OK) { psgpu_proj_free(p); return rc; }
    *out = p;
    return PSGPU_OK;
}

static int proj_store_adapter(psgpu_proj_t *p, int32_t slot, int32_t rank, const void *a, const void *b, float scale)
{
    const size_t es = net_dtype_size(p->dtype);
    std::vector<char> ba, bb;
    if (rank) {
        pad_rows(ba, a, rank, p->d_in, p->rp, p->kp, es);
        pad_rows(bb, b, p->d_out, rank, p->np, p->rp, es);
    }
    PSGPU_HIP(hipDeviceSynchronize());              // calls that read the slot have ended; later ones see it whole
    const int32_t none = 0;
    PSGPU_HIP(hipMemcpy(p->rank + slot, &none, 4, hipMemcpyHostToDevice));      // (a copy that fails leaves the slot empty)
    if (!rank) return PSGPU_OK;
    PSGPU_HIP(hipMemcpy(p->a + slot * ba.size(), ba.data(), ba.size(), hipMemcpyHostToDevice));
    PSGPU_HIP(hipMemcpy(p->b + slot * bb.size(), bb.data(), bb.size(), hipMemcpyHostToDevice));
    PSGPU_HIP(hipMemcpy(p->scale + slot, &scale, 4, hipMemcpyHostToDevice));
    PSGPU_HIP(hipMemcpy(p->rank + slot, &rank, 4, hipMemcpyHostToDevice));
    return PSGPU_OK;
}

extern "C" int psgpu_proj_set_adapter(psgpu_proj_t *p, int32_t slot, int32_t rank, const void *a, const void *b, float scale)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(p, "psgpu_proj_set_adapter: NULL argument");
    PSGPU_REQUIRE(slot >= 0 && slot < p->max_adapters, "psgpu_proj_set_adapter: slot %d of %d", slot, p->max_adapters);
    PSGPU_REQUIRE(rank >= 0 && rank <= p->max_rank, "psgpu_proj_set_adapter: rank %d (0..%d)", rank, p->max_rank);
    PSGPU_REQUIRE(rank == 0 || (a && b), "psgpu_proj_set_adapter: NULL argument");
    PSGPU_REQUIRE(rank == 0 || std::isfinite(scale), "psgpu_proj_set_adapter: scale %g", (double)scale);
    PSGPU_REQUIRE(psgpu_get_device() == p->device, "psgpu_proj_set_adapter: the projection lives on device %d, the current one is %d", p->device, psgpu_get_device());
    try { return proj_store_adapter(p, slot, rank, a, b, scale); }
    catch (const std::bad_alloc &) { psgpu_set_error("psgpu_proj_set_adapter: out of memory"); return PSGPU_ENOMEM; }
}

extern "C" int32_t psgpu_proj_d_in(const psgpu_proj_t *p) { return p ? p->d_in : PSGPU_EINVAL; }
extern "C" int32_t psgpu_proj_d_out(const psgpu_proj_t *p) { return p ? p->d_out : PSGPU_EINVAL; }

// workspace: row_slot [total], then h [total][rp]
static inline size_t proj_slot_bytes(int32_t total) { return ((size_t)total * 4 + 255) / 256 * 256; }

extern "C" size_t psgpu_proj_work_bytes(const psgpu_proj_t *p, int32_t total_frames)
{
    if (!p || total_frames <= 0) return 0;
    return proj_slot_bytes(total_frames) + (size_t)total_frames * p->rp * 4;
}

template <typename T, typename Y>
static void proj_launch(const psgpu_proj_t *p, const void *x, int64_t xs, const int32_t *off, const int32_t *adapter, int32_t n_utt,
                        int32_t total, void *y, int64_t ys, char *work, hipStream_t st)
{
    int32_t *slots = nullptr;
    float *h = nullptr;
    if (off) {
        slots = (int32_t *)work;
        h = (float *)(work + proj_slot_bytes(total));
        proj_shrink_kernel<T><<<(uint32_t)total, 64, 0, st>>>((const T *)x, xs, p->d_in, p->kp, (const T *)p->a, p->rp, p->rank, p->scale,
                                                              p->max_adapters, off, adapter, n_utt, slots, h);
    }
    const dim3 grid((uint32_t)((p->d_out + kTile - 1) / kTile), (uint32_t)((total + kTile - 1) / kTile));
    proj_tile_kernel<T, Y><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, p->kp, (const T *)p->w, p->bias, p->d_out, (const T *)p->b,
                                                 p->np, p->rp, p->rank, slots, h, (Y *)y, ys);
}

extern "C" int psgpu_proj_run_dev(psgpu_proj_t *p, const void *x_dev, int64_t x_stride, const int32_t *utt_off_dev,
                                  const int32_t *adapter_dev, int32_t n_utt, int32_t total_frames, void *y_dev, int64_t y_stride,
                                  int32_t y_dtype, void *work_dev, size_t work_bytes, void *stream)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(p, "psgpu_proj_run_dev: NULL argument");
    PSGPU_REQUIRE(total_frames >= 0 && total_frames <= 65535 * kTile, "psgpu_proj_run_dev: %d frames", total_frames);
    PSGPU_REQUIRE(x_stride >= p->d_in && y_stride >= p->d_out, "psgpu_proj_run_dev: a row stride is below the row's %d inputs or %d outputs", p->d_in, p->d_out);
    PSGPU_REQUIRE(y_dtype == p->dtype || y_dtype == PSGPU_DT_F32, "psgpu_proj_run_dev: y_dtype %d (the projection's own, %d, or 32 bits)", y_dtype, p->dtype);
    PSGPU_REQUIRE(utt_off_dev || !adapter_dev, "psgpu_proj_run_dev: adapters without utterance offsets");
    PSGPU_REQUIRE(!utt_off_dev || n_utt >= 0, "psgpu_proj_run_dev: %d utterances", n_utt);
    if (total_frames == 0) return PSGPU_OK;
    PSGPU_REQUIRE(x_dev && y_dev, "psgpu_proj_run_dev: NULL device buffer");
    const size_t nx = net_span(total_frames, x_stride, p->d_in, net_dtype_size(p->dtype)), ny = net_span(total_frames, y_stride, p->d_out, net_dtype_size(y_dtype));
    const size_t need = utt_off_dev ? psgpu_proj_work_bytes(p, total_frames) : 0;
    PSGPU_REQUIRE(net_disjoint(x_dev, nx, y_dev, ny), "psgpu_proj_run_dev: the output overlaps the input");
    PSGPU_REQUIRE(work_bytes >= need && (work_dev || !need), "psgpu_proj_run_dev: %zu bytes of workspace, psgpu_proj_work_bytes asks for %zu", work_bytes, need);
    PSGPU_REQUIRE(((uintptr_t)work_dev & 15) == 0, "psgpu_proj_run_dev: the workspace is not aligned to 16 bytes");
    PSGPU_REQUIRE(!need || (net_disjoint(x_dev, nx, work_dev, need) && net_disjoint(y_dev, ny, work_dev, need)), "psgpu_proj_run_dev: the workspace overlaps the input or the output");
    const int rc = psgpu_check_device();
    if (rc != PSGPU_OK) return rc;
    PSGPU_REQUIRE(psgpu_get_device() == p->device, "psgpu_proj_run_dev: the projection lives on device %d, the current one is %d", p->device, psgpu_get_device());
    const hipStream_t st = (hipStream_t)stream;
    char *work = (char *)work_dev;
#define RUN(T, Y) proj_launch<T, Y>(p, x_dev, x_stride, utt_off_dev, adapter_dev, n_utt, total_frames, y_dev, y_stride, work, st)
    if (p->dtype == PSGPU_DT_F32) RUN(float, float);
    else if (p->dtype == PSGPU_DT_F16) { if (y_dtype == PSGPU_DT_F32) RUN(psg_half, float); else RUN(psg_half, psg_half); }
    else { if (y_dtype == PSGPU_DT_F32) RUN(psg_bf16, float); else RUN(psg_bf16, psg_bf16); }
#undef RUN
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
