// psgpu_proj.hip -- a shared projection of packed rows with low-rank adapters of many utterances.
//
//   y[t, o] = bias[o] + sum_k W[o, k] x[t, k] + s_a sum_r B_a[o, r] h[t, r],   h[t, r] = sum_k A_a[r, k] x[t, k]
//
// a = the adapter of the utterance row t belongs to: the speaker's correction of a transform that all share (what -lda is for the
// features, reference src/feat/lda.c:139-159, and -mllr for the means of one decoder's speaker, src/ps_mllr.c).  Products of the inputs'
// type, sums in 32 bits, one rounding at the end.
//
// psgpu_proj_t keeps the weights and every loaded adapter on the device, laid out once in the order in which a wavefront's lanes hold
// the first operand of a matrix instruction (a "fragment": 16 rows x 64 bytes of the reduced axis, 16 bytes a lane, 1 KB in a piece):
//   W   [outs / 64][chunks][4][64 lanes][16 bytes]          a chunk: KC = 64 bytes of d_in
//   A   [slot][chunks][ranks / 16][64 lanes][16 bytes]
//   B   [slot][parts][outs / 64][ranks / KC][4][64 lanes][16 bytes]
// zeros in the padding.  The outputs are dealt to the rows of four fragments so that one store of a wavefront writes 64 neighbouring
// bytes of each of 16 frames (proj_out_of).
//
// The adapters' h is kept in 32 bits, for the half types as three bfloat16 parts of 8 bits each, cut, not rounded, so that their sum is h
// exactly.  They go through the matrix instructions as more pieces of the reduced axis, against B in bfloat16: float16's B is two
// parts (exact); the product of the smallest two, 2^-25 of the term, is left out.  In float16 itself h could overflow.  (Two parts
// were 2^-18 of h; an adapter's term of rank 32 in 32 bits was off by 2.5e-6 in the mean square, in float16 3.7e-6, and is by 1.2e-7 and
// 1.5e-7.  The third costs 22 of 1058 us for
// 384 k rows of 1024 to 1024 in bfloat16 with rank 32, the two more 18 of 660 us for 48 k rows of 1024 to 5126 in float16.)
// A value that is not finite is a third part alone: against B's second part, often 0, an infinity would be a NaN.
#include "psgpu_net_dev.h"
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <type_traits>

struct psgpu_proj_s {
    int device = 0;
    int32_t dtype = 0, d_in = 0, d_out = 0, max_adapters = 0, max_rank = 0;
    int32_t kp = 0, np = 0, rp = 0;                 // padded d_in, d_out, max_rank
    size_t a_slot = 0, b_slot = 0;                  // bytes of a slot
    char *w = nullptr;
    float *bias = nullptr;                          // [np], zeros where there is none
    char *a = nullptr, *b = nullptr;                // [max_adapters] slots
    int32_t *rank = nullptr;                        // [max_adapters], 0: nothing loaded
    float *scale = nullptr;
    char *raw = nullptr;                            // an adapter as it comes, before it is laid out
    // held by a load from before it waits for the device until its adapter is whole (`raw` is one for all slots), and by a run while it
    // queues its launches: those in front of a load have ended before it begins, those behind it find it done
    std::mutex busy;
};

constexpr int kProjNoRow = -2;                      // rows of no utterance: left as they are

template <typename T> struct proj_geo {
    static constexpr int E = 16 / sizeof(T);        // elements a lane, elements a chunk
    static constexpr int KC = 4 * E;
    static constexpr int parts = sizeof(T) == 4 ? 1 : 3;    // of h
    static constexpr int h_bytes = sizeof(T) == 4 ? 4 : 6;  // an h takes in all its parts
    typedef typename net_frag<T>::type frag;
};
template <typename T> struct proj_b_type { typedef psg_bf16 type; static constexpr int parts = 1; };     // what B is kept in
template <> struct proj_b_type<float> { typedef float type; static constexpr int parts = 1; };
template <> struct proj_b_type<psg_half> { typedef psg_bf16 type; static constexpr int parts = 2; };

// the output of 64 that row m of fragment f holds: a lane's four rows m = 4 q .. 4 q + 3 of a fragment (of two, for halves) are 16 bytes
template <typename T>
__device__ __forceinline__ int proj_out_of(int f, int m)
{
    return sizeof(T) == 4 ? f * 16 + m : (f >> 1) * 32 + (m >> 2) * 8 + (f & 1) * 4 + (m & 3);
}

// the two bfloat16 parts of a float16 (an infinity has a second part of 0)
__device__ __forceinline__ void proj_split(float v, psg_bf16 &hi, psg_bf16 &lo)
{
    hi = net_cast<psg_bf16>(v);
    const float rest = v - net_f32(hi);
    lo = net_cast<psg_bf16>(__builtin_isinf(net_f32(hi)) ? 0.0f : rest);
}

// the three bfloat16 parts of a float
__device__ __forceinline__ void proj_split3(float v, psg_bf16 &hi, psg_bf16 &mid, psg_bf16 &lo)
{
    const bool fin = __builtin_isfinite(v);
    const float a = fin ? __uint_as_float(__float_as_uint(v) & 0xffff0000u) : 0.0f, b = __uint_as_float(__float_as_uint(fin ? v - a : 0.0f) & 0xffff0000u);
    hi.bits = (uint16_t)(__float_as_uint(a) >> 16);
    mid.bits = (uint16_t)(__float_as_uint(b) >> 16);
    lo = net_cast<psg_bf16>((v - a) - b);
}

// ---- layouts, one 16-byte lane's share a work-item --------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256)
void proj_lay_w_kernel(const T *__restrict__ src, int32_t rows, int32_t cols, int32_t chunks, size_t n, T *__restrict__ dst)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int lane = i & 63, f = (i >> 6) & 3, c = (int)((i >> 8) % chunks);
    const int o = (int)((i >> 8) / chunks) * 64 + proj_out_of<T>(f, lane & 15), k = c * KC + (lane >> 4) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[i * E + e] = o < rows && k + e < cols ? src[(size_t)o * cols + k + e] : T{};
}

template <typename T>
__global__ __launch_bounds__(256)
void proj_lay_a_kernel(const T *__restrict__ src, int32_t rank, int32_t d_in, int32_t rank_frags, size_t n, T *__restrict__ dst)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int lane = i & 63, q = (int)((i >> 6) % rank_frags), c = (int)((i >> 6) / rank_frags);
    const int r = q * 16 + (lane & 15), k = c * KC + (lane >> 4) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[i * E + e] = r < rank && k + e < d_in ? src[(size_t)r * d_in + k + e] : T{};
}

template <typename T>
__global__ __launch_bounds__(256)
void proj_lay_b_kernel(const T *__restrict__ src, int32_t d_out, int32_t rank, int32_t rank_chunks, size_t n, typename proj_b_type<T>::type *__restrict__ dst)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int lane = i & 63, f = (i >> 6) & 3, c = (int)((i >> 8) % rank_chunks);
    const int o = (int)((i >> 8) / rank_chunks) * 64 + proj_out_of<T>(f, lane & 15), r = c * KC + (lane >> 4) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const T v = o < d_out && r + e < rank ? src[(size_t)o * rank + r + e] : T{};
        if constexpr (proj_b_type<T>::parts == 2) {
            psg_bf16 hi, lo;
            proj_split(net_f32(v), hi, lo);
            dst[i * E + e] = hi;
            dst[(n + i) * E + e] = lo;
        } else dst[i * E + e] = v;
    }
}

// an adapter that is laid out becomes a slot's
__global__ void proj_load_kernel(int32_t *rank, float *scale, int32_t slot, int32_t r, float s) { rank[slot] = r; scale[slot] = s; }

// which adapter a row has; the lane's row is row0 + lane, kProjNoRow beyond `total`
__device__ __forceinline__ int proj_slot_of_rows(const int32_t *utt_off, const int32_t *adapter, int n_utt, const int32_t *rank, int max_adapters, int row0, int total)
{
    const int u = net_utt_of_rows(utt_off, n_utt, row0);
    if (u < 0 || row0 + (int)(threadIdx.x & 63) >= total) return kProjNoRow;
    const int slot = adapter ? adapter[u] : -1;
    return slot >= 0 && slot < max_adapters && rank[slot] > 0 ? slot : -1;
}

// ---- h --------------------------------------------------------------------------------------------------------------------------------
// ranks r .. r + 3 of frame t.  Those from `rank` on are 0, whatever A's padding made of an infinity: B's padding would make a NaN of it
template <typename T>
__device__ __forceinline__ void proj_store_h(net_f32x4 v, float scale, char *h, size_t t, int rp, int r, int rank)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (r + i >= rank) v[i] = 0.0f;
    if constexpr (sizeof(T) == 4) {
        net_f32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = v[i] * scale;
        *(net_f32x4 *)((float *)h + t * rp + r) = o;
    } else {
        net_pack<psg_bf16, 4> hi, mid, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) proj_split3(v[i] * scale, hi.v[i], mid.v[i], lo.v[i]);
        psg_bf16 *to = (psg_bf16 *)h + t * 3 * rp + r;
        *(uint64_t *)to = __builtin_bit_cast(uint64_t, hi);
        *(uint64_t *)(to + rp) = __builtin_bit_cast(uint64_t, mid);
        *(uint64_t *)(to + 2 * rp) = __builtin_bit_cast(uint64_t, lo);
    }
}

// Many rows: MR 16 a wavefront, all of an adapter's ranks at once, x once from memory (that is what bounds it: 384 k rows of 1024 in
// bfloat16, rank 32: 207 us, 4.1 TB/s with h), A from the caches (as many bytes as x with 32 rows and 32 ranks).
template <typename T, int RF, int MR>
__global__ __launch_bounds__(256)
void proj_shrink_kernel(const T *__restrict__ x, int64_t x_stride, int32_t total, int32_t d_in, int32_t chunks, const char *__restrict__ a, size_t a_slot,
                        int32_t rp, const int32_t *__restrict__ rank, const float *__restrict__ scale, int32_t max_adapters,
                        const int32_t *__restrict__ utt_off, const int32_t *__restrict__ adapter, int32_t n_utt,
                        int32_t *__restrict__ row_slot, char *__restrict__ h)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    typedef typename proj_geo<T>::frag frag;
    const int lane = threadIdx.x & 63;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (MR * 16);
    if (row0 >= total) return;
    const int slot = proj_slot_of_rows(utt_off, adapter, n_utt, rank, max_adapters, (int)row0, total);
    if (lane < MR * 16 && row0 + lane < total) row_slot[row0 + lane] = slot;
    if (!a) return;
    const int rank_frags = rp / 16;
    const T *xr[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) xr[m] = x + min(row0 + m * 16 + (lane & 15), (int64_t)total - 1) * x_stride;
    uint64_t todo = __ballot(lane < MR * 16 && slot >= 0);
    while (todo) {
        const int s = __shfl(slot, __builtin_ctzll(todo));
        const uint64_t mine = __ballot(slot == s);
        todo &= ~mine;
        const frag *as = (const frag *)(a + s * a_slot) + lane;
        net_f32x4 acc[MR][RF] = {};
#pragma unroll 2
        for (int c = 0; c < chunks; ++c) {
            const int k = c * KC + (lane >> 4) * E;
            frag f[MR];
#pragma unroll
            for (int m = 0; m < MR; ++m) f[m] = net_load_chunk(xr[m], k, d_in);
#pragma unroll
            for (int q = 0; q < RF; ++q) {
                const frag w = as[(c * rank_frags + min(q, rank_frags - 1)) * 64];
#pragma unroll
                for (int m = 0; m < MR; ++m) acc[m][q] = net_mfma(w, f[m], acc[m][q]);
            }
        }
        const float sc = scale[s];
        const int rank_of = rank[s];
#pragma unroll
        for (int m = 0; m < MR; ++m)
            if (mine >> (m * 16 + (lane & 15)) & 1)
#pragma unroll
                for (int q = 0; q < RF; ++q)
                    if (q < rank_frags) proj_store_h<T>(acc[m][q], sc, h, (size_t)row0 + m * 16 + (lane & 15), rp, q * 16 + (lane >> 4) * 4, rank_of);
    }
}

// Few rows: `tile` (1 .. 16) a workgroup, whose four wavefronts share the reduced axis.
template <typename T, int RF>
__global__ __launch_bounds__(256)
void proj_shrink_few_kernel(const T *__restrict__ x, int64_t x_stride, int32_t total, int32_t d_in, int32_t chunks, const char *__restrict__ a, size_t a_slot,
                            int32_t rp, const int32_t *__restrict__ rank, const float *__restrict__ scale, int32_t max_adapters,
                            const int32_t *__restrict__ utt_off, const int32_t *__restrict__ adapter, int32_t n_utt, int32_t tile,
                            int32_t *__restrict__ row_slot, char *__restrict__ h)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    typedef typename proj_geo<T>::frag frag;
    __shared__ net_f32x4 s_part[4][RF][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15;
    const int64_t row0 = (int64_t)blockIdx.x * tile;
    int slot = proj_slot_of_rows(utt_off, adapter, n_utt, rank, max_adapters, (int)row0, total);
    if (lane >= tile) slot = kProjNoRow;
    if (threadIdx.x < tile && row0 + lane < total) row_slot[row0 + lane] = slot;
    if (!a) return;
    const int rank_frags = rp / 16;
    const T *xr = x + min(row0 + col, (int64_t)total - 1) * x_stride;
    uint64_t todo = __ballot(slot >= 0);
    while (todo) {                                  // (the same in all four)
        const int s = __shfl(slot, __builtin_ctzll(todo));
        const uint64_t mine = __ballot(slot == s);
        todo &= ~mine;
        const frag *as = (const frag *)(a + s * a_slot) + lane;
        const int used = (rank[s] + 15) / 16;           // (the ranks behind them are zeros)
        net_f32x4 acc[RF] = {};
#pragma unroll 4
        for (int c = wave; c < chunks; c += 4) {
            frag f = {};
            if (mine >> col & 1) f = net_load_chunk(xr, c * KC + (lane >> 4) * E, d_in);
#pragma unroll
            for (int q = 0; q < RF; ++q)
                if (q < used) acc[q] = net_mfma(as[(c * rank_frags + q) * 64], f, acc[q]);
        }
#pragma unroll
        for (int q = 0; q < RF; ++q) s_part[wave][q][lane] = acc[q];
        __syncthreads();
        const float sc = scale[s];
        for (int q = wave; q < rank_frags; q += 4) {
            net_f32x4 v = s_part[0][q][lane];
            for (int w = 1; w < 4; ++w) v += s_part[w][q][lane];
            if (mine >> col & 1) proj_store_h<T>(v, sc, h, (size_t)row0 + col, rp, q * 16 + (lane >> 4) * 4, rank[s]);
        }
        __syncthreads();
    }
}

// ---- the product in tiles -----------------------------------------------------------------------------------------------------------
// acc of 16 frames (column lane & 15) += B_s h over the ranks of adapter s, for the frames whose slot it is; the others' h is zero here,
// and what they held is put back behind the products: an infinity in B_s makes a NaN of zero
template <typename T>
__device__ __forceinline__ void proj_expand(net_f32x4 (&acc)[4], bool mine, const char *bs, size_t b_part, int chunks, const char *ht, int rp)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    typedef typename proj_b_type<T>::type B;
    typedef typename net_frag<B>::type bfrag;
    const int lane = threadIdx.x & 63;
    net_f32x4 was[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) was[f] = acc[f];
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
        bfrag hp[proj_geo<T>::parts] = {};
        if (mine)
#pragma unroll
            for (int i = 0; i < proj_geo<T>::parts; ++i) hp[i] = *(const bfrag *)((const B *)ht + i * rp + c * KC + (lane >> 4) * E);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const bfrag w = ((const bfrag *)bs)[(c * 4 + f) * 64 + lane];
#pragma unroll
            for (int i = 0; i < proj_geo<T>::parts; ++i) acc[f] = net_mfma(w, hp[i], acc[f]);
            if constexpr (proj_b_type<T>::parts == 2) {
                const bfrag w2 = ((const bfrag *)(bs + b_part))[(c * 4 + f) * 64 + lane];
                acc[f] = net_mfma(w2, hp[0], acc[f]);
                acc[f] = net_mfma(w2, hp[1], acc[f]);
            }
        }
    }
    if (!mine)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f] = was[f];
}

// A tile of BM = WM MF 16 frames x BN = WN 64 outputs a workgroup; a wavefront MF 16 x 64.  A ring of three stages in LDS of 64 bytes
// of the reduced axis: while one is multiplied the next is there or nearly and the one behind it is on its way.  x lies in rows of 64
// bytes whose 16-byte pieces are exchanged by the row (piece p of row r at p ^ (r / 2 & 3)), so that 8 lanes meet no bank twice; W
// lies as in memory.  131072 rows of 1024 to 1024 in bfloat16: with 256 x 256 a workgroup (8 wavefronts, one a compute unit) 323 to 336 us,
// 820 to 850 TFLOP/s; 256 x 128 (two a compute unit, whose first loads and last stores pass under the other's products) was 7 % slower.  A stage
// is a barrier, 12 KB of reads and 32 matrix instructions a wavefront one behind the other, all wavefronts in step: the matrix units are
// 48 % busy, LDS by its bytes (12 KB read, 4 KB written at 128 a cycle) about as much, and neither is full.
// DMA: x goes to LDS without a register, 16 bytes a lane where it is aligned to them, else 4 bytes (rows of 429 floats),
// or 0: through registers.  A last stage that d_in does not fill goes through registers.
// Where all of a tile's frames have one adapter its h and B are more stages of the same ring (h's parts against B's); else every
// fragment of frames takes its adapters in turn behind them.
template <typename T, typename Y, int DMA, int WM, int WN, int MF>
__global__ __launch_bounds__(WM * WN * 64, 2)
void proj_tile_kernel(const T *__restrict__ x, int64_t x_stride, int32_t rows, int32_t d_in, int32_t chunks, const char *__restrict__ w,
                      const float *__restrict__ bias, int32_t d_out, const char *__restrict__ b, size_t b_slot, size_t b_part, int32_t rp,
                      const int32_t *__restrict__ rank, const int32_t *__restrict__ row_slot, const char *__restrict__ h,
                      Y *__restrict__ y, int64_t y_stride, int32_t tiles_m, int32_t tiles_n)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC, W = WM * WN, BM = WM * MF * 16, XB = BM * 64, WB = WN * 4096, ST = XB + WB;
    constexpr int XI = BM / 16 / W, WI = WN * 4 / W;        // 1 KB pieces of a stage a wavefront
    constexpr int XP = DMA == 4 ? 4 : 1, XL = XI * XP;      // loads of a piece of x, of all
    static_assert(XI * W * 16 == BM && WI * W == WN * 4, "a stage is shared evenly");
    typedef typename proj_geo<T>::frag frag;
    __shared__ __attribute__((aligned(1024))) char s_buf[3 * ST];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;

    // neighbouring tiles on one die (workgroups are dealt to the 8 dies in turn), 8 rows of tiles deep: they share x and W in its L2
    const int n_tiles = tiles_m * tiles_n, per = n_tiles >> 3, more = n_tiles & 7, die = blockIdx.x & 7;
    const int id = die * per + min(die, more) + (blockIdx.x >> 3);
    const int strip = id / (8 * tiles_n), deep = min(8, tiles_m - strip * 8), in = id - strip * 8 * tiles_n;
    const int64_t m0 = (int64_t)(strip * 8 + in % deep) * BM;
    const int g0 = (in / deep) * WN;                        // first group of 64 outputs

    // where this lane's pieces come from: x at a 32-bit offset from the tile's first row (DMA; the host sees to that), W one offset for all
    const int xk = ((lane & 3) ^ (lane >> 3 & 3)) * E;      // element of the stage (rows of a piece start at a multiple of 16)
    const char *xt = (const char *)(x + m0 * x_stride);
    const char *wt = w + (size_t)g0 * chunks * 4096;
    typedef typename std::conditional<DMA != 0, uint32_t, uint64_t>::type offs;
    offs xo[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        // a load of 4 bytes a lane brings 4 rows: lane = row, piece, word
        const int in = DMA == 4 ? (i & 3) * 4 + (lane >> 4) : lane >> 2;
        const int64_t r = min((int64_t)(wave * XI + i / XP) * 16 + in, (int64_t)rows - 1 - m0);
        xo[i] = (offs)(r * x_stride * (int64_t)sizeof(T) + (DMA == 4 ? ((lane >> 2 & 3) ^ (in >> 1 & 3)) * 16 + (lane & 3) * 4 : xk * (int)sizeof(T)));
    }
    const int full = d_in / KC;                             // stages that d_in fills
    const int stages = (d_in + KC - 1) / KC;
    int total = stages, slot0 = -1, rchunks = 0;            // with an adapter's stages

    frag xr[DMA ? 1 : XI];
    const uint32_t lds = net_lds_at(s_buf);
    auto fetch_full = [&](int st, int buf) {                // a stage that d_in fills
        const uint32_t to = lds + buf * ST;
        const char *ws = wt + (size_t)st * 4096, *from = xt + (size_t)st * 64;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int q = wave * WI + i;                    // [group][4 KB]
            net_load_lds<16>(ws + (size_t)(q >> 2) * chunks * 4096 + (q & 3) * 1024, lane * 16, to + XB + q * 1024);
        }
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            if constexpr (DMA == 16) net_load_lds<16>(from, xo[i], to + (wave * XI + i) * 1024);
            else if constexpr (DMA == 4) net_load_lds<4>(from, xo[i], to + wave * XI * 1024 + i * 256);
            else xr[i] = __builtin_bit_cast(frag, *(const net_pack<T, E> *)(from + xo[i]));
        }
    };
    auto fetch = [&](int st, int buf) {
        if (st < full) {
            fetch_full(st, buf);
            return;
        }
        const uint32_t to = lds + buf * ST;
        // the last stage of d_in, or an adapter's: B's parts 0, 0, 0, 1, 1 against h's 0, 1, 2, 0, 1
        const bool own = st < stages;
        const int part = own ? 0 : (st - stages) / rchunks, c = own ? st : (st - stages) - part * rchunks;
        const size_t group = own ? (size_t)chunks * 4096 : (size_t)rp * 64 * sizeof(typename proj_b_type<T>::type);
        const char *ws = (own ? wt : b + slot0 * b_slot + (part >= 3 ? b_part : 0) + (size_t)g0 * group) + (size_t)c * 4096;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int q = wave * WI + i;
            net_load_lds<16>(ws + (size_t)(q >> 2) * group + (q & 3) * 1024, lane * 16, to + XB + q * 1024);
        }
        const char *hs = h + (size_t)m0 * rp * proj_geo<T>::h_bytes + (part >= 3 ? part - 3 : part) * rp * 2 + (size_t)c * 64;
#pragma unroll 1
        for (int i = 0; i < XI; ++i) {
            const int64_t r = min((int64_t)(wave * XI + i) * 16 + (lane >> 2), (int64_t)rows - 1 - m0);
            if (own) *(frag *)(s_buf + buf * ST + (wave * XI + i) * 1024 + lane * 16) = net_load_chunk(x + (m0 + r) * x_stride, st * KC + xk, d_in);
            else net_load_lds<16>(hs, (uint32_t)((int)r * rp * proj_geo<T>::h_bytes + xk * (int)sizeof(T)), to + (wave * XI + i) * 1024);
        }
    };
    auto put = [&](int st, int buf) {                       // the pieces that came through registers
        if constexpr (!DMA) {
            if (st >= full) return;
#pragma unroll
            for (int i = 0; i < XI; ++i) *(frag *)(s_buf + buf * ST + (wave * XI + i) * 1024 + lane * 16) = xr[i];
        }
    };

    net_f32x4 acc[MF][4] = {};
    fetch(0, 0);
    put(0, 0);
    if (stages > 1) {
        fetch(1, 1);
        put(1, 1);
    }
    bool mixed = false;
    if (row_slot && b) {
        slot0 = __builtin_amdgcn_readfirstlane(row_slot[m0]);
        int same = 1;
        for (int r = threadIdx.x; r < BM; r += W * 64) same &= row_slot[min(m0 + r, (int64_t)rows - 1)] == slot0;
        mixed = !__syncthreads_and(same);
        if (!mixed && slot0 >= 0) {
            rchunks = (rank[slot0] + KC - 1) / KC;
            total += rchunks * (proj_geo<T>::parts + (proj_b_type<T>::parts == 2 ? 2 : 0));
        }
        if (stages == 1 && total > 1) fetch(1, 1);
    }
    int buf = 0;                                            // st % 3
    auto step = [&](int st, auto of, auto steady) {
        typedef decltype(of) F;
        // this wavefront's pieces of stage st lie in LDS (the loads of stage st + 1, issued behind them, may be on their way: XL + WI,
        // or XI + WI of an adapter's, or none but W's), its reads of stage st - 1 are done; behind the barrier: everybody's
        if (steady.value || st + 1 < full) net_wait_barrier<XL + WI>();
        else if (st + 1 < total) net_wait_barrier<XI + WI>();
        else net_wait_barrier<0>();
        const int ahead = buf == 0 ? 2 : buf - 1;           // (st + 2) % 3
        if (steady.value) fetch_full(st + 2, ahead);
        else if (st + 2 < total) fetch(st + 2, ahead);
        const char *from = s_buf + buf * ST;
        F wf[4], xf[MF];
#pragma unroll
        for (int f = 0; f < 4; ++f) wf[f] = *(const F *)(from + XB + wn * 4096 + f * 1024 + lane * 16);
#pragma unroll
        for (int m = 0; m < MF; ++m) {
            const int r = (wm * MF + m) * 16 + (lane & 15);
            xf[m] = *(const F *)(from + r * 64 + (((lane >> 4) ^ (r >> 1 & 3)) * 16));
        }
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
            for (int f = 0; f < 4; ++f) acc[m][f] = net_mfma(wf[f], xf[m], acc[m][f]);
        if (steady.value || st + 2 < stages) put(st + 2, ahead);
        buf = buf == 2 ? 0 : buf + 1;
    };
    typedef typename net_frag<typename proj_b_type<T>::type>::type bfrag;
    int st = 0;
    for (; st + 2 < full; ++st) step(st, frag(), std::true_type());
    if constexpr (std::is_same<frag, bfrag>::value)
        for (; st < total; ++st) step(st, frag(), std::false_type());
    else {
        for (; st < stages; ++st) step(st, frag(), std::false_type());
        for (; st < total; ++st) step(st, bfrag(), std::false_type());
    }

    int64_t t[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) t[m] = m0 + (wm * MF + m) * 16 + (lane & 15);
    int slot[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) slot[m] = t[m] >= rows ? kProjNoRow : row_slot ? row_slot[t[m]] : -1;
    if (mixed) {
        const char *bg = b + (size_t)(g0 + wn) * rp * 64 * sizeof(typename proj_b_type<T>::type);
#pragma unroll
        for (int m = 0; m < MF; ++m) {
            uint64_t todo = __ballot(slot[m] >= 0);
            while (todo) {
                const int s = __shfl(slot[m], __builtin_ctzll(todo));
                todo &= ~__ballot(slot[m] == s);
                proj_expand<T>(acc[m], slot[m] == s, bg + s * b_slot, b_part, (rank[s] + KC - 1) / KC, h + (size_t)t[m] * rp * proj_geo<T>::h_bytes, rp);
            }
        }
    }

    constexpr int SE = 16 / sizeof(Y);
    int o[4];                                               // this lane's outputs, four a fragment
    float bo[4][4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        o[f] = (g0 + wn) * 64 + proj_out_of<T>(f, (lane >> 4) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) bo[f][j] = bias[o[f] + j];
    }
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        if (slot[m] == kProjNoRow) continue;
        Y *yr = y + t[m] * y_stride;
#pragma unroll
        for (int f = 0; f < 4; f += SE / 4) {
            net_pack<Y, SE> v;
#pragma unroll
            for (int j = 0; j < SE; ++j) v.v[j] = net_cast<Y>(acc[m][f + (j >> 2)][j & 3] + bo[f + (j >> 2)][j & 3]);
            if (o[f] + SE <= d_out) *(net_pack<Y, SE> *)(yr + o[f]) = v;
            else
#pragma unroll
                for (int j = 0; j < SE; ++j)
                    if (o[f] + j < d_out) yr[o[f] + j] = v.v[j];
        }
    }
}

// ---- the product for few rows -----------------------------------------------------------------------------------------------------
// MF 16 frames x NF 16 outputs a workgroup, whose wavefronts share the reduced axis; no LDS on the way in (nothing is used twice), all of
// a wavefront's loads on their way at once.  The adapters' terms are taken by the vector units, a lane one frame and four outputs:
// neighbouring rows seldom share an adapter here.
// OWN_H (up to kProjOwnRows rows): every workgroup computes the frames' h for itself, in 32 bits, so that one launch does.
constexpr int kProjOwnRows = 4;
template <typename T, typename Y, int NW, int MF, int NF, bool OWN_H>
__global__ __launch_bounds__(NW * 64)
void proj_few_kernel(const T *__restrict__ x, int64_t x_stride, int32_t rows, int32_t d_in, int32_t chunks, const char *__restrict__ w,
                     const float *__restrict__ bias, int32_t d_out, const char *__restrict__ b, size_t b_slot, size_t b_part, int32_t rp,
                     const int32_t *__restrict__ rank, const int32_t *__restrict__ row_slot, const char *__restrict__ h,
                     Y *__restrict__ y, int64_t y_stride, const char *__restrict__ a, size_t a_slot, const float *__restrict__ scale,
                     int32_t max_adapters, const int32_t *__restrict__ utt_off, const int32_t *__restrict__ adapter, int32_t n_utt)
{
    constexpr int E = proj_geo<T>::E, KC = proj_geo<T>::KC;
    typedef typename proj_geo<T>::frag frag;
    typedef typename proj_b_type<T>::type B;
    static_assert(!OWN_H || MF == 1, "frames of one fragment");
    __shared__ net_f32x4 s_part[NW][MF * NF][64];
    __shared__ __attribute__((aligned(16))) float s_h[OWN_H ? kProjOwnRows * PSGPU_PROJ_MAX_RANK : 4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.y * MF * 16;
    const int n0 = blockIdx.x * NF, g = n0 >> 2, f0 = n0 & 3;
    const T *xp[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) xp[m] = x + min(m0 + m * 16 + (lane & 15), (int64_t)rows - 1) * x_stride;
    const frag *wp = (const frag *)(w + (size_t)g * chunks * 4096) + f0 * 64 + lane;
    int slots[MF], ranks[MF];                               // of this lane's frames, asked for in front of the products
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        const int64_t t = m0 + m * 16 + (lane & 15);
        if constexpr (OWN_H) slots[m] = __shfl(proj_slot_of_rows(utt_off, adapter, n_utt, rank, max_adapters, 0, rows), lane & 15);
        else slots[m] = t >= rows ? kProjNoRow : row_slot ? row_slot[t] : -1;
        ranks[m] = slots[m] >= 0 && b ? rank[slots[m]] : 0;
    }
    net_f32x4 acc[MF][NF] = {};
#pragma unroll 4
    for (int c = wave; c < chunks; c += NW) {
        frag xf[MF], wf[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) wf[f] = wp[(size_t)c * 256 + f * 64];
#pragma unroll
        for (int m = 0; m < MF; ++m) xf[m] = net_load_chunk(xp[m], c * KC + (lane >> 4) * E, d_in);
#pragma unroll
        for (int m = 0; m < MF; ++m)
#pragma unroll
            for (int f = 0; f < NF; ++f) acc[m][f] = net_mfma(wf[f], xf[m], acc[m][f]);
    }
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int f = 0; f < NF; ++f) s_part[wave][m * NF + f][lane] = acc[m][f];
    if constexpr (OWN_H) {
        for (int i = threadIdx.x; i < kProjOwnRows * rp; i += NW * 64) s_h[i] = 0.0f;
        uint64_t todo = __ballot(lane < kProjOwnRows && slots[0] >= 0 && b);    // (the same in all wavefronts)
        const int rank_frags = rp / 16;
        __shared__ net_f32x4 s_hp[NW][64];
        while (todo) {
            const int s = __shfl(slots[0], __builtin_ctzll(todo));
            todo &= ~__ballot(slots[0] == s);
            const frag *as = (const frag *)(a + s * a_slot) + lane;
            const float sc = scale[s];
            for (int q = 0; q < (rank[s] + 15) / 16; ++q) {
                net_f32x4 v = {};
#pragma unroll 4
                for (int c = wave; c < chunks; c += NW) {
                    frag xf = {};
                    if (slots[0] == s) xf = net_load_chunk(xp[0], c * KC + (lane >> 4) * E, d_in);
                    v = net_mfma(as[(c * rank_frags + q) * 64], xf, v);
                }
                s_hp[wave][lane] = v;
                __syncthreads();
                if (wave == 0 && slots[0] == s && (lane & 15) < kProjOwnRows) {
                    for (int i = 1; i < NW; ++i) v += s_hp[i][lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = q * 16 + (lane >> 4) * 4 + i;
                        s_h[(lane & 15) * rp + r] = r < rank[s] ? v[i] * sc : 0.0f;       // (as proj_store_h)
                    }
                }
                __syncthreads();
            }
        }
    }
    __syncthreads();
    for (int q = wave; q < MF * NF; q += NW) {
        const int m = q / NF, f = q % NF;
        const int64_t t = m0 + m * 16 + (lane & 15);
        int slot = slots[0], rank_of = ranks[0];
#pragma unroll
        for (int i = 1; i < MF; ++i)
            if (m == i) { slot = slots[i]; rank_of = ranks[i]; }
        const int o = g * 64 + proj_out_of<T>(f0 + f, (lane >> 4) * 4);
        net_f32x4 v = s_part[0][q][lane];
        for (int i = 1; i < NW; ++i) v += s_part[i][q][lane];
        if (slot >= 0 && b) {
            const int chunks_r = (rank_of + KC - 1) / KC;
            const B *bs = (const B *)(b + slot * b_slot) + (size_t)g * rp * 64 + (f0 + f) * 64 * E;
            const B *hr = (const B *)h + t * proj_geo<T>::parts * rp;
            for (int p = 0; p < chunks_r * 4; ++p) {        // E ranks at a time
                float hv[E];
                if constexpr (OWN_H) {
#pragma unroll
                    for (int e = 0; e < E; ++e) hv[e] = s_h[(lane & 15) * rp + p * E + e];
                } else {
                    net_pack<B, E> hp[proj_geo<T>::parts];
#pragma unroll
                    for (int i = 0; i < proj_geo<T>::parts; ++i) hp[i] = *(const net_pack<B, E> *)(hr + i * rp + p * E);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        hv[e] = net_f32(hp[0].v[e]);
                        if constexpr (proj_geo<T>::parts == 3) hv[e] = (hv[e] + net_f32(hp[1].v[e])) + net_f32(hp[2].v[e]);      // exact
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const B *bp = bs + ((p >> 2) * 256 + (p & 3) * 16 + (lane >> 4) * 4 + i) * E;
                    const net_pack<B, E> b1 = *(const net_pack<B, E> *)bp;
                    net_pack<B, E> b2 = {};
                    if constexpr (proj_b_type<T>::parts == 2) b2 = *(const net_pack<B, E> *)(bp + b_part / sizeof(B));
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float be = net_f32(b1.v[e]) + (proj_b_type<T>::parts == 2 ? net_f32(b2.v[e]) : 0.0f);
                        v[i] = __builtin_fmaf(hv[e], be, v[i]);
                    }
                }
            }
        }
        if (slot == kProjNoRow) continue;
        net_pack<Y, 4> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out.v[i] = net_cast<Y>(v[i] + bias[o + i]);
        Y *yr = y + t * y_stride + o;
        if (o + 4 <= d_out) *(net_pack<Y, 4> *)yr = out;
        else
            for (int i = 0; i < 4; ++i)
                if (o + i < d_out) yr[i] = out.v[i];
    }
}

static inline int32_t round_up(int32_t v, int32_t m) { return (v + m - 1) / m * m; }

// the object's device current in a scope
struct proj_on_device {
    int cur = -1;
    explicit proj_on_device(int device) { if (hipGetDevice(&cur) != hipSuccess || cur == device || hipSetDevice(device) != hipSuccess) cur = -1; }
    ~proj_on_device() { if (cur >= 0) (void)hipSetDevice(cur); }
};

extern "C" void psgpu_proj_free(psgpu_proj_t *p)
{
    if (!p) return;
    proj_on_device on(p->device);
    (void)hipFree(p->w); (void)hipFree(p->bias); (void)hipFree(p->a); (void)hipFree(p->b); (void)hipFree(p->rank); (void)hipFree(p->scale);
    (void)hipFree(p->raw);
    delete p;
}

template <typename T>
static void proj_lay_w(const psgpu_proj_t *p, const char *raw)
{
    const size_t n = (size_t)p->np * (p->kp / proj_geo<T>::KC) * 4;
    proj_lay_w_kernel<T><<<(uint32_t)((n + 255) / 256), 256>>>((const T *)raw, p->d_out, p->d_in, p->kp / proj_geo<T>::KC, n, (T *)p->w);
}

template <typename T>
static void proj_lay_ab(const psgpu_proj_t *p, int32_t slot, int32_t rank, const char *a, const char *b)
{
    const size_t na = p->a_slot / 16, nb = p->b_slot / 16 / proj_b_type<T>::parts;
    proj_lay_a_kernel<T><<<(uint32_t)((na + 255) / 256), 256>>>((const T *)a, rank, p->d_in, p->rp / 16, na, (T *)(p->a + slot * p->a_slot));
    proj_lay_b_kernel<T><<<(uint32_t)((nb + 255) / 256), 256>>>((const T *)b, p->d_out, rank, p->rp / proj_geo<T>::KC, nb,
                                                                (typename proj_b_type<T>::type *)(p->b + slot * p->b_slot));
}

// where an address lies: the device whose memory it is in, -1: the host
static int proj_device_of(const void *v)
{
    hipPointerAttribute_t at;
    if (hipPointerGetAttributes(&at, v) != hipSuccess) { (void)hipGetLastError(); return -1; }
    return at.type == hipMemoryTypeDevice ? at.device : -1;
}

// what the device of these weights still has to do may be to write them (the current device is waited for anyway)
static int proj_wait_for(const psgpu_proj_t *p, const void *v)
{
    const int device = v ? proj_device_of(v) : -1;
    if (device < 0 || device == p->device) return PSGPU_OK;
    proj_on_device on(device);
    PSGPU_HIP(hipDeviceSynchronize());
    return PSGPU_OK;
}

static int proj_fill(psgpu_proj_t *p, const void *weight, const float *bias)
{
    const size_t es = net_dtype_size(p->dtype), na = (size_t)p->max_adapters;
    const size_t raw_w = (size_t)p->d_out * p->d_in * es, raw_ab = na ? (size_t)p->max_rank * (p->d_in + p->d_out) * es + 32 : 0;
    PSGPU_HIP(hipDeviceSynchronize());              // (weights in device memory are whole)
    int rc = proj_wait_for(p, weight);
    if (rc == PSGPU_OK) rc = proj_wait_for(p, bias);
    if (rc != PSGPU_OK) return rc;
    PSGPU_HIP(hipMalloc((void **)&p->w, (size_t)p->np * p->kp * es));
    PSGPU_HIP(hipMalloc((void **)&p->bias, (size_t)p->np * 4));
    PSGPU_HIP(hipMalloc((void **)&p->raw, raw_w > raw_ab ? raw_w : raw_ab));
    PSGPU_HIP(hipMemcpy(p->raw, weight, raw_w, hipMemcpyDefault));
    PSGPU_HIP(hipMemset(p->bias, 0, (size_t)p->np * 4));
    if (bias) PSGPU_HIP(hipMemcpy(p->bias, bias, (size_t)p->d_out * 4, hipMemcpyDefault));
    if (p->dtype == PSGPU_DT_F32) proj_lay_w<float>(p, p->raw);
    else if (p->dtype == PSGPU_DT_F16) proj_lay_w<psg_half>(p, p->raw);
    else proj_lay_w<psg_bf16>(p, p->raw);
    PSGPU_HIP(hipGetLastError());
    PSGPU_HIP(hipDeviceSynchronize());
    if (!na) {
        PSGPU_HIP(hipFree(p->raw));
        p->raw = nullptr;
        return PSGPU_OK;
    }
    PSGPU_HIP(hipMalloc((void **)&p->a, na * p->a_slot));
    PSGPU_HIP(hipMalloc((void **)&p->b, na * p->b_slot));
    PSGPU_HIP(hipMalloc((void **)&p->rank, na * 4));
    PSGPU_HIP(hipMalloc((void **)&p->scale, na * 4));
    PSGPU_HIP(hipMemset(p->rank, 0, na * 4));
    PSGPU_HIP(hipMemset(p->scale, 0, na * 4));
    PSGPU_HIP(hipDeviceSynchronize());
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
    int device = -1, rc = net_check_device(&device);
    if (rc != PSGPU_OK) return rc;
    psgpu_proj_t *p = new (std::nothrow) psgpu_proj_t;
    if (!p) { psgpu_set_error("psgpu_proj_create: out of memory"); return PSGPU_ENOMEM; }
    p->device = device;
    p->dtype = dtype; p->d_in = d_in; p->d_out = d_out; p->max_adapters = max_adapters; p->max_rank = max_adapters ? max_rank : 0;
    const int32_t es = (int32_t)net_dtype_size(dtype);
    p->kp = round_up(d_in, 128 / es); p->np = round_up(d_out, 256); p->rp = round_up(p->max_rank, 64 / es);
    p->a_slot = (size_t)p->rp * p->kp * es;
    p->b_slot = (size_t)p->rp * p->np * es * (dtype == PSGPU_DT_F16 ? 2 : 1);
    rc = proj_fill(p, weight, bias);
    if (rc != PSGPU_OK) { psgpu_proj_free(p); return rc; }
    *out = p;
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
    const size_t es = net_dtype_size(p->dtype), raw_a = (size_t)rank * p->d_in * es, at_b = (raw_a + 15) / 16 * 16;
    std::lock_guard<std::mutex> lock(p->busy);
    PSGPU_HIP(hipDeviceSynchronize());              // calls that read the slot have ended; later ones see it whole
    proj_load_kernel<<<1, 1>>>(p->rank, p->scale, slot, 0, 0.0f);                   // (a copy that fails leaves the slot empty)
    PSGPU_HIP(hipGetLastError());
    if (rank) {
        int rc = proj_wait_for(p, a);
        if (rc == PSGPU_OK) rc = proj_wait_for(p, b);
        if (rc != PSGPU_OK) return rc;
        // in this device's memory, at an address that its type asks for
        auto here = [&](const void *v) { return proj_device_of(v) == p->device && ((uintptr_t)v & (es - 1)) == 0; };
        if (!here(a)) {
            PSGPU_HIP(hipMemcpy(p->raw, a, raw_a, hipMemcpyDefault));
            a = p->raw;
        }
        if (!here(b)) {
            PSGPU_HIP(hipMemcpy(p->raw + at_b, b, (size_t)rank * p->d_out * es, hipMemcpyDefault));
            b = p->raw + at_b;
        }
        if (p->dtype == PSGPU_DT_F32) proj_lay_ab<float>(p, slot, rank, (const char *)a, (const char *)b);
        else if (p->dtype == PSGPU_DT_F16) proj_lay_ab<psg_half>(p, slot, rank, (const char *)a, (const char *)b);
        else proj_lay_ab<psg_bf16>(p, slot, rank, (const char *)a, (const char *)b);
        PSGPU_HIP(hipGetLastError());
        proj_load_kernel<<<1, 1>>>(p->rank, p->scale, slot, rank, scale);
        PSGPU_HIP(hipGetLastError());
    }
    PSGPU_HIP(hipDeviceSynchronize());
    return PSGPU_OK;
}

extern "C" int32_t psgpu_proj_d_in(const psgpu_proj_t *p) { return p ? p->d_in : PSGPU_EINVAL; }
extern "C" int32_t psgpu_proj_d_out(const psgpu_proj_t *p) { return p ? p->d_out : PSGPU_EINVAL; }

// workspace: row_slot [total], then h [total][parts][rp]
static inline size_t proj_slot_bytes(int32_t total) { return ((size_t)total * 4 + 255) / 256 * 256; }

extern "C" size_t psgpu_proj_work_bytes(const psgpu_proj_t *p, int32_t total_frames)
{
    if (!p || total_frames <= 0) return 0;
    return proj_slot_bytes(total_frames) + (size_t)total_frames * p->rp * (p->dtype == PSGPU_DT_F32 ? proj_geo<float>::h_bytes : proj_geo<psg_half>::h_bytes);
}

template <typename T>
static void proj_shrink(const psgpu_proj_t *p, const void *x, int64_t xs, const int32_t *off, const int32_t *adapter, int32_t n_utt,
                        int32_t total, int32_t *slots, char *h, hipStream_t st)
{
    const int32_t chunks = p->kp / proj_geo<T>::KC;
    const char *a = adapter ? p->a : nullptr;
    // Few rows: 1, 4 or 16 a workgroup.  With the product of 64 outputs behind it, 1024 inputs, rank 16, us:
    // in utterances of 100 rows
    //   bfloat16   1024 rows 17.4 / 16.5 / 18.6   2048 rows 19.8 / 17.1 / 18.7   8192 rows 4: 25.4, 16: 22.5, many: 45.1
    //   float32    1024 rows 26.2 / 22.6 / 27.6   2048 rows 39.1 / 30.9 / 27.6   8192 rows 4: 44.3, 16: 45.7, many: 89.5
    // and where every row has another adapter, which a workgroup takes in turn, 1 / 4 / 16: 512 rows 18.0 / 24.4 / 53.6, float32 25.2 / 37.6 / 93.3; 2048
    // rows 21.7 / 25.4 / 52.7, 38.2 / 47.3 / 93.9.  Few against many rows: 16384 rows 34.4 / 51.4 and 63.9 / 105.3, 32768 rows 46.3 / 60.1 and 117
    // / 151.  32 against 64 rows a wavefront: 131072 rows of bfloat16 129 / 133 with ranks 16 and 32, 186 / 156 with rank 64; of float32 428 /
    // 428, 464 / 450, 513 / 501.
    const bool few = total <= 16384;
    const int32_t tile = total <= 2048 ? 1 : total <= 8192 ? 4 : 16;
    const bool wide = total >= 131072;
    const uint32_t grid = few ? (uint32_t)((total + tile - 1) / tile) : (uint32_t)(((int64_t)total + (wide ? 255 : 127)) / (wide ? 256 : 128));
#define SHRINK(RF) do { \
        if (few) proj_shrink_few_kernel<T, RF><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, a, p->a_slot, p->rp, p->rank, p->scale, p->max_adapters, off, adapter, n_utt, tile, slots, h); \
        else if (wide) proj_shrink_kernel<T, RF, 4><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, a, p->a_slot, p->rp, p->rank, p->scale, p->max_adapters, off, adapter, n_utt, slots, h); \
        else proj_shrink_kernel<T, RF, 2><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, a, p->a_slot, p->rp, p->rank, p->scale, p->max_adapters, off, adapter, n_utt, slots, h); \
    } while (0)
    if (p->rp <= 16) SHRINK(1);
    else if (p->rp <= 32) SHRINK(2);
    else if (p->rp <= 64) SHRINK(4);
    else SHRINK(8);
#undef SHRINK
}

template <typename T, typename Y>
static void proj_launch(const psgpu_proj_t *p, const void *x, int64_t xs, const int32_t *off, const int32_t *adapter, int32_t n_utt,
                        int32_t total, void *y, int64_t ys, char *work, hipStream_t st)
{
    const int32_t chunks = p->kp / proj_geo<T>::KC;
    int32_t *slots = nullptr;
    char *h = nullptr;
    const int64_t t128 = (((int64_t)total + 127) / 128) * ((p->d_out + 127) / 128), t256 = (((int64_t)total + 255) / 256) * ((p->d_out + 255) / 256);
    const bool own_h = off && total <= kProjOwnRows && t128 < 256;
    if (off && !own_h) {
        slots = (int32_t *)work;
        h = work + proj_slot_bytes(total);
        proj_shrink<T>(p, x, xs, off, adapter, n_utt, total, slots, h, st);
    }
    const char *b = adapter ? p->b : nullptr;
    const size_t b_part = p->b_slot / proj_b_type<T>::parts;
    const uintptr_t at = (uintptr_t)x | (uintptr_t)(xs * sizeof(T));
    // Tiles of 128 x 128 from 256 of them on (fewer leave compute units idle).  Few rows against tiles, 1024 to 1024, rank 16, us:
    //   bfloat16   512 rows 19.7 / 28.1   1024 rows 25.5 / 28.8   2048 rows 40.1 / 32.0   4000 rows 60.1 / 32.3   8000 rows 106 / 42
    //   float32    512 rows 29.8 / 86.5   1024 rows 51.2 / 92.8   2048 rows 82.7 / 99.3   4000 rows 130 / 97      8000 rows 239 / 162
    // (at the rule, 4096 rows, tiles are ahead already: in bfloat16 from 128 of them on).  Tiles of 256 x 256 from 512 of them on, 128 / 256 us in
    // bfloat16: 8192 rows 42.0 / 55.1   16384 rows 65.7 / 62.7   32768 rows 122 / 120   65536 rows 208 / 208; not for outputs that leave much of
    // them empty: 65536 rows to 1040 244 / 261, to 1100 244 / 265, to 2100 412 / 433, to 1280 267 / 268.
    const bool near_rows = xs < ((int64_t)1 << 30) / 256 / (int64_t)sizeof(T);      // (a tile's rows at 32-bit offsets)
    const int dma = !near_rows ? 0 : (at & 15) == 0 ? 16 : (at & 3) == 0 ? 4 : 0;
#define TILE(D, WM, WN, MF) do { \
        const int32_t tm = (int32_t)(((int64_t)total + WM * MF * 16 - 1) / (WM * MF * 16)), tn = (p->d_out + WN * 64 - 1) / (WN * 64); \
        proj_tile_kernel<T, Y, D, WM, WN, MF><<<(uint32_t)tm * (uint32_t)tn, WM * WN * 64, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, p->w, p->bias, p->d_out, \
            b, p->b_slot, b_part, p->rp, p->rank, slots, h, (Y *)y, ys, tm, tn); \
    } while (0)
    if (t128 < 256) {
#define FEW_REST p->a, p->a_slot, p->scale, p->max_adapters, off, adapter, n_utt
        if (own_h) {
            const dim3 grid((uint32_t)((p->d_out + 63) / 64 * 4), 1);
            proj_few_kernel<T, Y, 4, 1, 1, true><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, p->w, p->bias, p->d_out, b, p->b_slot, b_part, p->rp, p->rank, slots, h, (Y *)y, ys, FEW_REST);
        } else if (total <= 16) {       // 16 / 64 outputs a workgroup, 16 rows: 16.5 / 17.4 us, float32 18.7 / 22.1; 64 rows: 19.8 / 19.2, 18.8 / 22.5
            const dim3 grid((uint32_t)((p->d_out + 63) / 64 * 4), 1);
            proj_few_kernel<T, Y, 4, 1, 1, false><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, p->w, p->bias, p->d_out, b, p->b_slot, b_part, p->rp, p->rank, slots, h, (Y *)y, ys, FEW_REST);
        } else if ((int64_t)((p->d_out + 63) / 64) * ((total + 31) / 32) < 512) {
            // 16 / 32 frames, 512 rows to 1024: 20.0 / 20.6 us; 1024 rows: 26.8 / 25.3; 2048 rows: 45.0 / 39.6
            const dim3 grid((uint32_t)((p->d_out + 63) / 64), (uint32_t)((total + 15) / 16));
            proj_few_kernel<T, Y, 4, 1, 4, false><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, p->w, p->bias, p->d_out, b, p->b_slot, b_part, p->rp, p->rank, slots, h, (Y *)y, ys, FEW_REST);
        } else {
            const dim3 grid((uint32_t)((p->d_out + 63) / 64), (uint32_t)((total + 31) / 32));
            proj_few_kernel<T, Y, 4, 2, 4, false><<<grid, 256, 0, st>>>((const T *)x, xs, total, p->d_in, chunks, p->w, p->bias, p->d_out, b, p->b_slot, b_part, p->rp, p->rank, slots, h, (Y *)y, ys, FEW_REST);
        }
    } else if (sizeof(T) == 4 || t256 < 512 || round_up(p->d_out, 256) > p->d_out / 4 * 5) {       // (a quarter of the outputs' tiles in vain)
        if (dma == 16) TILE(16, 2, 2, 4); else if (dma == 4) TILE(4, 2, 2, 4); else TILE(0, 2, 2, 4);
    } else {
        if constexpr (sizeof(T) == 2) { if (dma == 16) TILE(16, 2, 4, 8); else if (dma == 4) TILE(4, 2, 4, 8); else TILE(0, 2, 4, 8); }
    }
#undef TILE
#undef FEW_REST
}

extern "C" int psgpu_proj_run_dev(psgpu_proj_t *p, const void *x_dev, int64_t x_stride, const int32_t *utt_off_dev,
                                  const int32_t *adapter_dev, int32_t n_utt, int32_t total_frames, void *y_dev, int64_t y_stride,
                                  int32_t y_dtype, void *work_dev, size_t work_bytes, void *stream)
{
    psgpu_clear_error();
    PSGPU_REQUIRE(p, "psgpu_proj_run_dev: NULL argument");
    PSGPU_REQUIRE(total_frames >= 0 && (int64_t)total_frames * ((p->d_out + 127) / 128) <= (int64_t)1 << 37, "psgpu_proj_run_dev: %d frames of %d outputs", total_frames, p->d_out);
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
    int device = -1;
    const int rc = net_check_device(&device);
    if (rc != PSGPU_OK) return rc;
    PSGPU_REQUIRE(device == p->device, "psgpu_proj_run_dev: the projection lives on device %d, the current one is %d", p->device, device);
    const hipStream_t st = (hipStream_t)stream;
    char *work = (char *)work_dev;
    std::lock_guard<std::mutex> lock(p->busy);
#define RUN(T, Y) proj_launch<T, Y>(p, x_dev, x_stride, utt_off_dev, adapter_dev, n_utt, total_frames, y_dev, y_stride, work, st)
    if (p->dtype == PSGPU_DT_F32) RUN(float, float);
    else if (p->dtype == PSGPU_DT_F16) { if (y_dtype == PSGPU_DT_F32) RUN(psg_half, float); else RUN(psg_half, psg_half); }
    else { if (y_dtype == PSGPU_DT_F32) RUN(psg_bf16, float); else RUN(psg_bf16, psg_bf16); }
#undef RUN
    PSGPU_HIP(hipGetLastError());
    return PSGPU_OK;
}
