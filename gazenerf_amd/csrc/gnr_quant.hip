// gnr_quant.hip -- 8-bit rows on gfx950: quantise rows, write feature maps into the slots of a cache, read them back.
//
// Mathematics: gnr_int8.h.  All three kernels are bound by memory: a value is read once (4 or 2 bytes) and written once (1 byte),
// or the other way round, with some ten operations in between.  What they are built around is the change of layout: maps are
// channels first (a channel's pixels contiguous), rows are pixels first (a pixel's channels contiguous), so a workgroup owns a
// tile of pixels -- 32 of them: 128 bytes of a channel in fp32, a whole line, 64 in 16 bits; half of that while there are few tiles -- and the
// bytes change sides in LDS.
#include "gnr_int8.h"

namespace gnr {

__device__ __forceinline__ long tile_start(unsigned i, int tp, long n) {
    const long p = (long)i * tp;
    return p + tp <= n || n < tp ? p : n - tp;
}

// ---------------------------------------------------------------------------------------------
// channels-first maps [B][C][P] -> rows.  A tile is 32 pixels: LPX lanes x 16 bytes cover them in one channel (a line of 128 bytes in
// fp32), a thread keeps R quads of channels in registers between the row maximum and the quantisation, so x is read once up to
// 2048 channels (fp32; 4096 in 16 bits: 1024 threads, R = 4); wider rows are read twice.  Bound by memory: 64 maps of 258 x 4096 in
// fp32 (339 MB) take 87 us = 3.9 TB/s, 32 of them (170 MB) 52 us = 3.3, 8 maps of 1024 x 4096 in fp16 (101 MB, half lines) 34 us = 3.0; a large
// copy on this card: 4.7.
// ---------------------------------------------------------------------------------------------
template <typename T, int LPX, int R>
__global__ __launch_bounds__(1024) void quant_maps_kernel(const GnrRowsProblem p, unsigned tiles, int ld) {
    constexpr int V = Vec<T>::N, TP = LPX * V;
    extern __shared__ unsigned smem[];
    const int NT = (int)blockDim.x, G = NT / LPX, tid = (int)threadIdx.x, l = tid % LPX, g = tid / LPX;
    const unsigned at = xcd_block(gridDim.x);
    const long b = at / tiles, p0 = tile_start(at % tiles, TP, p.n_pix);
    unsigned* tile = smem;                                  // [TP][ld]: one quad of channels of one pixel a word
    unsigned* amax = smem + TP * ld;                        // [NT / 64][LPX][4]
    const int C = p.channels;
    // a tile that would reach over the map's end moves back to end with it, and so do the lanes of a map smaller than a tile: some
    // pixels are done twice, with the same results, and every access is a whole vector unless the map itself is smaller
    const bool whole = p.n_pix >= V;
    const long pl = whole ? (p0 + l * V < p.n_pix - V ? p0 + l * V : p.n_pix - V) : 0;
    const int nv = whole ? V : (int)p.n_pix;
    const T* xb = (const T*)p.x + b * p.x_batch + pl;
    const int step = 4 * G * R, n_chunk = (C + step - 1) / step;

    Raw16 x[R][4];
    auto load = [&](int c0) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = c0 + 4 * (r * G + g) + e;
                if (c < C) x[r][e] = load_raw(xb + (long)c * p.x_stride, nv);
                else x[r][e] = Raw16{};
            }
    };
    load(0);
    long slot = b;
    if (p.slots) {
        const SlotRef ref = slot_of(p.slots, p.n_slots, b);
        if (ref.state) return;                              // the whole workgroup; x is on its way meanwhile
        slot = ref.slot;
        // the same slot again later in the list: the LAST map stays, whichever workgroup runs first
        int again = 0;
        for (long j = b + 1 + tid; j < p.batch; j += NT) again |= p.slots[j] == slot;
        if (__syncthreads_or(again)) return;
    }
    unsigned a[4] = {};
    for (int k = 0; k < n_chunk; ++k) {
        if (k) load(k * step);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < 4; ++w) a[w] = max_bits<T>(a[w], x[r][e].w[w]);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
#pragma unroll
        for (int m = LPX; m < 64; m <<= 1) a[w] = max_bits<T>(a[w], (unsigned)__shfl_xor((int)a[w], m));
        if ((tid & 63) < LPX) amax[((tid >> 6) * LPX + l) * 4 + w] = a[w];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w)
        for (int i = 0; i < NT >> 6; ++i) a[w] = max_bits<T>(a[w], amax[(i * LPX + l) * 4 + w]);
    float per[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float s;
        row_scale(__float_as_uint(raw_value<T>(a, v)), s, per[v]);
        if (g == 0 && v < nv) p.scale[slot * p.scale_batch + pl + v] = s;
    }
    int8_t* qb = p.q + slot * p.q_batch;
    const int rows = p.n_pix - p0 < TP ? (int)(p.n_pix - p0) : TP;
    const int shift = (int)(pl - p0);                       // this lane's first row in the tile
    for (int k = 0; k < n_chunk; ++k) {
        if (n_chunk > 1) {
            load(k * step);
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v < nv && 4 * (k * G * R + r * G + g) < C)
                    tile[(shift + v) * ld + r * G + g] =
                        pack4(row_step(raw_value<T>(x[r][0].w, v), per[v]), row_step(raw_value<T>(x[r][1].w, v), per[v]),
                              row_step(raw_value<T>(x[r][2].w, v), per[v]), row_step(raw_value<T>(x[r][3].w, v), per[v]));
        __syncthreads();
        const int c0 = k * step, cols = C - c0 < step ? C - c0 : step, per_row = (cols + 15) >> 4;      // 16-byte pieces of a row
        for (int i = tid; i < rows * per_row; i += NT) {
            const int row = i / per_row, c = 16 * (i - row * per_row);
            Vec<int8_t> o;
            __builtin_memcpy(&o, __builtin_assume_aligned(tile + row * ld + (c >> 2), 16), 16);
            store_part(qb + (p0 + row) * p.q_pitch + c0 + c, o, cols - c);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// rows [N][C] -> rows: L lanes share a row and keep J pieces of 16 bytes each; rows wider than L J V are read twice
// ---------------------------------------------------------------------------------------------
template <typename T, int L, int J>
__global__ __launch_bounds__(256) void quant_rows_kernel(const GnrRowsProblem p, long first, long total) {
    constexpr int V = Vec<T>::N;
    const int lane = (int)threadIdx.x % L;
    const long n = first + (long)blockIdx.x * (256 / L) + (int)threadIdx.x / L;
    const bool ok = n < total;
    const unsigned b = ok ? (unsigned)n / (unsigned)p.n_pix : 0, pix = ok ? (unsigned)n - b * (unsigned)p.n_pix : 0;     // rows: at most 2^31
    const T* x = (const T*)p.x + b * p.x_batch + pix * p.x_stride;
    int8_t* q = p.q + b * p.q_batch + pix * p.q_pitch;
    const int C = p.channels, step = L * J * V, n_chunk = (C + step - 1) / step;
    Raw16 r[J];
    auto load = [&](int c0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int c = c0 + (j * L + lane) * V;
            if (ok && c < C) r[j] = load_raw(x + (C < V ? 0 : (c < C - V ? c : C - V)), C);
            else r[j] = Raw16{};
        }
    };
    unsigned a[4] = {};
    for (int k = 0; k < n_chunk; ++k) {
        load(k * step);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) a[w] = max_bits<T>(a[w], r[j].w[w]);
    }
    a[0] = max_bits<T>(max_bits<T>(a[0], a[1]), max_bits<T>(a[2], a[3]));
#pragma unroll
    for (int m = 1; m < L; m <<= 1) a[0] = max_bits<T>(a[0], (unsigned)__shfl_xor((int)a[0], m));
    if constexpr (sizeof(T) == 2) a[0] = max_bits<T>(a[0], a[0] >> 16);
    float s, per;
    row_scale(__float_as_uint(raw_value<T>(a, 0)), s, per);
    if (!ok) return;
    if (lane == 0) p.scale[b * p.scale_batch + pix] = s;
    for (int k = 0; k < n_chunk; ++k) {
        if (n_chunk > 1) load(k * step);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            int c = k * step + (j * L + lane) * V;
            if (c >= C) continue;
            if (C >= V && c > C - V) c = C - V;            // the last lane moves back: a few values twice, with the same results
            unsigned o[V / 4];
#pragma unroll
            for (int w = 0; w < V / 4; ++w)
                o[w] = pack4(row_step(raw_value<T>(r[j].w, 4 * w), per), row_step(raw_value<T>(r[j].w, 4 * w + 1), per),
                             row_step(raw_value<T>(r[j].w, 4 * w + 2), per), row_step(raw_value<T>(r[j].w, 4 * w + 3), per));
            if (c + V <= C) {
                __builtin_memcpy(q + c, o, V);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (c + v < C) q[c + v] = (int8_t)(o[v >> 2] >> 8 * (v & 3));
            }
        }
    }
}

// q * scale rounded to fp32, then to T: one answer for all three types.  The empty asm keeps the product in a register; without
// it the compiler folds product and conversion to fp16 into one instruction that rounds once.
template <typename T> __device__ __forceinline__ T row_value(int q, float s) {
    float v = (float)q * s;
    if (sizeof(T) == 2) asm("" : "+v"(v));
    return (T)v;
}

// ---------------------------------------------------------------------------------------------
// cached rows -> channels-first maps [B][C][P].  A tile's rows go to LDS whole and ONE barrier later the workgroup only stores: with a
// barrier per 128 channels every one of them waited for the stores before it.  The stores bypass the caches: four bytes leave for each
// that came, and through the caches they push out the rows that the neighbouring tile is about to read.  64 maps of 258 x 4096, fp32
// (339 MB), the same again and again, so that their rows (72 MB) stay in the caches: 112 us with stores through them, 51 us past them (in the
// tile -> XCD order of quant_maps_kernel 54).  Rows that come from memory: 73 us = 4.6 TB/s.
// ---------------------------------------------------------------------------------------------
template <typename T, int LPX>
__global__ __launch_bounds__(256) void read_maps_kernel(const GnrRowsProblem p, unsigned tiles, unsigned parts, int ld, int step) {
    constexpr int V = Vec<T>::N, TP = LPX * V, U = 4;
    extern __shared__ unsigned smem[];                      // [TP][ld]
    const int NT = (int)blockDim.x, G = NT / LPX, tid = (int)threadIdx.x, l = tid % LPX, g = tid / LPX;
    // maps whose channels are whole lines: past the caches, any order.  Others: neighbouring tiles share lines, which one L2 puts together
    // (64 maps of 258 x 4095, fp32: 93 us, past the caches 159)
    const bool lines = (p.x_stride * (long)sizeof(T)) % 128 == 0;
    const unsigned blk = lines ? blockIdx.x : xcd_block(gridDim.x), at = blk / parts;
    const long b = at / tiles, p0 = tile_start(at % tiles, TP, p.n_pix);
    const SlotRef ref = slot_of(p.slots, p.n_slots, b);
    const int C = p.channels, rows = p.n_pix - p0 < TP ? (int)(p.n_pix - p0) : TP;
    const int8_t* qb = p.q + ref.slot * p.q_batch + p0 * p.q_pitch;
    const bool whole = p.n_pix >= V;
    const long pl = whole ? (p0 + l * V < p.n_pix - V ? p0 + l * V : p.n_pix - V) : 0;
    const int nv = whole ? V : (int)p.n_pix, shift = (int)(pl - p0);
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
        s[v] = ref.state ? (ref.state == 1 ? 0.0f : __uint_as_float(0x7fc00000u)) : (v < nv ? p.scale[ref.slot * p.scale_batch + pl + v] : 0.0f);
    T* yb = (T*)p.x + b * p.x_batch + pl;
    for (int c0 = (int)(blk % parts) * step; c0 < C; c0 += (int)parts * step) {      // once, unless the rows of a tile exceed the LDS
        const int cols = C - c0 < step ? C - c0 : step, per_row = (cols + 15) >> 4, n = ref.state ? 0 : rows * per_row;
        if (c0 >= (int)parts * step) __syncthreads();
        for (int i0 = tid; i0 < n; i0 += NT * U) {
            Vec<int8_t> o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + NT * u, row = i / per_row, c = 16 * (i - row * per_row);
                if (i < n) o[u] = load_part(qb + row * p.q_pitch + c0 + c, cols - c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + NT * u, row = i / per_row, c = 16 * (i - row * per_row);
                if (i < n) __builtin_memcpy(__builtin_assume_aligned(smem + row * ld + (c >> 2), 16), &o[u], 16);
            }
        }
        __syncthreads();
        for (int q = g; 4 * q < cols; q += G) {
            Vec<T> y[4];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int w = v < nv && !ref.state ? (int)smem[(shift + v) * ld + q] : 0;
                y[0].v[v] = row_value<T>((int8_t)w, s[v]);
                y[1].v[v] = row_value<T>((int8_t)(w >> 8), s[v]);
                y[2].v[v] = row_value<T>((int8_t)(w >> 16), s[v]);
                y[3].v[v] = row_value<T>(w >> 24, s[v]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * q + e < cols) {
                    T* yp = yb + (long)(c0 + 4 * q + e) * p.x_stride;
                    if (lines) store_part<true>(yp, y[e], nv);
                    else store_part(yp, y[e], nv);
                }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
static int check_rows(const GnrRowsProblem* p, const char* what) {
    if (!p) return fail("%s: problem is NULL", what);
    if (p->struct_size != sizeof(GnrRowsProblem))
        return fail("%s: GnrRowsProblem.struct_size is %u but this libgnr.so (ABI %d) has sizeof = %zu: the caller was built "
                    "against a different include/gnr.h (or did not set struct_size)", what, p->struct_size, GNR_ABI_VERSION,
                    sizeof(GnrRowsProblem));
    if (p->dtype != GNR_F32 && p->dtype != GNR_BF16 && p->dtype != GNR_F16) return fail("%s: unknown dtype %d", what, p->dtype);
    if (p->batch < 0 || p->n_pix < 0) return fail("%s: batch and n_pix must be >= 0", what);
    if (p->channels < 1 || p->channels > 1 << 30) return fail("%s: channels must be 1 .. 2^30 (got %d)", what, p->channels);
    if (p->batch == 0 || p->n_pix == 0) return 0;
    if (p->n_pix > (1LL << 31) / p->batch) return fail("%s: %d x %lld rows exceed 2^31", what, p->batch, (long long)p->n_pix);
    if (!p->x || !p->q || !p->scale) return fail("%s: NULL pointer", what);
    if (p->x_batch < 0 || p->x_stride < 0 || p->q_batch < 0 || p->scale_batch < 0) return fail("%s: negative stride", what);
    if (p->q_pitch < p->channels) return fail("%s: q_pitch (%lld) < channels (%d)", what, (long long)p->q_pitch, p->channels);
    if (p->slots && p->n_slots < 1) return fail("%s: slots are given but n_slots is %lld", what, (long long)p->n_slots);
    return 0;
}

template <typename T, int LPX> static int quant_maps_lpx(const GnrRowsProblem& p, int nt, hipStream_t st) {
    constexpr int TP = LPX * Vec<T>::N;
    const unsigned tiles = (unsigned)((p.n_pix + TP - 1) / TP);
    const int quads = (p.channels + 3) / 4, G = nt / LPX;
    const int R = quads >= 4 * G ? 4 : (quads + G - 1) / G;
    const int words = quads < G * R ? quads : G * R, ld = (words + 15) / 16 * 16 + 4;
    const size_t lds = sizeof(unsigned) * ((size_t)TP * ld + (size_t)nt / 64 * LPX * 4);
    if (check_grid("gnr_quantize_rows", (long)tiles * p.batch, nt)) return 1;
    const dim3 grid(tiles * (unsigned)p.batch), block((unsigned)nt);
#define GNR_MAPS(RR) case RR: hipLaunchKernelGGL((quant_maps_kernel<T, LPX, RR>), grid, block, lds, st, p, tiles, ld); break
    switch (R) { GNR_MAPS(1); GNR_MAPS(2); GNR_MAPS(3); GNR_MAPS(4); }
#undef GNR_MAPS
    return 0;
}
// 32 pixels a tile, 16 where they would leave CUs without one (one map of 258 x 4096 in fp32: 5.1 / 5.5 us, two of 690 x 900 in bf16: 6.6 / 7.5;
// five of 129 x 1369 in bf16 the other way round: 6.3 / 5.9).  Threads: the fewest that
// keep a row in 4 quads of channels each (64 such maps: 78 us with 256 threads, 84 with 512), twice that while there are few of them (one
// map: 6.8 / 5.5; five of 129 x 1369, bf16: 6.9 / 5.9).
template <typename T> static int quant_maps(const GnrRowsProblem& p, hipStream_t st) {
    constexpr int LPX = 32 / Vec<T>::N;
    const int quads = (p.channels + 3) / 4;
    const long tiles = (p.n_pix + 31) / 32 * p.batch;
    int nt = 64;
    while (nt < 1024 && quads > nt / LPX * 4) nt *= 2;
    while (nt < 512 && tiles * nt < 131072 && quads > nt / LPX) nt *= 2;
    if (tiles < (sizeof(T) == 4 ? 192 : 128) && nt > 64) return quant_maps_lpx<T, LPX / 2>(p, nt, st);
    return quant_maps_lpx<T, LPX>(p, nt, st);
}

template <typename T, int L, int J> static void quant_rows_lj(const GnrRowsProblem& p, hipStream_t st) {
    const long total = (long)p.batch * p.n_pix, most = (1L << 27) / L * 16;    // a launch's threads: 2^31
    for (long first = 0; first < total; first += most) {
        const long n = total - first < most ? total - first : most;
        hipLaunchKernelGGL((quant_rows_kernel<T, L, J>), dim3((unsigned)((n + 256 / L - 1) / (256 / L))), dim3(256), 0, st, p, first, total);
    }
}
template <typename T> static int quant_rows(const GnrRowsProblem& p, hipStream_t st) {
    constexpr int V = Vec<T>::N;
    const int C = p.channels;
#define GNR_ROWS(L, J) quant_rows_lj<T, L, J>(p, st)
    switch ((C + 16 * V - 1) / (16 * V)) {                     // 16 lanes a row while eight pieces a lane hold it
        case 1: GNR_ROWS(16, 1); break;
        case 2: GNR_ROWS(16, 2); break;
        case 3: GNR_ROWS(16, 3); break;
        case 4: GNR_ROWS(16, 4); break;
        case 5: GNR_ROWS(16, 5); break;
        case 6: GNR_ROWS(16, 6); break;
        case 7: case 8: GNR_ROWS(16, 8); break;
        default:
            if (C <= 256 * V) GNR_ROWS(64, 4);
            else GNR_ROWS(64, 8);
    }
#undef GNR_ROWS
    return 0;
}

int launch_quantize(const GnrRowsProblem& p, hipStream_t st) {
    int rc;
    if (p.channels_first) rc = p.dtype == GNR_F32 ? quant_maps<float>(p, st) : p.dtype == GNR_BF16 ? quant_maps<__bf16>(p, st) : quant_maps<_Float16>(p, st);
    else rc = p.dtype == GNR_F32 ? quant_rows<float>(p, st) : p.dtype == GNR_BF16 ? quant_rows<__bf16>(p, st) : quant_rows<_Float16>(p, st);
    if (rc) return 1;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("gnr_quantize_rows: launch failed: %s", hipGetErrorString(e));
}

template <typename T, int LPX> static int read_maps_lpx(const GnrRowsProblem& p, int want, hipStream_t st) {
    constexpr int TP = LPX * Vec<T>::N;
    const unsigned tiles = (unsigned)((p.n_pix + TP - 1) / TP);
    int step = ((p.channels + want - 1) / want + 63) / 64 * 64;
    step = step < 1920 ? step : 1920;
    const unsigned parts = (unsigned)(want > 1 ? (p.channels + step - 1) / step : 1);
    const int ld = step / 4 + 4;
    int nt = 64;                                               // a quad of channels a thread and turn: no more threads than quads
    while (nt < 256 && (step < p.channels ? step : p.channels) > nt / LPX * 4) nt *= 2;
    if (check_grid("gnr_read_rows", (long)tiles * p.batch * parts, nt)) return 1;
    hipLaunchKernelGGL((read_maps_kernel<T, LPX>), dim3(tiles * (unsigned)p.batch * parts), dim3((unsigned)nt), sizeof(unsigned) * TP * ld, st, p,
                       tiles, parts, ld, step);
    return 0;
}
// 32 pixels a tile; while there are few, up to eight workgroups share one's channels (258 x 4096 in fp32, one map: 3.6 / 6.1 us, four: 4.7 / 6.2,
// sixteen: 17.1 / 15.2; two of 690 x 900 in bf16: 4.2 / 9.9)
template <typename T> static int read_maps(const GnrRowsProblem& p, hipStream_t st) {
    return read_maps_lpx<T, 32 / (sizeof(T) == 4 ? 4 : 8)>(p, (p.n_pix + 31) / 32 * p.batch < 1024 ? 8 : 1, st);
}

}  // namespace gnr

using namespace gnr;

extern "C" {

int gnr_quantize_rows(const GnrRowsProblem* p, void* stream) {
    if (check_rows(p, "gnr_quantize_rows")) return 1;
    if (p->slots && !p->channels_first) return fail("gnr_quantize_rows: slots are for channels-first maps");
    if (p->batch == 0 || p->n_pix == 0) return 0;
    return launch_quantize(*p, (hipStream_t)stream);
}

int gnr_read_rows(const GnrRowsProblem* p, void* stream) {
    if (check_rows(p, "gnr_read_rows")) return 1;
    if (!p->channels_first) return fail("gnr_read_rows: reads into channels-first maps only");
    if (p->batch == 0 || p->n_pix == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == GNR_F32 ? read_maps<float>(*p, st) : p->dtype == GNR_BF16 ? read_maps<__bf16>(*p, st) : read_maps<_Float16>(*p, st)) return 1;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("gnr_read_rows: launch failed: %s", hipGetErrorString(e));
}

}  // extern "C"
