// gnr_quant.hip -- 8-bit rows on gfx950: quantise rows, write feature maps into the slots of a cache, read them back.
//
// Mathematics: gnr_int8.h.  All three kernels are bound by memory: a value is read once (4 or 2 bytes) and written once (1 byte),
// or the other way round, with some ten operations in between.  What they are built around is the change of layout: maps are
// channels first (a channel's pixels contiguous), rows are pixels first (a pixel's channels contiguous), so a workgroup owns a
// tile of pixels whose 128 bytes per channel are whole lines, and the bytes change sides in LDS.
#include "gnr_int8.h"

namespace gnr {

// ---------------------------------------------------------------------------------------------
// channels-first maps [B][C][P] -> rows.  8 lanes x 16 bytes cover the tile's pixels of one channel (128 bytes: a whole line), a
// thread keeps R quads of channels in registers between the row maximum and the quantisation, so x is read once up to 2048
// channels (1024 threads, R = 4); wider rows are read twice.
// ---------------------------------------------------------------------------------------------
template <typename T, int R>
__global__ __launch_bounds__(1024) void quant_maps_kernel(const GnrRowsProblem p, unsigned tiles) {
    constexpr int V = Vec<T>::N, TP = 8 * V;
    extern __shared__ unsigned smem[];
    const int NT = (int)blockDim.x, G = NT >> 3, tid = (int)threadIdx.x, l = tid & 7, g = tid >> 3;
    const long b = blockIdx.x / tiles, p0 = (long)(blockIdx.x % tiles) * TP;
    long slot = b;
    if (p.slots) {
        const SlotRef ref = slot_of(p.slots, p.n_slots, b);
        if (ref.state) return;                              // the whole workgroup
        slot = ref.slot;
        // the same slot again later in the list: the LAST map stays, whichever workgroup runs first
        int again = 0;
        for (long j = b + 1 + tid; j < p.batch; j += NT) again |= p.slots[j] == slot;
        if (__syncthreads_or(again)) return;
    }
    unsigned* tile = smem;                                  // [TP][G + 4]: one quad of channels of one pixel a word
    unsigned* amax = smem + TP * (G + 4);                   // [NT / 64][TP]
    const int C = p.channels, ld = G + 4;
    const T* xb = (const T*)p.x + b * p.x_batch + p0 + l * V;
    const long left = p.n_pix - p0 - l * V;
    const int nv = left >= V ? V : (left > 0 ? (int)left : 0);
    const int step = 4 * G * R, n_chunk = (C + step - 1) / step;

    Vec<T> x[R][4];
    auto load = [&](int c0) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = c0 + 4 * (r * G + g) + e;
                x[r][e] = load_part(xb + (long)(c < C ? c : 0) * p.x_stride, c < C ? nv : 0);
            }
    };
    unsigned a[V] = {};
    for (int k = 0; k < n_chunk; ++k) {
        load(k * step);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const unsigned u = abs_bits((float)x[r][e].v[v]);
                    a[v] = u > a[v] ? u : a[v];
                }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int m = 8; m < 64; m <<= 1) {
            const unsigned u = (unsigned)__shfl_xor((int)a[v], m);
            a[v] = u > a[v] ? u : a[v];
        }
        if ((tid & 63) < 8) amax[(tid >> 6) * TP + l * V + v] = a[v];
    }
    __syncthreads();
    float per[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        unsigned m = 0;
        for (int w = 0; w < NT >> 6; ++w) {
            const unsigned u = amax[w * TP + l * V + v];
            m = u > m ? u : m;
        }
        float s;
        row_scale(m, s, per[v]);
        if (g == 0 && v < nv) p.scale[slot * p.scale_batch + p0 + l * V + v] = s;
    }
    int8_t* qb = p.q + slot * p.q_batch + p0 * p.q_pitch;
    for (int k = 0; k < n_chunk; ++k) {
        if (n_chunk > 1) load(k * step);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                tile[(l * V + v) * ld + g] =
                    pack4(row_step((float)x[r][0].v[v], per[v]), row_step((float)x[r][1].v[v], per[v]),
                          row_step((float)x[r][2].v[v], per[v]), row_step((float)x[r][3].v[v], per[v]));
            __syncthreads();
            const int cr = k * step + 4 * r * G, per_row = G >> 2;          // 16-byte pieces of a row in this pass
            for (int i = tid; i < TP * per_row; i += NT) {
                const int row = i / per_row, c = cr + 16 * (i % per_row);
                if (p0 + row < p.n_pix && c < C) {
                    Vec<int8_t> o;
                    __builtin_memcpy(&o, tile + row * ld + 4 * (i % per_row), 16);
                    store_part(qb + (long)row * p.q_pitch + c, o, C - c);
                }
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------------------------
// rows [N][C] -> rows: L lanes share a row and keep J pieces of 16 bytes each; rows wider than L J V are read twice
// ---------------------------------------------------------------------------------------------
template <typename T, int L, int J>
__global__ __launch_bounds__(256) void quant_rows_kernel(const GnrRowsProblem p, long total) {
    constexpr int V = Vec<T>::N;
    const int lane = (int)threadIdx.x % L;
    const long n = (long)blockIdx.x * (256 / L) + (int)threadIdx.x / L;
    const bool ok = n < total;
    const long b = ok ? n / p.n_pix : 0, pix = ok ? n % p.n_pix : 0;
    const T* x = (const T*)p.x + b * p.x_batch + pix * p.x_stride;
    int8_t* q = p.q + b * p.q_batch + pix * p.q_pitch;
    const int C = p.channels, step = L * J * V, n_chunk = (C + step - 1) / step;
    Vec<T> r[J];
    auto load = [&](int c0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int c = c0 + (j * L + lane) * V;
            r[j] = load_part(x + (c < C ? c : 0), ok ? C - c : 0);
        }
    };
    unsigned a = 0;
    for (int k = 0; k < n_chunk; ++k) {
        load(k * step);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const unsigned u = abs_bits((float)r[j].v[v]);
                a = u > a ? u : a;
            }
    }
#pragma unroll
    for (int m = 1; m < L; m <<= 1) {
        const unsigned u = (unsigned)__shfl_xor((int)a, m);
        a = u > a ? u : a;
    }
    float s, per;
    row_scale(a, s, per);
    if (!ok) return;
    if (lane == 0) p.scale[b * p.scale_batch + pix] = s;
    for (int k = 0; k < n_chunk; ++k) {
        if (n_chunk > 1) load(k * step);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int c = k * step + (j * L + lane) * V;
            if (c >= C) continue;
            unsigned o[V / 4];
#pragma unroll
            for (int w = 0; w < V / 4; ++w)
                o[w] = pack4(row_step((float)r[j].v[4 * w], per), row_step((float)r[j].v[4 * w + 1], per),
                             row_step((float)r[j].v[4 * w + 2], per), row_step((float)r[j].v[4 * w + 3], per));
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
// cached rows -> channels-first maps [B][C][P]: 128 channels of a tile of pixels pass through LDS at a time
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void read_maps_kernel(const GnrRowsProblem p, unsigned tiles) {
    constexpr int V = Vec<T>::N, TP = 8 * V, G = 32, LD = G + 4, PIECES = TP * 8 / 256;
    __shared__ unsigned tile[TP * LD];
    const int tid = (int)threadIdx.x, l = tid & 7, g = tid >> 3;
    const long b = blockIdx.x / tiles, p0 = (long)(blockIdx.x % tiles) * TP;
    const SlotRef ref = slot_of(p.slots, p.n_slots, b);
    const int C = p.channels;
    const int8_t* qb = p.q + ref.slot * p.q_batch;
    const long left = p.n_pix - p0 - l * V;
    const int nv = left >= V ? V : (left > 0 ? (int)left : 0);
    float s[V];
#pragma unroll
    for (int v = 0; v < V; ++v)
        s[v] = ref.state ? (ref.state == 1 ? 0.0f : __uint_as_float(0x7fc00000u))
                         : (v < nv ? p.scale[ref.slot * p.scale_batch + p0 + l * V + v] : 0.0f);
    T* yb = (T*)p.x + b * p.x_batch + p0 + l * V;
    for (int c0 = 0; c0 < C; c0 += 4 * G) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int row = (tid + 256 * i) >> 3, piece = tid & 7, c = c0 + 16 * piece;
            Vec<int8_t> o = {};
            if (!ref.state && p0 + row < p.n_pix && c < C) {
                if (c + 16 <= C) {
                    o = load_vec(qb + (p0 + row) * p.q_pitch + c);
                } else {
                    for (int e = 0; e < 16; ++e)
                        if (c + e < C) o.v[e] = qb[(p0 + row) * p.q_pitch + c + e];
                }
            }
            __builtin_memcpy(tile + row * LD + 4 * piece, &o, 16);
        }
        __syncthreads();
        const int c = c0 + 4 * g;
        if (c < C && nv > 0) {
            Vec<T> y[4];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int w = (int)tile[(l * V + v) * LD + g];
                y[0].v[v] = row_value<T>((int8_t)w, s[v]);
                y[1].v[v] = row_value<T>((int8_t)(w >> 8), s[v]);
                y[2].v[v] = row_value<T>((int8_t)(w >> 16), s[v]);
                y[3].v[v] = row_value<T>(w >> 24, s[v]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < C) store_part(yb + (long)(c + e) * p.x_stride, y[e], nv);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
int check_rows(const GnrRowsProblem* p, const char* what) {
    if (!p) return fail("%s: problem is NULL", what);
    if (p->struct_size != sizeof(GnrRowsProblem))
        return fail("%s: GnrRowsProblem.struct_size is %u but this libgnr.so (ABI %d) has sizeof = %zu: the caller was built "
                    "against a different include/gnr.h (or did not set struct_size)", what, p->struct_size, GNR_ABI_VERSION,
                    sizeof(GnrRowsProblem));
    if (p->dtype != GNR_F32 && p->dtype != GNR_BF16 && p->dtype != GNR_F16) return fail("%s: unknown dtype %d", what, p->dtype);
    if (p->batch < 0 || p->n_pix < 0) return fail("%s: batch and n_pix must be >= 0", what);
    if (p->channels < 1) return fail("%s: channels must be >= 1 (got %d)", what, p->channels);
    if (p->batch == 0 || p->n_pix == 0) return 0;
    if (p->n_pix > (1LL << 31) / p->batch) return fail("%s: %d x %lld rows exceed 2^31", what, p->batch, (long long)p->n_pix);
    if (!p->x || !p->q || !p->scale) return fail("%s: NULL pointer", what);
    if (p->x_batch < 0 || p->x_stride < 0 || p->q_batch < 0 || p->scale_batch < 0) return fail("%s: negative stride", what);
    if (p->q_pitch < p->channels) return fail("%s: q_pitch (%lld) < channels (%d)", what, (long long)p->q_pitch, p->channels);
    if (p->slots && p->n_slots < 1) return fail("%s: slots are given but n_slots is %lld", what, (long long)p->n_slots);
    return 0;
}

template <typename T> static void quant_maps(const GnrRowsProblem& p, hipStream_t st) {
    constexpr int TP = 8 * Vec<T>::N;
    const unsigned tiles = (unsigned)((p.n_pix + TP - 1) / TP);
    const int quads = (p.channels + 3) / 4;
    int nt = 64;
    while (nt < 1024 && quads > nt / 8 * 4) nt *= 2;         // the fewest threads that keep the row in 4 quads each
    const int G = nt / 8, R = quads >= 4 * G ? 4 : (quads + G - 1) / G;
    const size_t lds = sizeof(unsigned) * ((size_t)TP * (G + 4) + (size_t)nt / 64 * TP);
    const dim3 grid(tiles * (unsigned)p.batch), block((unsigned)nt);
    switch (R) {
        case 1: hipLaunchKernelGGL((quant_maps_kernel<T, 1>), grid, block, lds, st, p, tiles); break;
        case 2: hipLaunchKernelGGL((quant_maps_kernel<T, 2>), grid, block, lds, st, p, tiles); break;
        case 3: hipLaunchKernelGGL((quant_maps_kernel<T, 3>), grid, block, lds, st, p, tiles); break;
        default: hipLaunchKernelGGL((quant_maps_kernel<T, 4>), grid, block, lds, st, p, tiles); break;
    }
}

template <typename T> static void quant_rows(const GnrRowsProblem& p, hipStream_t st) {
    constexpr int V = Vec<T>::N;
    const long total = (long)p.batch * p.n_pix;
    const int C = p.channels;
#define GNR_ROWS(L, J) hipLaunchKernelGGL((quant_rows_kernel<T, L, J>), dim3((unsigned)((total + 256 / L - 1) / (256 / L))), dim3(256), 0, st, p, total)
    if (C <= 16 * V) GNR_ROWS(16, 1);
    else if (C <= 32 * V) GNR_ROWS(16, 2);
    else if (C <= 64 * V) GNR_ROWS(16, 4);
    else if (C <= 128 * V) GNR_ROWS(64, 2);
    else if (C <= 256 * V) GNR_ROWS(64, 4);
    else GNR_ROWS(64, 8);
#undef GNR_ROWS
}

int launch_quantize(const GnrRowsProblem& p, hipStream_t st) {
    if (p.channels_first) {
        if (p.dtype == GNR_F32) quant_maps<float>(p, st);
        else if (p.dtype == GNR_BF16) quant_maps<__bf16>(p, st);
        else quant_maps<_Float16>(p, st);
    } else {
        if (p.dtype == GNR_F32) quant_rows<float>(p, st);
        else if (p.dtype == GNR_BF16) quant_rows<__bf16>(p, st);
        else quant_rows<_Float16>(p, st);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("gnr_quantize_rows: launch failed: %s", hipGetErrorString(e));
}

template <typename T> static void read_maps(const GnrRowsProblem& p, hipStream_t st) {
    constexpr int TP = 8 * Vec<T>::N;
    const unsigned tiles = (unsigned)((p.n_pix + TP - 1) / TP);
    hipLaunchKernelGGL(read_maps_kernel<T>, dim3(tiles * (unsigned)p.batch), dim3(256), 0, st, p, tiles);
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
    if (p->dtype == GNR_F32) read_maps<float>(*p, st);
    else if (p->dtype == GNR_BF16) read_maps<__bf16>(*p, st);
    else read_maps<_Float16>(*p, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("gnr_read_rows: launch failed: %s", hipGetErrorString(e));
}

}  // extern "C"
