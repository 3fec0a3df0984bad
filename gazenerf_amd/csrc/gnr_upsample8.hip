// gnr_upsample8.hip -- the 2-D upsampler (gnr_upsample.hip's network, inference) in 8 bits: its 1x1 convolutions are gnr_int8_linear.
//
//   block i:  a1 = lrelu(W1 net + b1);  a2 = lrelu(W2 a1 + b2)
//             u  = pixel_shuffle(a2 + repeat(net, 4), 2);  v = blur(u);  net = lrelu(Wf v + bf);  rgb += conv_rgb(i+1)(net)
//
// Everything between the input and the image is in rows (a pixel's channels contiguous): the products read and write rows, a row is
// what shares a scale, and the shuffle needs the four channels 4c .. 4c + 3 of a pixel together.  Activations between the products
// are kept in bf16: rounding them costs 2^-9 of each value, the 8-bit rows that every consumer but the residual makes of them half a
// step = 2^-8 of the row's LARGEST value; the bytes of the three convolutions halve.  The blur, the RGB branch and the
// epilogues are fp32.  The input's residual and RGB taps come from its 8-bit rows, too, so that an image is the same bit for bit
// whether its map came as fp32 or from the slots of a cache.
#include "gnr_int8.h"
#include "gnr_upsample.h"

namespace gnr {

// rows of values: 8-bit ones with their scales (through the slots of a cache if there is a list), or bf16
struct RowsView {
    const int8_t* q; long batch, pitch;           // bytes
    const float* scale; long scale_batch;
    const int64_t* slots; long n_slots;
    const __bf16* v;                              // != NULL: [B][P][C]
};
struct RowsAt {                                   // one batch entry
    const int8_t* q; const float* scale; const __bf16* v;
    float dead;                                   // not 1: the entry has no slot, every value is 0 * dead
};
__device__ __forceinline__ RowsAt rows_at(const RowsView& r, long b, long P, int C) {
    if (r.v) return RowsAt{nullptr, nullptr, r.v + b * P * C, 1.0f};
    const SlotRef s = slot_of(r.slots, r.n_slots, b);
    return RowsAt{r.q + s.slot * r.batch, r.scale + s.slot * r.scale_batch, nullptr,
                  s.state ? (s.state == 1 ? 0.0f : __uint_as_float(0x7fc00000u)) : 1.0f};
}
__device__ __forceinline__ float row_factor(const RowsAt& r, long pix) { return r.dead == 1.0f ? r.scale[pix] : r.dead; }

// ---------------------------------------------------------------------------------------------
// v = blur(pixel_shuffle(a2 + repeat(net, 4))) as 8-bit rows.  A group of C threads (one channel each) walks 4 low-resolution pixels of an
// image row; of a neighbour it needs the four values 4c .. 4c + 3 of a2 (8 bytes) and of the repeated residual, and keeps the vertically
// blurred columns of the last three pixels, so 3 neighbours are loaded per pixel instead of 9.  Clamping the neighbour's
// coordinates IS the blur's reflection: u row -1 reflects onto row 1 = (pixel 0, second sub-row), which is what the clamped
// neighbour above hands over.  The 16 output rows of a group meet in LDS, where eight lanes a row find its maximum and quantise it.
// ---------------------------------------------------------------------------------------------
constexpr int SB_RUN = 4, SB_THREADS = 320;

// the residual's values (4c .. 4c + 3) % C of a row, r0 = 4c % C: one load, and where C is no multiple of 4 a second one of the row's
// first values, shifted together (the four wrap around for one c in C / 4)
template <typename T4, bool WRAP, typename E> __device__ __forceinline__ T4 four_of(const E* row, int r0, int C) {
    if constexpr (!WRAP) {
        T4 t;
        __builtin_memcpy(&t, row + r0, sizeof(T4));
        return t;
    } else {
        const int at = r0 < C - 4 ? r0 : C - 4, d = 8 * (int)sizeof(E) * (r0 - at);
        T4 x, y;
        __builtin_memcpy(&x, row + at, sizeof(T4));
        __builtin_memcpy(&y, row, sizeof(T4));
        return d ? (T4)(x >> d | y << (8 * (int)sizeof(T4) - d)) : x;
    }
}

template <bool ROWS8, bool WRAP>
__global__ __launch_bounds__(SB_THREADS, 4) void shuffle_blur_rows_kernel(const __bf16* __restrict__ a2, const RowsView res, int C, int lg, int groups,
                                                                         int8_t* __restrict__ q, long q_pitch, float* __restrict__ scale) {
    extern __shared__ float vals[];                // [groups * SB_RUN * 4][C | 1]
    const int tid = (int)threadIdx.x, ld = C | 1, S = 1 << lg;                 // S x S low-resolution pixels, S a power of two
    const int P = S * S, runs = P / SB_RUN, run0 = (int)blockIdx.x * groups;
    const long b = blockIdx.y;
    const RowsAt r = rows_at(res, b, P, C);
    const __bf16* ab = a2 + b * P * 4 * C;
    const int per = groups > 1 ? C : SB_THREADS, grp = groups > 1 ? tid / C : 0;
    if (grp < groups && run0 + grp < runs) {
        const int p0 = (run0 + grp) * SB_RUN, y = p0 >> lg, x0 = p0 & (S - 1);
        const int rows3[3] = {(y > 0 ? y - 1 : 0) * S, y * S, (y + 1 < S ? y + 1 : S - 1) * S};
        for (int c = groups > 1 ? tid - grp * C : tid; c < C; c += per) {
            const int r0 = 4 * c % C;
            struct Raw { unsigned long a, v; float f; };       // what one neighbour holds for channel c
            auto load = [&](int xx, Raw (&o)[3]) {
                xx = xx < 0 ? 0 : (xx < S ? xx : S - 1);
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const long pix = rows3[k] + xx;
                    __builtin_memcpy(&o[k].a, ab + (pix * C + c) * 4, 8);
                    if constexpr (ROWS8) {
                        o[k].v = four_of<unsigned, WRAP>(r.q + pix * res.pitch, r0, C);
                        o[k].f = row_factor(r, pix);
                    } else {
                        o[k].v = four_of<unsigned long, WRAP>(r.v + pix * C, r0, C);
                    }
                }
            };
            auto u4 = [&](const Raw& o, float (&u)[4]) {       // the 2 x 2 block of u
                typedef __bf16 b4 __attribute__((ext_vector_type(4)));
                const b4 av = __builtin_bit_cast(b4, o.a);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (ROWS8) u[k] = fmaf((float)(int8_t)(o.v >> 8 * k), o.f, (float)av[k]);
                    else u[k] = (float)av[k] + (float)__builtin_bit_cast(b4, o.v)[k];
                }
            };
            // a pixel's column pair, vertically blurred: vb[2 i + j] for output sub-row i
            auto column = [&](const Raw (&o)[3], float (&vb)[4]) {
                float up[4], mid[4], dn[4];
                u4(o[0], up);
                u4(o[1], mid);
                u4(o[2], dn);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    vb[j] = (0.25f * up[2 + j] + 0.5f * mid[j]) + 0.25f * mid[2 + j];
                    vb[2 + j] = (0.25f * mid[j] + 0.5f * mid[2 + j]) + 0.25f * dn[j];
                }
            };
            Raw now[3], next[3];
            float L[4], M[4], R[4];
            load(x0 - 1, now);
            load(x0, next);
            column(now, L);
            load(x0 + 1, now);
            column(next, M);
#pragma unroll 1                                               // unrolled, the loads of a whole run are in registers: half the waves
            for (int i = 0; i < SB_RUN; ++i) {
                if (i + 1 < SB_RUN) load(x0 + i + 2, next);    // under this one
                column(now, R);
#pragma unroll
                for (int s = 0; s < 2; ++s) {                  // output pixel (2y + s, 2x + j) -> LDS row 4 i + 2 s + j of the group
                    float* o = vals + (long)(grp * SB_RUN * 4 + 4 * i + 2 * s) * ld + c;
                    o[0] = (0.25f * L[2 * s + 1] + 0.5f * M[2 * s]) + 0.25f * M[2 * s + 1];
                    o[ld] = (0.25f * M[2 * s] + 0.5f * M[2 * s + 1]) + 0.25f * R[2 * s];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) { L[k] = M[k]; M[k] = R[k]; }
#pragma unroll
                for (int k = 0; k < 3; ++k) now[k] = next[k];
            }
        }
    }
    __syncthreads();
    for (int row = tid >> 3; row < groups * SB_RUN * 4; row += SB_THREADS / 8) {
        const int g = row / (SB_RUN * 4), k = row % (SB_RUN * 4), l = tid & 7;
        if (run0 + g >= runs) continue;                        // eight lanes share a row: they stay together
        const float* vr = vals + (long)row * ld;
        unsigned m = 0;
        for (int c = l; c < C; c += 8) m = max_bits<float>(m, __float_as_uint(vr[c]));
#pragma unroll
        for (int i = 1; i < 8; i <<= 1) m = max_bits<float>(m, (unsigned)__shfl_xor((int)m, i));
        float s, per1;
        row_scale(m, s, per1);
        const int p0 = (run0 + g) * SB_RUN + (k >> 2);
        const long out = b * 4 * P + ((2 * (p0 >> lg) + ((k >> 1) & 1)) << (lg + 1)) + 2 * (p0 & (S - 1)) + (k & 1);
        if (l == 0) scale[out] = s;
        int8_t* qr = q + out * q_pitch;
        for (int c = 4 * l; c < C; c += 32) {
            int t[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = row_step(c + e < C ? vr[c + e] : 0.0f, per1);
            const unsigned w = pack4(t[0], t[1], t[2], t[3]);  // behind C: zeros, inside the row's pitch
            __builtin_memcpy(qr + c, &w, 4);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// the 3-channel RGB branch on rows: eight lanes a pixel, 16 bf16 or 16 bytes a lane and turn, summed over the lanes in a fixed tree
// ---------------------------------------------------------------------------------------------
template <bool ROWS8>
__global__ __launch_bounds__(256) void rgb_rows_kernel(const RowsView net, int C, long P, const float* __restrict__ w, const float* __restrict__ bias,
                                                       float* __restrict__ rgb, int accumulate, int sigmoid, float* __restrict__ out) {
    extern __shared__ float ws[];                  // [3][C]
    for (int i = (int)threadIdx.x; i < 3 * C; i += 256) ws[i] = w[i];
    __syncthreads();
    const long b = blockIdx.y, p = (long)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int l = (int)threadIdx.x & 7;
    if (p >= P) return;                                        // eight lanes share a pixel: they stay together
    const RowsAt r = rows_at(net, b, P, C);
    const float f = ROWS8 ? row_factor(r, p) : 1.0f;
    float a[3] = {0.0f, 0.0f, 0.0f};
    for (int c0 = 8 * l; c0 < C; c0 += 64) {
        float v[8];
        if constexpr (ROWS8) {
            const int8_t* qr = r.q + p * net.pitch + c0;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c0 + e < C ? (float)qr[e] * f : 0.0f;
        } else {
            const Vec<__bf16> t = load_part(r.v + p * C + c0, C - c0);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)t.v[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + e < C)
#pragma unroll
                for (int o = 0; o < 3; ++o) a[o] = fmaf(ws[o * C + c0 + e], v[e], a[o]);
    }
#pragma unroll
    for (int o = 0; o < 3; ++o)
#pragma unroll
        for (int i = 1; i < 8; i <<= 1) a[o] += __shfl_xor(a[o], i);
    if (l < 3) {
        float t = (l == 0 ? a[0] : (l == 1 ? a[1] : a[2])) + bias[l];
        float* rp = rgb + (b * 3 + l) * P + p;
        if (accumulate) t += *rp;
        if (sigmoid) t = 1.0f / (1.0f + expf(-t));
        if (out) out[(b * 3 + l) * P + p] = t;
        else *rp = t;
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct Up8Ws {
    int8_t* q0; float* s0;        // rows of a block's input          [B P][pitch(C)]
    __bf16* a;                    // a1, then a2                      [B P][4 C]
    int8_t* q1; float* s1;        // rows of a1                       [B P][pitch(2 C)]
    int8_t* q2; float* s2;        // rows of v                        [B 4P][pitch(C)]
    __bf16* net[2];               // the blocks' outputs, in turn     [B 4P][Cn]
    float* rgb[2];                // the running RGB image, in turn   [B][3][..]
};
static long pitch8(long k) { return (k + 63) & ~63L; }

static size_t up8_carve(const UpDims& d, int batch, bool cached, char* base, Up8Ws* s) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char* p = base ? base + off : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return p;
    };
    const size_t B = (size_t)batch;
    size_t q0 = 0, r0 = 0, a = 0, q1 = 0, r1 = 0, q2 = 0, r2 = 0, net = 0;
    for (int i = 0; i < d.n_blocks; ++i) {
        const size_t C = d.ch[i], Cn = d.ch[i + 1], n = B * (size_t)d.side[i] * d.side[i];
        if (i || !cached) {
            if (n * pitch8(C) > q0) q0 = n * pitch8(C);
            if (n > r0) r0 = n;
        }
        if (n * 4 * C * 2 > a) a = n * 4 * C * 2;
        if (n * pitch8(2 * C) > q1) q1 = n * pitch8(2 * C);
        if (n > r1) r1 = n;
        if (4 * n * pitch8(C) > q2) q2 = 4 * n * pitch8(C);
        if (4 * n > r2) r2 = 4 * n;
        if (4 * n * Cn * 2 > net) net = 4 * n * Cn * 2;
    }
    const size_t Pn = (size_t)d.side[d.n_blocks] * d.side[d.n_blocks];
    Up8Ws z{};
    z.q0 = (int8_t*)take(q0); z.s0 = (float*)take(r0 * 4);
    z.a = (__bf16*)take(a);
    z.q1 = (int8_t*)take(q1); z.s1 = (float*)take(r1 * 4);
    z.q2 = (int8_t*)take(q2); z.s2 = (float*)take(r2 * 4);
    for (int i = 0; i < 2; ++i) z.net[i] = (__bf16*)take(net);
    for (int i = 0; i < 2; ++i) z.rgb[i] = (float*)take(B * 3 * Pn * 4);
    if (s) *s = z;
    return off;
}

static int check_up8(const GnrUpsampleProblem* p, const GnrUpsampleInt8* q, UpDims* d) {
    if (!p) return fail("gnr_upsample_int8: problem is NULL");
    if (!q) return fail("gnr_upsample_int8: GnrUpsampleInt8 is NULL");
    if (q->struct_size != sizeof(GnrUpsampleInt8))
        return fail("gnr_upsample_int8: GnrUpsampleInt8.struct_size is %u but this libgnr.so (ABI %d) has sizeof = %zu: the caller "
                    "was built against a different include/gnr.h (or did not set struct_size)", q->struct_size, GNR_ABI_VERSION,
                    sizeof(GnrUpsampleInt8));
    GnrUpsampleProblem t = *p;
    if (!t.x) t.x = (const float*)q->x_q;                     // cached rows stand in for the map
    if (up_dims(&t, d)) return 1;
    if (p->x && q->x_q) return fail("gnr_upsample_int8: both x and x_q are given");
    if (q->x_q) {
        if (!q->x_scale) return fail("gnr_upsample_int8: x_scale is NULL");
        if (q->slots && q->n_slots < 1) return fail("gnr_upsample_int8: slots are given but n_slots is %lld", (long long)q->n_slots);
        if (q->x_pitch % 16 || q->x_pitch < ((p->feat_nc + 15) & ~15) || q->x_batch % 16 || q->x_batch < 0 || ((uintptr_t)q->x_q & 15) || q->x_scale_batch < 0)
            return fail("gnr_upsample_int8: cached rows must stand on a 16-byte boundary with strides that are multiples of 16 and hold feat_nc");
    }
    for (int i = 0; i < d->n_blocks; ++i)
        if (d->ch[i] < 4) return fail("gnr_upsample_int8: block %d has %d channels, at least 4 are needed", i, d->ch[i]);
    if (p->batch > 65535) return fail("gnr_upsample_int8: batch %d exceeds one launch", p->batch);
    return 0;
}

}  // namespace gnr

using namespace gnr;

extern "C" {

size_t gnr_upsample_int8_workspace_bytes(const GnrUpsampleProblem* p, const GnrUpsampleInt8* q) {
    UpDims d;
    if (check_up8(p, q, &d)) return 0;
    return up8_carve(d, p->batch, q->x_q != nullptr, nullptr, nullptr);
}

int gnr_upsample_int8_fwd(const GnrUpsampleProblem* p, const GnrUpsampleWeights* w, const GnrUpsampleInt8* q, float* img, void* workspace,
                          size_t ws_bytes, void* stream) {
    UpDims d;
    if (check_up8(p, q, &d)) return 1;
    if (!w) return fail("gnr_upsample_int8_fwd: weights are NULL");
    for (int i = 0; i < d.n_blocks; ++i)
        if (!w->up1_b[i] || !w->up2_b[i] || !w->feat_b[i] || !q->up1_w[i] || !q->up1_s[i] || !q->up2_w[i] || !q->up2_s[i] || !q->feat_w[i] || !q->feat_s[i])
            return fail("gnr_upsample_int8_fwd: a block-%d weight, scale or bias pointer is NULL", i);
    for (int i = 0; i <= d.n_blocks; ++i)
        if (!w->rgb_w[i] || !w->rgb_b[i]) return fail("gnr_upsample_int8_fwd: feat_2_rgb_list.%d pointer is NULL", i);
    if (!img) return fail("gnr_upsample_int8_fwd: output image is NULL");
    const size_t need = up8_carve(d, p->batch, q->x_q != nullptr, nullptr, nullptr);
    if (!workspace || ws_bytes < need) return fail("gnr_upsample_int8_fwd: workspace too small (%zu < %zu bytes)", ws_bytes, need);
    if ((uintptr_t)workspace & 255) return fail("gnr_upsample_int8_fwd: workspace must be 256-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    Up8Ws s;
    up8_carve(d, p->batch, q->x_q != nullptr, (char*)workspace, &s);
    const int B = p->batch;

    auto quantise = [&](const void* x, int dtype, int cf, long P, int C, int8_t* out, float* scale) {
        GnrRowsProblem r = GNR_INIT_ROWS_PROBLEM;
        r.dtype = dtype; r.channels_first = cf; r.batch = B; r.n_pix = P; r.channels = C;
        r.x = (void*)x; r.x_batch = P * C; r.x_stride = cf ? P : C;
        r.q = out; r.q_pitch = pitch8(C); r.q_batch = r.q_pitch * P; r.scale = scale; r.scale_batch = P;
        return gnr_quantize_rows(&r, stream);
    };
    auto product = [&](const RowsView& x, long P, int K, const int8_t* wq, long w_pitch, const float* wsc, const float* bias, int O, __bf16* y) {
        GnrInt8Problem g = GNR_INIT_INT8_PROBLEM;
        g.x_type = GNR_I8; g.y_type = GNR_BF16; g.leaky = 1; g.batch = B; g.n_pix = P; g.k = K; g.o = O;
        g.x = x.q; g.x_batch = x.batch; g.x_stride = x.pitch; g.x_scale = x.scale; g.x_scale_batch = x.scale_batch; g.slots = x.slots; g.n_slots = x.n_slots;
        g.w = wq; g.w_pitch = w_pitch; g.w_scale = wsc; g.bias = bias; g.y = y;
        return gnr_int8_linear(&g, nullptr, 0, stream);
    };
    auto rgb_rows = [&](const RowsView& net, int C, long P, int level, float* rgb, int accumulate, int sigmoid, float* out) {
        const dim3 grid((unsigned)((P + 31) / 32), (unsigned)B);
        if (net.v) hipLaunchKernelGGL(rgb_rows_kernel<false>, grid, dim3(256), 12 * C, st, net, C, P, w->rgb_w[level], w->rgb_b[level], rgb, accumulate, sigmoid, out);
        else hipLaunchKernelGGL(rgb_rows_kernel<true>, grid, dim3(256), 12 * C, st, net, C, P, w->rgb_w[level], w->rgb_b[level], rgb, accumulate, sigmoid, out);
    };

    const long P0 = (long)d.side[0] * d.side[0];
    RowsView in{};                                             // the block's input as 8-bit rows
    if (q->x_q) {
        in.q = q->x_q; in.batch = q->x_batch; in.pitch = q->x_pitch; in.scale = q->x_scale; in.scale_batch = q->x_scale_batch;
        in.slots = q->slots; in.n_slots = q->n_slots;
    } else {
        if (quantise(p->x, GNR_F32, 1, P0, d.ch[0], s.q0, s.s0)) return 1;
        in.q = s.q0; in.pitch = pitch8(d.ch[0]); in.batch = in.pitch * P0; in.scale = s.s0; in.scale_batch = P0;
    }
    RowsView res = in;                                         // ... and as the residual takes it: bf16 from the second block on
    float* rgb = s.rgb[0];
    float* other = s.rgb[1];
    rgb_rows(in, d.ch[0], P0, 0, other, 0, 0, nullptr);
    up_rgb(other, rgb, B, d.side[0], st);
    for (int i = 0; i < d.n_blocks; ++i) {
        const int C = d.ch[i], Cn = d.ch[i + 1], S = d.side[i];
        const long P = (long)S * S;
        const bool last = i == d.n_blocks - 1;
        if (product(in, P, C, q->up1_w[i], q->up1_pitch[i], q->up1_s[i], w->up1_b[i], 2 * C, s.a)) return 1;
        if (quantise(s.a, GNR_BF16, 0, P, 2 * C, s.q1, s.s1)) return 1;
        RowsView r1{};
        r1.q = s.q1; r1.pitch = pitch8(2 * C); r1.batch = r1.pitch * P; r1.scale = s.s1; r1.scale_batch = P;
        if (product(r1, P, 2 * C, q->up2_w[i], q->up2_pitch[i], q->up2_s[i], w->up2_b[i], 4 * C, s.a)) return 1;
        int lg = 0;
        while (1 << lg < S) ++lg;
        const int groups = C <= SB_THREADS ? SB_THREADS / C : 1;
        const long runs = P / SB_RUN;
        const int g = groups < 8 ? groups : 8;                 // LDS: 16 rows a group
        const dim3 grid((unsigned)((runs + g - 1) / g), (unsigned)B);
        const size_t lds = sizeof(float) * (size_t)g * SB_RUN * 4 * (C | 1);
#define GNR_SB(ROWS8, WRAP) hipLaunchKernelGGL((shuffle_blur_rows_kernel<ROWS8, WRAP>), grid, dim3(SB_THREADS), lds, st, s.a, res, C, lg, g, s.q2, pitch8(C), s.s2)
        if (res.v) { if (C % 4) GNR_SB(false, true); else GNR_SB(false, false); }
        else { if (C % 4) GNR_SB(true, true); else GNR_SB(true, false); }
#undef GNR_SB
        RowsView r2{};
        r2.q = s.q2; r2.pitch = pitch8(C); r2.batch = r2.pitch * 4 * P; r2.scale = s.s2; r2.scale_batch = 4 * P;
        if (product(r2, 4 * P, C, q->feat_w[i], q->feat_pitch[i], q->feat_s[i], w->feat_b[i], Cn, s.net[i & 1])) return 1;
        RowsView net{};
        net.v = s.net[i & 1];
        rgb_rows(net, Cn, 4 * P, i + 1, rgb, 1, last && p->final_sigmoid, last ? img : nullptr);
        if (!last) {
            up_rgb(rgb, other, B, 2 * S, st);
            float* t = rgb; rgb = other; other = t;
            if (quantise(s.net[i & 1], GNR_BF16, 0, 4 * P, Cn, s.q0, s.s0)) return 1;
            in = RowsView{};
            in.q = s.q0; in.pitch = pitch8(Cn); in.batch = in.pitch * 4 * P; in.scale = s.s0; in.scale_batch = 4 * P;
            res = net;
        }
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("gnr_upsample_int8_fwd: launch failed: %s", hipGetErrorString(e));
}

}  // extern "C"
