// gnr_int8.hip -- the 8-bit matrix product of rows (gnr_int8.h) on the CDNA4 integer MFMA:
//
//     y(n, o) = act((sum_k x_q(n,k) w_q(o,k)) * x_scale(n) * w_scale(o) + bias(o)),   act = identity or LeakyReLU(0.2)
//
// The sum is exact in 32 bits (K <= 131071: 128 * 128 * K < 2^31), so the result does not depend on the order of the work;
// the epilogue is in fp32, y is rounded once.  Both operands have their contraction index contiguous, 16 bytes = one lane's
// share of v_mfma_i32_32x32x32_i8 (row l % 32, k = 16 (l / 32) ..), so tiles go to LDS and to the MFMA as they are.
//
// The MFMA's result has four consecutive ROWS of the first operand in a lane, so the operand whose index is contiguous in y is
// the first: the weights for y [N][O], the pixels for y [B][O][P] (CF).  "m" below is that index, "n" the other one.
#include "gnr_int8.h"

namespace gnr {

struct Int8Args {
    const int8_t* x; long x_batch, x_pitch;
    const float* xs; long xs_batch;
    const int64_t* slots; long n_slots;
    const int8_t* w; long w_pitch;
    const float* ws; const float* bias;
    void* y;
    long P, N;                    // rows per batch entry, all rows
    int K, O, leaky;
};

struct RowRef {
    const int8_t* p;
    float scale;
};
// row n of x: through the slot list if there is one
__device__ __forceinline__ RowRef x_row(const Int8Args& a, long b, long pix) {
    const SlotRef r = slot_of(a.slots, a.n_slots, b);
    RowRef o;
    o.p = a.x + r.slot * a.x_batch + (r.state ? 0 : pix) * a.x_pitch;
    o.scale = r.state ? (r.state == 1 ? 0.0f : __uint_as_float(0x7fc00000u)) : a.xs[r.slot * a.xs_batch + pix];
    return o;
}

__device__ __forceinline__ float leak(float v) { return v > 0.0f ? v : 0.2f * v; }

// ---------------------------------------------------------------------------------------------
// the tiled product: WM x WN waves, each TM x TN tiles of 32 x 32
// ---------------------------------------------------------------------------------------------
template <typename T, bool CF, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(64 * WM * WN) void int8_tile_kernel(const Int8Args a, unsigned tiles_m, unsigned tiles_n) {
    constexpr int NW = WM * WN, NT = 64 * NW, BM = 32 * WM * TM, BN = 32 * WN * TN, BK = 64, PIECES = BK / 16;
    constexpr int ROWS = BM + BN, LOADS = (ROWS * PIECES + NT - 1) / NT;                  // 16-byte pieces a thread stages per step
    constexpr int EM = 32 * TM, ELD = EM + 4;                                  // epilogue: fp32 [32][EM + 4] per wave
    constexpr int STAGE = ROWS * BK, EPI = NW * 32 * ELD * 4;
    __shared__ __align__(16) char lds[STAGE > EPI ? STAGE : EPI];
    __shared__ float sc[ROWS], bi[CF ? BN : BM];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wn = wave / WM;
    const unsigned tm = blockIdx.x % tiles_m, rest = blockIdx.x / tiles_m, tn = rest % tiles_n;
    const long b = rest / tiles_n;                                             // CF: batch entry; otherwise 0
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const long M = CF ? a.P : a.O, N = CF ? a.O : a.N;

    // scales and bias of the tile's rows, and where each staged piece comes from
    for (int i = tid; i < ROWS; i += NT) {
        const bool is_m = i < BM;
        const long r = is_m ? m0 + i : n0 + i - BM;
        const bool is_x = is_m == CF;
        float s = 0.0f, z = 0.0f;
        if (r < (is_m ? M : N)) {
            if (is_x) s = x_row(a, CF ? b : r / a.P, CF ? r : r % a.P).scale;
            else { s = a.ws[r]; z = a.bias ? a.bias[r] : 0.0f; }
        }
        sc[i] = s;
        if (!is_x) bi[is_m ? i : i - BM] = z;
    }
    const int8_t* src[LOADS];
    int dst[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int idx = tid + j * NT, i = idx / PIECES, piece = idx % PIECES;
        const bool is_m = i < BM;
        const long lim = is_m ? M : N;
        long r = is_m ? m0 + i : n0 + i - BM;
        r = i < ROWS && r < lim ? r : lim - 1;
        src[j] = (is_m == CF ? x_row(a, CF ? b : r / a.P, CF ? r : r % a.P).p : a.w + r * a.w_pitch) + 16 * piece;
        dst[j] = i * BK + 16 * (piece ^ ((i >> 1) & 3));                       // any 8 lanes of a fragment read: 8 different 16-byte slots
    }
    const int my_piece = tid % PIECES;
    Vec<int> stage[LOADS];
    auto load = [&](int k0) {
        const int k = k0 + 16 * my_piece, left = a.K - k;                      // the bytes behind K of a row count as 0
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            Vec<int> v = {};
            if (left > 0) {
                __builtin_memcpy(&v, src[j] + k0, 16);
                if (left < 16)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        v.v[e] &= left >= 4 * e + 4 ? -1 : (left <= 4 * e ? 0 : (1 << 8 * (left - 4 * e)) - 1);
            }
            stage[j] = v;
        }
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};

    load(0);
    for (int k0 = 0; k0 < a.K; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
            if (tid + j * NT < ROWS * PIECES) __builtin_memcpy(lds + dst[j], &stage[j], 16);
        __syncthreads();
        if (k0 + BK < a.K) load(k0 + BK);
#pragma unroll
        for (int s = 0; s < BK / 32; ++s) {
            if (k0 + 32 * s >= a.K) break;
            const int piece = 2 * s + (lane >> 5);
            i32x4 fm[TM], fn[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int r = 32 * (wm * TM + i) + (lane & 31);
                fm[i] = *(const i32x4*)(lds + r * BK + 16 * (piece ^ ((r >> 1) & 3)));
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int r = BM + 32 * (wn * TN + j) + (lane & 31);
                fn[j] = *(const i32x4*)(lds + r * BK + 16 * (piece ^ ((r >> 1) & 3)));
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fm[i], fn[j], acc[i][j], 0, 0, 0);
        }
    }
    __syncthreads();

    // epilogue: scale, bias, activation in fp32; the wave's 32 x EM block turns in LDS so that stores run along m
    float* e = (float*)lds + wave * 32 * ELD;
    T* y = (T*)a.y + b * (long)a.O * a.P;
    const int mw = 32 * TM * wm;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int nl = 32 * (wn * TN + j) + (lane & 31);
        const float sn = sc[BM + nl], bn = CF ? bi[nl] : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = 32 * i + 8 * q + 4 * (lane >> 5);
                fv4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float sm = sc[mw + ml + r];
                    // x_scale first: the larger of the two factors as a rule, the same order for both layouts
                    const float t = (float)acc[i][j][4 * q + r] * (CF ? sm : sn) * (CF ? sn : sm) + (CF ? bn : bi[mw + ml + r]);
                    v[r] = a.leaky ? leak(t) : t;
                }
                *(fv4*)(e + (lane & 31) * ELD + ml) = v;
            }
        constexpr int V = Vec<T>::N, LPR = EM / V, RPI = 64 / LPR;             // lanes per row of m, rows per instruction
#pragma unroll
        for (int it = 0; it < 32 / RPI; ++it) {
            const int row = it * RPI + lane / LPR, m = (lane % LPR) * V;
            const long n = n0 + 32 * (wn * TN + j) + row, mg = m0 + mw + m;
            Vec<T> o;
#pragma unroll
            for (int v = 0; v < V; ++v) o.v[v] = (T)e[row * ELD + m + v];
            const long left = M - mg;
            if (n < N && left > 0) store_part(y + n * M + mg, o, left < V ? (int)left : V);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
static int check_int8(const GnrInt8Problem* p) {
    if (!p) return fail("gnr_int8_linear: problem is NULL");
    if (p->struct_size != sizeof(GnrInt8Problem))
        return fail("gnr_int8_linear: GnrInt8Problem.struct_size is %u but this libgnr.so (ABI %d) has sizeof = %zu: the caller was "
                    "built against a different include/gnr.h (or did not set struct_size)", p->struct_size, GNR_ABI_VERSION,
                    sizeof(GnrInt8Problem));
    const bool rows8 = p->x_type == GNR_I8;
    if (!rows8 && p->x_type != GNR_F32 && p->x_type != GNR_BF16 && p->x_type != GNR_F16) return fail("gnr_int8_linear: unknown x_type %d", p->x_type);
    if (p->y_type != GNR_F32 && p->y_type != GNR_BF16 && p->y_type != GNR_F16) return fail("gnr_int8_linear: unknown y_type %d", p->y_type);
    if (p->batch < 0 || p->n_pix < 0) return fail("gnr_int8_linear: batch and n_pix must be >= 0");
    if (p->k < 1 || p->o < 1) return fail("gnr_int8_linear: k and o must be >= 1 (got %d, %d)", p->k, p->o);
    if (p->k > GNR_INT8_MAX_K) return fail("gnr_int8_linear: k = %d exceeds %d: the 32-bit sum could overflow", p->k, GNR_INT8_MAX_K);
    if (p->x_channels_first && rows8) return fail("gnr_int8_linear: 8-bit rows have their channels last");
    if (p->slots && !rows8) return fail("gnr_int8_linear: slots name rows of a cache, x must be 8-bit rows");
    if (p->slots && p->n_slots < 1) return fail("gnr_int8_linear: slots are given but n_slots is %lld", (long long)p->n_slots);
    if (p->batch == 0 || p->n_pix == 0) return 0;
    if (p->n_pix > (1LL << 31) / p->batch) return fail("gnr_int8_linear: %d x %lld rows exceed 2^31", p->batch, (long long)p->n_pix);
    if (!p->x || !p->w || !p->w_scale || !p->y) return fail("gnr_int8_linear: NULL pointer");
    if (rows8 && !p->x_scale) return fail("gnr_int8_linear: x_scale is NULL (8-bit rows need one scale a row)");
    const int64_t k16 = ((int64_t)p->k + 15) & ~15LL;
    if (p->w_pitch % 16 || p->w_pitch < k16 || ((uintptr_t)p->w & 15))
        return fail("gnr_int8_linear: w must stand on a 16-byte boundary with a pitch that is a multiple of 16 and holds k (pitch %lld, k %d)", (long long)p->w_pitch, p->k);
    if (rows8 && (p->x_stride % 16 || p->x_stride < k16 || p->x_batch % 16 || p->x_batch < 0 || ((uintptr_t)p->x & 15)))
        return fail("gnr_int8_linear: 8-bit x must stand on a 16-byte boundary with strides that are multiples of 16 and hold k (x_stride %lld, "
                    "x_batch %lld, k %d)", (long long)p->x_stride, (long long)p->x_batch, p->k);
    if (p->x_batch < 0 || p->x_stride < 0 || p->x_scale_batch < 0) return fail("gnr_int8_linear: negative stride");
    return 0;
}

struct Int8Ws {
    size_t q_pitch, q_bytes, bytes;
};
static Int8Ws int8_ws(const GnrInt8Problem* p) {                     // floating x: its rows and their scales
    Int8Ws w{};
    if (p->x_type == GNR_I8) return w;
    const size_t n = (size_t)p->batch * (size_t)p->n_pix;
    w.q_pitch = ((size_t)p->k + 15) & ~(size_t)15;
    w.q_bytes = (n * w.q_pitch + 255) & ~(size_t)255;
    w.bytes = w.q_bytes + ((n * sizeof(float) + 255) & ~(size_t)255);
    return w;
}

template <typename T, bool CF, int WM, int WN, int TM, int TN> static int launch_tile(const Int8Args& a, long batch, hipStream_t st) {
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
    const long M = CF ? a.P : a.O, N = CF ? a.O : a.N;
    const long tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN, blocks = tm * tn * (CF ? batch : 1);
    if (blocks >= (1L << 31)) return fail("gnr_int8_linear: %ld tiles exceed one launch", blocks);
    hipLaunchKernelGGL((int8_tile_kernel<T, CF, WM, WN, TM, TN>), dim3((unsigned)blocks), dim3(64 * WM * WN), 0, st, a, (unsigned)tm, (unsigned)tn);
    return 0;
}

template <typename T> static int launch_int8(const Int8Args& a, long batch, bool cf, hipStream_t st) {
    if (cf) {
        if (a.O <= 32) return launch_tile<T, true, 4, 1, 2, 1>(a, batch, st);
        if (a.O <= 64) return launch_tile<T, true, 4, 1, 2, 2>(a, batch, st);
        return launch_tile<T, true, 2, 2, 2, 2>(a, batch, st);
    }
    if (a.O <= 64) return launch_tile<T, false, 1, 4, 2, 2>(a, batch, st);
    return launch_tile<T, false, 2, 2, 2, 2>(a, batch, st);
}

}  // namespace gnr

using namespace gnr;

extern "C" {

size_t gnr_int8_linear_workspace_bytes(const GnrInt8Problem* p) {
    if (check_int8(p)) return 0;
    const size_t n = int8_ws(p).bytes;
    return n ? n : 256;
}

int gnr_int8_linear(const GnrInt8Problem* p, void* workspace, size_t ws_bytes, void* stream) {
    if (check_int8(p)) return 1;
    if (p->batch == 0 || p->n_pix == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    Int8Args a{};
    a.P = p->n_pix; a.N = (long)p->batch * p->n_pix; a.K = p->k; a.O = p->o; a.leaky = p->leaky != 0;
    a.w = p->w; a.w_pitch = p->w_pitch; a.ws = p->w_scale; a.bias = p->bias; a.y = p->y;
    if (p->x_type == GNR_I8) {
        a.x = (const int8_t*)p->x; a.x_batch = p->x_batch; a.x_pitch = p->x_stride; a.xs = p->x_scale; a.xs_batch = p->x_scale_batch;
        a.slots = p->slots; a.n_slots = p->n_slots;
    } else {
        const Int8Ws w = int8_ws(p);
        if (!workspace || ws_bytes < w.bytes) return fail("gnr_int8_linear: workspace too small (%zu < %zu bytes)", ws_bytes, w.bytes);
        if ((uintptr_t)workspace & 255) return fail("gnr_int8_linear: workspace must be 256-byte aligned");
        GnrRowsProblem r = GNR_INIT_ROWS_PROBLEM;
        r.dtype = p->x_type; r.channels_first = p->x_channels_first; r.batch = p->batch; r.channels = p->k; r.n_pix = p->n_pix;
        r.x = (void*)p->x; r.x_batch = p->x_batch; r.x_stride = p->x_stride;
        r.q = (int8_t*)workspace; r.q_pitch = (int64_t)w.q_pitch; r.q_batch = r.q_pitch * p->n_pix;
        r.scale = (float*)((char*)workspace + w.q_bytes); r.scale_batch = p->n_pix;
        if (launch_quantize(r, st)) return 1;
        a.x = r.q; a.x_batch = r.q_batch; a.x_pitch = r.q_pitch; a.xs = r.scale; a.xs_batch = p->n_pix;
    }
    int rc;
    if (p->y_type == GNR_F32) rc = launch_int8<float>(a, p->batch, p->y_channels_first != 0, st);
    else if (p->y_type == GNR_BF16) rc = launch_int8<__bf16>(a, p->batch, p->y_channels_first != 0, st);
    else rc = launch_int8<_Float16>(a, p->batch, p->y_channels_first != 0, st);
    if (rc) return 1;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("gnr_int8_linear: launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // extern "C"
