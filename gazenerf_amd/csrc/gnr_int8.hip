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
#include <type_traits>

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
    const void* xf; long xf_batch, xf_pitch;     // floating rows or maps that a kernel quantises itself
    int flat;                     // no slots, and every row of x a.x_pitch behind the one before (scales alike)
};

// Row r of x and its scale.  y [N][O]: r counts all rows; y [B][O][P]: r counts the pixels of entry b.
__device__ __forceinline__ void x_at(const Int8Args& a, long& b, long& r, bool cf) {
    if (!cf && !a.flat) {
        b = (unsigned)r / (unsigned)a.P;
        r = (unsigned)r - (unsigned)b * (unsigned)a.P;
    }
}
__device__ __forceinline__ const int8_t* x_row(const Int8Args& a, long b, long r, bool cf) {
    x_at(a, b, r, cf);
    const SlotRef s = slot_of(a.slots, a.n_slots, b);
    return a.x + s.slot * a.x_batch + r * a.x_pitch;          // an entry without a slot reads slot 0 and is multiplied by 0 or NaN
}
__device__ __forceinline__ float x_scale(const Int8Args& a, long b, long r, bool cf) {
    x_at(a, b, r, cf);
    const SlotRef s = slot_of(a.slots, a.n_slots, b);
    return s.state ? (s.state == 1 ? 0.0f : __uint_as_float(0x7fc00000u)) : a.xs[s.slot * a.xs_batch + r];
}

__device__ __forceinline__ float leak(float v) { return fmaxf(v, 0.2f * v); }

// sum * x_scale * w_scale + bias in this order, two roundings; the same order for both layouts, hence the same bits.  The first product can
// leave fp32's normal range where the result does not: |sum| <= 2^31, so only for an x_scale FAR from 1 (a row whose largest value exceeds
// 2^103, a subnormal scale).  Then 2^64 goes from one scale to the other, exactly for every result in range.  A wave that sees no such scale
// does without: a test of every product cost 28672 x 516 -> 1032 2.4 us of 46.4.
__device__ __forceinline__ bool scale_is_far(float s) {
    const float m = fabsf(s);
    return m > 0x1p96f || (m < 0x1p-126f && m > 0.0f);
}
template <bool FAR> __device__ __forceinline__ float scaled(float sum, float sx, float sw, float b) {
    if constexpr (FAR) {
        constexpr int INF = 0x204, SUBNORMAL = 0x090;          // of v_cmp_class, both signs
        const float t = sum * sx;
        const bool big = __builtin_amdgcn_classf(t, INF), small = __builtin_amdgcn_classf(t, SUBNORMAL);
        sx *= big ? 0x1p-64f : (small ? 0x1p64f : 1.0f);
        sw *= big ? 0x1p64f : (small ? 0x1p-64f : 1.0f);
    }
    return fmaf(sum * sx, sw, b);
}

// ---------------------------------------------------------------------------------------------
// the tiled product: WM x WN waves, each TM x TN tiles of 32 x 32.
//
// K runs in stages of 64 bytes through a ring of NST LDS buffers that LDS-DMA fills (16 bytes a lane, no registers in between).  A stage
// is two MFMA steps; while one is multiplied the fragments of the next are read, across the one barrier of a stage too:
//     stage s + 1 has landed, barrier | step 1 of s, reading step 0 of s + 1 and requesting stage s + NST - 1 | step 0 of s + 1, reading step 1
// (an odd number of steps leaves out step 0 of the FIRST stage: at the end, a step that may be left out costs a second set of accumulators).
// The barrier of stage s stands behind every wave's reads of stage s - 1, whose buffer that request fills.  Reads and requests stand
// between the MFMAs (in front of them they cost 1945 against 2124 TOP/s at 8192^3).
// A 16-byte piece of tile row r sits at piece ^ ((r >> 1) & 3) of its 64 bytes (the swizzle is applied to the source address): the eight
// lanes that read together hit eight different 16-byte columns.
//
// What a workgroup waits for (its first stage, its stores) is covered by the other workgroups of the CU, so registers and LDS are kept
// low: accumulators in plain registers (launch bounds of two waves a SIMD), no more buffers than there are stages, an epilogue that turns
// 4 KiB blocks a wave.  (Workgroups that walk several tiles and request the next one's stages under the epilogue were built: they need
// twice the registers, and 262144 x 64 -> 32 took 9.2 us against 8.5, 458752 x 128 -> 256 64 against 56.)
// ---------------------------------------------------------------------------------------------
// m0 holds the LDS address; the compiler may keep a value of its own there and takes no clobber for it (a reserved register): it is put back
__device__ __forceinline__ void dma16(const int8_t* p, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(p), "s"(lds) : "memory");
}
template <int N> __device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N < 63 ? N : 63) : "memory");     // six bits; fewer than allowed is only stricter
}
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// the bytes at and behind `left` of a lane's 16 count as 0
__device__ __forceinline__ i32x4 keep_bytes(i32x4 v, int left) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] &= left >= 4 * e + 4 ? -1 : (left <= 4 * e ? 0 : (1 << 8 * (left - 4 * e)) - 1);
    return v;
}

template <int WM, int WN, int TM, int TN, int NST> struct TileShape {
    static constexpr int NW = WM * WN, NT = 64 * NW, BM = 32 * WM * TM, BN = 32 * WN * TN, ROWS = BM + BN;
    static constexpr int LOADS = (ROWS + 16 * NW - 1) / (16 * NW);             // requests of a wave per stage: 1 KiB = 16 rows each
    static constexpr int STAGE = LOADS * NW * 1024, TURN = NW * 4096;
};

template <typename T, bool CF, int WM, int WN, int TM, int TN, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void int8_tile_kernel(const Int8Args a, unsigned tiles_m, unsigned tiles_n) {
    typedef TileShape<WM, WN, TM, TN, NST> S;
    constexpr int BM = S::BM, BN = S::BN, ROWS = S::ROWS, LOADS = S::LOADS, STAGE = S::STAGE, NT = S::NT, BK = 64;
    constexpr int PAIR = sizeof(T) == 2 && TM % 2 == 0 ? 2 : 1;                // tiles of 32 x 32 that turn together
    constexpr int EM = 32 * PAIR, RB = EM * (int)sizeof(T), PPR = RB / 16;     // their row of m: values, bytes, 16-byte pieces
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ __attribute__((aligned(16))) float sc[ROWS], bi[CF ? BN : BM];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave % WM, wn = wave / WM;
    const int half = lane >> 5, sw = (lane >> 1) & 3, piece = (lane & 3) ^ ((lane >> 3) & 3);
    const long M = CF ? a.P : a.O, N = CF ? a.O : a.N;
    const int K16 = (a.K + 15) & ~15, steps = (a.K + 31) / 32, odd = steps & 1, nst = (steps + odd) / 2;
    const unsigned at = xcd_block(gridDim.x), tm = at % tiles_m, rest = at / tiles_m;
    const long m0 = (long)tm * BM, n0 = (long)(rest % tiles_n) * BN, b = rest / tiles_n;       // b: CF, the batch entry; otherwise 0

    const int8_t* src[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int i = (wave * LOADS + j) * 16 + (lane >> 2);
        const bool is_m = i < BM;
        const long lim = is_m ? M : N;
        long r = is_m ? m0 + i : n0 + i - BM;
        r = r < lim ? r : lim - 1;
        src[j] = is_m == CF ? x_row(a, b, r, CF) : a.w + r * a.w_pitch;
    }
    constexpr int SCN = (ROWS + NT - 1) / NT;
    float rs[SCN], rz[SCN];                                    // scales and bias of the tile's rows: requested first, needed last
#pragma unroll
    for (int j = 0; j < SCN; ++j) {
        const int i = tid + j * NT;
        const bool is_m = i < BM, is_x = is_m == CF;
        const long r = is_m ? m0 + i : n0 + i - BM;
        rs[j] = rz[j] = 0.0f;
        if (i < ROWS && r < (is_m ? M : N)) {
            if (is_x) rs[j] = x_scale(a, b, r, CF);
            else { rs[j] = a.ws[r]; rz[j] = a.bias ? a.bias[r] : 0.0f; }
        }
    }
    const unsigned lds0 = (unsigned)(size_t)&lds[0] + (unsigned)wave * LOADS * 1024u;
    auto request_at = [&](int s, int& k, unsigned& d) {
        k = s * BK - 32 * odd + 16 * piece;
        k = k < 0 ? 0 : (k < K16 ? k : K16 - 16);              // inside the row always: the step before the first is not multiplied, what is
                                                               // behind the last is masked
        d = lds0 + (unsigned)(s % NST) * STAGE;
    };
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < nst) {
            int k; unsigned d;
            request_at(s, k, d);
#pragma unroll
            for (int j = 0; j < LOADS; ++j) dma16(src[j] + k, d + j * 1024u);
        }
    i32x16 acc[TM][TN];
    i32x4 f[2][TM + TN];
    const int row_m = 32 * TM * wm + (lane & 31), row_n = BM + 32 * TN * wn + (lane & 31);
    auto read = [&](int s, int step, int i) {
        const char* base = lds + (s % NST) * STAGE + 16 * ((2 * step + half) ^ sw);
        f[step][i] = *(const i32x4*)(base + (i < TM ? row_m + 32 * i : row_n + 32 * (i - TM)) * BK);
    };
    // the MFMAs of one step; behind each of them: a fragment of the step that follows (next_s < 0: none), and the requests of a stage
    auto multiply = [&](int step, int next_s, int next_step, int req) {
        constexpr int MF = TM * TN, RD = TM + TN;
        int k; unsigned d;
        request_at(req < 0 ? 0 : req, k, d);
#pragma unroll
        for (int t = 0; t < MF; ++t) {
            acc[t / TN][t % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f[step][t / TN], f[step][TM + t % TN], acc[t / TN][t % TN], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < RD; ++i)
                if (i * MF / RD == t && next_s >= 0) read(next_s, next_step, i);
#pragma unroll
            for (int j = 0; j < LOADS; ++j)
                if (j * MF / LOADS == t && req >= 0 && req < nst) dma16(src[j] + k, d + j * 1024u);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};
    // Loads leave vmcnt in the order they were issued: what may stay outstanding is what was issued behind the stage that is needed
    if (NST > 3 && nst > 2) wait_vm<2 * LOADS>();
    else if (nst > 1) wait_vm<LOADS>();
    else wait_vm<0>();
    tile_barrier();
    if (odd) {                                                 // the first stage has one step
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) read(0, 1, i);
    } else {
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) read(0, 0, i);
        multiply(0, 0, 1, -1);
    }
    for (int s = 0; s < nst - 1; ++s) {
        if (NST > 3 && s + 2 < nst) wait_vm<LOADS>();
        else wait_vm<0>();
        tile_barrier();
        multiply(1, s + 1, 0, s + NST - 1);
        multiply(0, s + 1, 1, -1);
    }
    const int left = a.K - 32 * (steps - 1);                   // 1 .. 32 bytes of the last step exist
    if (left < 32)
#pragma unroll
        for (int i = 0; i < TM + TN; ++i) f[1][i] = keep_bytes(f[1][i], left - 16 * half);
    multiply(1, -1, 0, -1);
#pragma unroll
    for (int j = 0; j < SCN; ++j) {
        const int i = tid + j * NT;
        if (i < ROWS) {
            sc[i] = rs[j];
            if ((i < BM) != CF) bi[i < BM ? i : i - BM] = rz[j];
        }
    }
    tile_barrier();                                            // every wave is done with the ring, too

    // epilogue: scale, bias, activation in fp32; 32 rows of n x EM values turn in LDS so that a row leaves as whole lines
    char* turn = lds + wave * 4096;
    // past the caches: whole lines, or 16-bit rows that do not fit them anyway (53528 x 624 -> 4092, 438 MB of partial lines: 224 / 261 us; in
    // fp32 26764 x 624 -> 4092 232 / 184, maps of 233 x 220001 -> 570 362 / 195)
    const bool inside = m0 + BM <= M && n0 + BN <= N, past = M * sizeof(T) % 128 == 0 || (!CF && sizeof(T) == 2 && a.N * a.O * (long)sizeof(T) >= CACHES);
    const int mw = 32 * TM * wm;
    // a scale far from 1 among the wave's rows: value by value through LDS in a loop, stored as they come.  (Unrolled, or as a second copy of
    // the epilogue below, it takes 57 registers more: two waves a SIMD instead of four, 28672 x 258 -> 516 25 us instead of 21.)
    const float* xsc = CF ? sc + mw : sc + BM + 32 * TN * wn;
    bool far = false;
#pragma unroll
    for (int i = 0; i < (CF ? TM : TN); ++i) far |= scale_is_far(xsc[32 * i + (lane & 31)]);
    if (__any(far)) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) *(i32x4*)(turn + 1024 * q + 16 * lane) = i32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
#pragma unroll 1
                for (int r = 0; r < 16; ++r) {
                    const int ml = mw + 32 * i + 8 * (r >> 2) + 4 * half + (r & 3), nl = 32 * (wn * TN + j) + (lane & 31);
                    if (m0 + ml < M && n0 + nl < N) {
                        float v = scaled<true>((float)*(const int*)(turn + 1024 * (r >> 2) + 16 * lane + 4 * (r & 3)), sc[CF ? ml : BM + nl], sc[CF ? BM + nl : ml], bi[CF ? nl : ml]);
                        if (a.leaky) v = leak(v);
                        ((T*)a.y)[b * (long)a.O * a.P + (n0 + nl) * M + m0 + ml] = (T)v;
                    }
                }
            }
        return;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int nl = 32 * (wn * TN + j), nr = lane & 31;
        const float sn = sc[BM + nl + nr], bn = CF ? bi[nl + nr] : 0.0f;
        T* yn = (T*)a.y + b * (long)a.O * a.P + (n0 + nl) * M + m0 + mw;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int ml = 8 * q + 4 * half;
                const fv4 sm = *(const fv4*)(sc + mw + 32 * i + ml), bm = CF ? fv4{bn, bn, bn, bn} : *(const fv4*)(bi + mw + 32 * i + ml);
                typedef T t4 __attribute__((ext_vector_type(4)));
                t4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = scaled<false>((float)acc[i][j][4 * q + r], CF ? sm[r] : sn, CF ? sn : sm[r], bm[r]);
                    if (a.leaky) v = leak(v);
                    o[r] = (T)v;
                }
                const int at = 32 * (i % PAIR) + ml;
                if constexpr (sizeof(T) == 4) *(t4*)(turn + nr * RB + 16 * ((at >> 2) ^ (nr & (PPR - 1)))) = o;
                else *(t4*)(turn + nr * RB + 16 * ((at >> 3) ^ (nr & (PPR - 1))) + 2 * (at & 4)) = o;
            }
            if (i % PAIR == PAIR - 1) {
#pragma unroll
                for (int it = 0; it < 32 * PPR / 64; ++it) {
                    const int row = it * (64 / PPR) + lane / PPR, pc = lane % PPR;
                    Vec<T> o;
                    __builtin_memcpy(&o, __builtin_assume_aligned(turn + row * RB + 16 * (pc ^ (row & (PPR - 1))), 16), 16);
                    const int ml = 32 * (i - PAIR + 1) + Vec<T>::N * pc;
                    T* p = yn + row * M + ml;
                    if (inside && past) store_part<true>(p, o, Vec<T>::N);
                    else if (inside) store_part(p, o, Vec<T>::N);
                    else if (n0 + nl + row < N && m0 + mw + ml < M) {
                        const long left = M - m0 - mw - ml;
                        store_part(p, o, left < Vec<T>::N ? (int)left : Vec<T>::N);
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// few rows: the time to read the weights.  A workgroup owns 16 outputs of 16 TT rows; its four waves share K in steps of 64 bytes
// (v_mfma_i32_16x16x64_i8: lane l holds row l % 16, bytes 16 (l / 16) ..) and keep eight steps of weights in flight, fragments
// straight from memory; the four partial sums are whole numbers and meet in LDS.  Floating x is quantised by every workgroup
// for itself (TT == 1): one launch instead of two.
// ---------------------------------------------------------------------------------------------
constexpr int FEW_MAX = 64, FEW_FUSED = 16, FEW_FUSED_K = 4096;

// floating rows -> 8-bit rows [n][ld] and scales in LDS, L lanes a row, eight pieces of 16 bytes a lane (longer rows are read twice)
template <typename X, int L> __device__ __forceinline__ void few_rows(const X* xb, long pitch, int N, int K, int K64, int ld, char* lds, float* xsc) {
    constexpr int V = Vec<X>::N, J = 8;
    const int lane = (int)threadIdx.x % L;
    for (int n = (int)threadIdx.x / L; n < N; n += 256 / L) {
        const X* row = xb + (long)n * pitch;
        Raw16 r[J];
        unsigned m[4] = {};
        auto get = [&](int j0) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c = ((j0 + j) * L + lane) * V;
                r[j] = c < K ? load_raw(row + c, K - c) : Raw16{};
            }
        };
        const int pieces = (K + L * V - 1) / (L * V);
        for (int j0 = 0; j0 < pieces; j0 += J) {
            get(j0);
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) m[i] = max_bits<X>(m[i], r[j].w[i]);
        }
        m[0] = max_bits<X>(max_bits<X>(m[0], m[1]), max_bits<X>(m[2], m[3]));
#pragma unroll
        for (int i = 1; i < L; i <<= 1) m[0] = max_bits<X>(m[0], (unsigned)__shfl_xor((int)m[0], i));
        if constexpr (sizeof(X) == 2) m[0] = max_bits<X>(m[0], m[0] >> 16);
        float s, per;
        row_scale(__float_as_uint(raw_value<X>(m, 0)), s, per);
        if (lane == 0) xsc[n] = s;
        for (int j0 = 0; j0 < pieces; j0 += J) {
            if (pieces > J) get(j0);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c = ((j0 + j) * L + lane) * V;       // bytes behind K become 0: load_raw filled up with 0
                if (c < K64) {
                    unsigned q[V / 4];
#pragma unroll
                    for (int i = 0; i < V / 4; ++i)
                        q[i] = pack4(row_step(raw_value<X>(r[j].w, 4 * i), per), row_step(raw_value<X>(r[j].w, 4 * i + 1), per),
                                     row_step(raw_value<X>(r[j].w, 4 * i + 2), per), row_step(raw_value<X>(r[j].w, 4 * i + 3), per));
                    __builtin_memcpy(__builtin_assume_aligned(lds + n * ld + c, V), q, V);
                }
            }
        }
    }
}

template <typename X, typename T, bool CF, int TT>
__global__ __launch_bounds__(256) void int8_few_kernel(const Int8Args a) {
    constexpr bool FLOAT = !__is_same(X, int8_t);
    constexpr int U = TT == 1 ? 8 : 4;                         // steps in flight
    extern __shared__ __attribute__((aligned(16))) char lds[];                 // FLOAT: rows of x, [16][ld]; then the partial sums
    __shared__ float xsc[16 * TT];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, kq = 16 * (lane >> 4);
    const long n0 = (long)blockIdx.y * 16 * TT;                // FLOAT: 0
    const int N = a.N - n0 < 16 * TT ? (int)(a.N - n0) : 16 * TT, K = a.K, K16 = (K + 15) & ~15, nst = (K + 63) / 64, o0 = (int)blockIdx.x * 16;
    const int ld = nst * 64 + 16;
    const int o = o0 + col < a.O ? o0 + col : a.O - 1;
    const int8_t* wp = a.w + (long)o * a.w_pitch;
    const int8_t* xp[TT];
    if constexpr (!FLOAT) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int n = 16 * t + col < N ? 16 * t + col : N - 1;
            xp[t] = x_row(a, 0, n0 + n, false);
        }
        if (tid < 16 * TT) xsc[tid] = x_scale(a, 0, n0 + (tid < N ? tid : N - 1), false);
    }
    i32x4 w[U], x[U][TT];
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + 4 * u;
            if (s < nst) {
                const int k = s * 64 + kq < K16 ? s * 64 + kq : K16 - 16;      // never behind a row; masked below
                w[u] = *(const i32x4*)(wp + k);
                if constexpr (!FLOAT)
#pragma unroll
                    for (int t = 0; t < TT; ++t) x[u][t] = *(const i32x4*)(xp[t] + k);
            }
        }
    };
    load(wave);                                                // under the quantisation
    if constexpr (FLOAT) {
        // one row a wave and turn, or four rows a wave where a sixteenth of one fits the same registers
        if (N > 4 && K <= 16 * 8 * Vec<X>::N) few_rows<X, 16>((const X*)a.xf, a.xf_pitch, N, K, nst * 64, ld, lds, xsc);
        else few_rows<X, 64>((const X*)a.xf, a.xf_pitch, N, K, nst * 64, ld, lds, xsc);
    }
    i32x4 acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = i32x4{};
    if constexpr (FLOAT) __syncthreads();
    for (int s0 = wave; s0 < nst; s0 += 4 * U) {
        if (s0 != wave) load(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + 4 * u;
            if (s >= nst) break;
            const int left = K - s * 64 - kq;
            if (K - s * 64 < 64) w[u] = keep_bytes(w[u], left);
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                if constexpr (FLOAT) x[u][t] = *(const i32x4*)(lds + (col < N ? col : 0) * ld + s * 64 + kq);
                else if (K - s * 64 < 64) x[u][t] = keep_bytes(x[u][t], left);
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[u], x[u][t], acc[t], 0, 0, 0);
            }
        }
    }
    __syncthreads();                                           // the rows in LDS have been read
    i32x4* part = (i32x4*)lds;                                 // [wave][TT][64]
#pragma unroll
    for (int t = 0; t < TT; ++t) part[(wave * TT + t) * 64 + lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < TT; t += 4) {
        i32x4 sum = part[t * 64 + lane];
#pragma unroll
        for (int v = 1; v < 4; ++v) sum += part[(v * TT + t) * 64 + lane];
        const int n = 16 * t + col;
        if (n >= N) continue;
        const float sx = xsc[n];
        const unsigned P = (unsigned)a.P, at = (unsigned)(n0 + n);
        T* y = CF ? (T*)a.y + (long)(at / P) * a.O * P + at % P : (T*)a.y + (n0 + n) * a.O;
        const bool far = __any(scale_is_far(sx));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int oo = o0 + 4 * (lane >> 4) + r;
            if (oo < a.O) {
                const float wb = a.bias ? a.bias[oo] : 0.0f;
                float v = far ? scaled<true>((float)sum[r], sx, a.ws[oo], wb) : scaled<false>((float)sum[r], sx, a.ws[oo], wb);
                if (a.leaky) v = leak(v);
                y[CF ? (long)oo * P : (long)oo] = (T)v;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// floating x, few outputs or few rows: quantise and multiply in one launch.  A workgroup turns 32 NMT rows of x into 8-bit rows in LDS (maps: as
// quant_maps_kernel reads them; rows: eight lanes a row) and multiplies them with `span` tiles of 32 outputs, the weights read from L2
// fragment by fragment, so neither the 8-bit rows nor a second launch pass through memory.  A wave takes one 32-row tile (wave % NMT) and
// every (4 / NMT)th output tile.  See the rule at int8_fuse.
// ---------------------------------------------------------------------------------------------
constexpr int FUSED_MAX_K = 512;
__host__ __device__ constexpr int fused_ld(int K) { return (K + 31) / 32 * 32 + 16; }       // a row in LDS; + 16: eight lanes hit different columns

template <typename X, typename T, bool CF, int NMT>
__global__ __launch_bounds__(256) void int8_fused_kernel(const Int8Args a, unsigned tiles, unsigned parts, int span) {
    constexpr int V = Vec<X>::N, TP = 32 * NMT, NW = 4, NT = 64 * NW, U = 8;        // U: steps of K whose weights are in flight
    extern __shared__ __attribute__((aligned(16))) char lds[];                 // [TP][ld] rows, then 4 KiB a wave for the epilogue
    __shared__ unsigned amax[NW][CF ? TP : 1];
    __shared__ __attribute__((aligned(16))) float xs[TP];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, K = a.K, ld = fused_ld(K), K32 = (K + 31) & ~31;
    const unsigned blk = xcd_block(gridDim.x), at = blk / parts;               // a tile's parts of the outputs are neighbours
    const long b = CF ? at / tiles : 0, P = CF ? a.P : a.N, p0 = (long)(CF ? at % tiles : at) * TP;
    const int rows = P - p0 < TP ? (int)(P - p0) : TP;
    constexpr int OW = NW / NMT;                               // waves that share a 32-row tile
    const int mt = wave % NMT, steps = K32 / 32, half = lane >> 5, K16 = (K + 15) & ~15, o_tiles = (a.O + 31) / 32;
    const int ot0 = (int)(blk % parts) * span + wave / NMT, ot1 = (int)(blk % parts) * span + span < o_tiles ? (int)(blk % parts) * span + span : o_tiles;
    i32x4 w[U];
    auto weights = [&](int ot, int s0) {
        const int o = 32 * ot + (lane & 31) < a.O ? 32 * ot + (lane & 31) : a.O - 1;
        const int8_t* wp = a.w + (long)o * a.w_pitch;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = 32 * (s0 + u) + 16 * half;
            if (s0 + u < steps) w[u] = *(const i32x4*)(wp + (k < K16 ? k : K16 - 16));     // never behind the row
        }
    };
    if (NMT == 1 && ot0 < ot1) weights(ot0, 0);                // under the quantisation (larger tiles: the registers cost more than it gives)

    if constexpr (CF) {                                        // maps: element (b, c, p) at xf[b xf_batch + c xf_pitch + p]
        constexpr int LPX = TP / V, G = NT / LPX, R = 4;
        const int l = tid % LPX, g = tid / LPX;
        const X* xb = (const X*)a.xf + b * a.xf_batch + p0 + l * V;
        const int nv = rows - l * V;
        Raw16 x[R][4];
        unsigned m[4] = {};
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = 4 * (r * G + g) + e;
                x[r][e] = c < K && nv > 0 ? load_raw(xb + (long)c * a.xf_pitch, nv) : Raw16{};
            }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int w = 0; w < 4; ++w) m[w] = max_bits<X>(m[w], x[r][e].w[w]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
#pragma unroll
            for (int i = LPX; i < 64; i <<= 1) m[w] = max_bits<X>(m[w], (unsigned)__shfl_xor((int)m[w], i));
            if (lane < LPX) amax[wave][l * 4 + w] = m[w];
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w)
            for (int i = 0; i < NW; ++i) m[w] = max_bits<X>(m[w], amax[i][l * 4 + w]);
        float per[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float s;
            row_scale(__float_as_uint(raw_value<X>(m, v)), s, per[v]);
            if (g == 0) xs[l * V + v] = s;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = 4 * (r * G + g);
            if (c < K32)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    *(unsigned*)(lds + (l * V + v) * ld + c) = pack4(row_step(raw_value<X>(x[r][0].w, v), per[v]), row_step(raw_value<X>(x[r][1].w, v), per[v]),
                                                                     row_step(raw_value<X>(x[r][2].w, v), per[v]), row_step(raw_value<X>(x[r][3].w, v), per[v]));
        }
    } else {                                                   // rows
        constexpr int LPR = NT / 32, J = FUSED_MAX_K / (LPR * V) > 0 ? FUSED_MAX_K / (LPR * V) : 1;      // 32 rows at a time
        const int l = tid % LPR;
#pragma unroll 1
        for (int t = 0; t < NMT; ++t) {
            const int i = 32 * t + tid / LPR;
            const X* row = (const X*)a.xf + (p0 + (i < rows ? i : rows - 1)) * a.xf_pitch;
            Raw16 x[J];
            unsigned m[4] = {};
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c = (j * LPR + l) * V;
                x[j] = c < K ? load_raw(row + c, K - c) : Raw16{};
            }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int w = 0; w < 4; ++w) m[w] = max_bits<X>(m[w], x[j].w[w]);
            m[0] = max_bits<X>(max_bits<X>(m[0], m[1]), max_bits<X>(m[2], m[3]));
#pragma unroll
            for (int e = 1; e < LPR; e <<= 1) m[0] = max_bits<X>(m[0], (unsigned)__shfl_xor((int)m[0], e));
            if constexpr (sizeof(X) == 2) m[0] = max_bits<X>(m[0], m[0] >> 16);
            float s, per;
            row_scale(__float_as_uint(raw_value<X>(m, 0)), s, per);
            if (l == 0) xs[i] = s;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int c = (j * LPR + l) * V;
                if (c < K32) {
                    unsigned q[V / 4];
#pragma unroll
                    for (int w = 0; w < V / 4; ++w)
                        q[w] = pack4(row_step(raw_value<X>(x[j].w, 4 * w), per), row_step(raw_value<X>(x[j].w, 4 * w + 1), per),
                                     row_step(raw_value<X>(x[j].w, 4 * w + 2), per), row_step(raw_value<X>(x[j].w, 4 * w + 3), per));
                    __builtin_memcpy(__builtin_assume_aligned(lds + i * ld + c, V), q, V);
                }
            }
        }
    }
    __syncthreads();

    const char* xr = lds + (32 * mt + (lane & 31)) * ld + 16 * half;
    float* turn = (float*)(lds + TP * ld) + wave * 1024;
    const long M = CF ? a.P : a.O;
    T* yb = (T*)a.y + (CF ? b * (long)a.O * a.P : 0);
    for (int ot = ot0; ot < ot1; ot += OW) {
        const int o = 32 * ot + (lane & 31) < a.O ? 32 * ot + (lane & 31) : a.O - 1;
        const float wsc = a.ws[o], wb = a.bias ? a.bias[o] : 0.0f;
        i32x16 acc = {};
        for (int s0 = 0; s0 < steps; s0 += U) {
            if (NMT > 1 || s0 || ot != ot0) weights(ot, s0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = 32 * (s0 + u);
                if (s0 + u >= steps) continue;
                const i32x4 xv = *(const i32x4*)(xr + k);      // the bytes behind K are 0 here: what stands there in w does not count
                acc = CF ? __builtin_amdgcn_mfma_i32_32x32x32_i8(xv, w[u], acc, 0, 0, 0) : __builtin_amdgcn_mfma_i32_32x32x32_i8(w[u], xv, acc, 0, 0, 0);
            }
        }
        // m: pixels (CF) or outputs; n = lane % 32: outputs (CF) or rows.  The 32 x 32 values turn in LDS so that stores run along m.
        const int nr = lane & 31;
        const float xn = xs[32 * mt + nr];
        auto scale_up = [&](auto is_far) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                fv4 v;
                const int ml = 8 * q + 4 * half;
                fv4 sm, bm;
                if constexpr (CF) {
                    sm = *(const fv4*)(xs + 32 * mt + ml);
                    bm = fv4{wb, wb, wb, wb};
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        sm[r] = __shfl(wsc, ml + r);
                        bm[r] = __shfl(wb, ml + r);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] = scaled<decltype(is_far)::value>((float)acc[4 * q + r], CF ? sm[r] : xn, CF ? wsc : sm[r], bm[r]);
                    if (a.leaky) v[r] = leak(v[r]);
                }
                *(fv4*)(turn + nr * 32 + 4 * ((ml >> 2) ^ (nr & 7))) = v;
            }
        };
        if (__any(scale_is_far(xn))) scale_up(std::true_type{});
        else scale_up(std::false_type{});
        constexpr int TV = Vec<T>::N, PPR = 32 / TV;           // 16-byte pieces of T in a row of 32
#pragma unroll
        for (int it = 0; it < 32 * PPR / 64; ++it) {
            const int row = it * (64 / PPR) + lane / PPR, m = (lane % PPR) * TV;
            Vec<T> out;
#pragma unroll
            for (int i = 0; i < TV; i += 4) {
                const fv4 v = *(const fv4*)(turn + row * 32 + 4 * (((m + i) >> 2) ^ (row & 7)));
#pragma unroll
                for (int r = 0; r < 4; ++r) out.v[i + r] = (T)v[r];
            }
            const long n = CF ? 32 * ot + row : p0 + 32 * mt + row, mg = CF ? p0 + 32 * mt + m : 32 * ot + m;
            const long left = M - mg;
            if (n < (CF ? (long)a.O : a.N) && left > 0) {
                if (CF && sizeof(T) == 4) store_part<true>(yb + n * M + mg, out, left < TV ? (int)left : TV);
                else store_part(yb + n * M + mg, out, left < TV ? (int)left : TV);
            }
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
    if (p->o > 1 << 27) return fail("gnr_int8_linear: o = %d exceeds 2^27", p->o);
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

// Which kernel takes floating x as it is (FUSE_NONE: x is quantised into the workspace first), us by fused / two launches:
//   FUSE_FEW  rows that the few-rows kernel takes
//   1 2 4     int8_fused_kernel with that many 32-row tiles a workgroup
// Up to 128 outputs a workgroup multiplies with all of them: x is read once and its 8-bit rows never reach memory (262144 x 64 -> 32, fp32
// maps: 18.8 / 27.9), with as many row tiles as keep four waves busy, fewer where a row of K does not fit a thread's registers or CUs would
// be left without a workgroup (1028 x 396 -> 16, fp32: one tile 5.8, four 11.2).
// Beyond, every workgroup takes four output tiles and the rows are quantised again for each: only while there is a CU for every workgroup,
// when what counts is one launch instead of two (88 x 456 -> 1701, fp16: 6.7 / 10.4; 4096 x 258 -> 516, 640 workgroups: 11.5 / 10.1).
enum { FUSE_NONE = 0, FUSE_FEW = 8 };
static int fused_parts(long O, int nmt, int* span) {
    const long o_tiles = (O + 31) / 32;
    *span = (int)(O <= 128 ? o_tiles : 4 / nmt);
    return (int)((o_tiles + *span - 1) / *span);
}
static int int8_fuse(const GnrInt8Problem* p) {
    if (p->x_type == GNR_I8 || p->x_channels_first != p->y_channels_first) return FUSE_NONE;
    const bool cf = p->x_channels_first != 0;
    const long N = (long)p->batch * p->n_pix;
    if (!cf && p->batch == 1 && N <= FEW_FUSED && p->k <= FEW_FUSED_K) return FUSE_FEW;
    if ((!cf && p->batch != 1) || p->k > FUSED_MAX_K) return FUSE_NONE;
    const int vec = p->x_type == GNR_F32 ? 4 : 8;
    int nmt = p->o <= 32 ? 4 : (p->o <= 64 ? 2 : 1), span;
    while (cf && nmt > 1 && p->k > 32 * vec * 4 / nmt) nmt /= 2;               // maps: 4 quads of channels a thread
    while (nmt > 1 && N < 32 * 256 * nmt) nmt /= 2;                            // a workgroup for every CU first
    if (cf && p->k > 32 * vec * 4 / nmt) return FUSE_NONE;
    const long groups = cf ? p->batch * ((p->n_pix + 32 * nmt - 1) / (32 * nmt)) : (N + 32 * nmt - 1) / (32 * nmt), parts = fused_parts(p->o, nmt, &span);
    if (groups * parts * 256 >= (1L << 32)) return FUSE_NONE;                  // check_grid
    return p->o <= 128 || groups * parts <= 256 ? nmt : FUSE_NONE;
}

struct Int8Ws {
    size_t q_pitch, q_bytes, bytes;
};
static Int8Ws int8_ws(const GnrInt8Problem* p) {                     // floating x: its rows and their scales
    Int8Ws w{};
    if (p->x_type == GNR_I8 || int8_fuse(p)) return w;
    const size_t n = (size_t)p->batch * (size_t)p->n_pix;
    w.q_pitch = ((size_t)p->k + 63) & ~(size_t)63;                   // a stage of a row never crosses a line: 28672 x 516 -> 1032 41 -> 38 us
    w.q_bytes = (n * w.q_pitch + 255) & ~(size_t)255;
    w.bytes = w.q_bytes + ((n * sizeof(float) + 255) & ~(size_t)255);
    return w;
}

template <typename T, bool CF, int WM, int WN, int TM, int TN, int NST = 4> static int launch_tile(const Int8Args& a, long batch, hipStream_t st) {
    typedef TileShape<WM, WN, TM, TN, NST> S;
    const long M = CF ? a.P : a.O, N = CF ? a.O : a.N;
    const long tm = (M + S::BM - 1) / S::BM, tn = (N + S::BN - 1) / S::BN, tiles = tm * tn * (CF ? batch : 1);
    if (check_grid("gnr_int8_linear", tiles, S::NT)) return 1;
    const int stages = (a.K + 63) / 64 < NST ? (a.K + 63) / 64 : NST, ring = stages * S::STAGE;
    hipLaunchKernelGGL((int8_tile_kernel<T, CF, WM, WN, TM, TN, NST>), dim3((unsigned)tiles), dim3(S::NT), ring > S::TURN ? ring : S::TURN, st, a,
                       (unsigned)tm, (unsigned)tn);
    return 0;
}

template <typename X, typename T, bool CF, int TT> static void launch_few(const Int8Args& a, hipStream_t st) {
    const int rows = 16 * (((a.K + 63) / 64) * 64 + 16), part = 4 * TT * 64 * 16;
    hipLaunchKernelGGL((int8_few_kernel<X, T, CF, TT>), dim3((unsigned)((a.O + 15) / 16), (unsigned)((a.N + 16 * TT - 1) / (16 * TT))), dim3(256),
                       !__is_same(X, int8_t) && rows > part ? rows : part, st, a);
}

// Which kernel.  Figures: us on one card, bf16 y unless stated, rows x K -> O.
//   at most 64 rows       the few-rows kernel (1 x 2048 -> 4096: 4.4 / 10 with 64 x 64 tiles)
//   little of y           the same with blocks of 16 or 32 rows, while a CU has about one: what counts is how K is shared (150 x 1422 -> 256: 4.0 /
//                         6.5, 100 x 2048 -> 834: 6.3 / 8.0; 512 x 2048 -> 834, 848 blocks of 32: 14.8 / 8.2)
//   O <= 32, 64           tiles as narrow as the layer (262144 x 64 -> 32, fp32 maps: 8.0 against 9.0 with 64 rows a wave)
//   256 x 256 tiles       where K is long, they fill the card and few of their values fall outside: 16384 x 2048 -> 4096 144 / 202
//                         with 128 x 128 (the products alone; 141 / 188 at best), but 28672 x 516 -> 1032 (a fifth outside) 43 / 41 and 28672 x 258 -> 516 23 / 18
//   128 x 256 rows        for K as long otherwise: 28672 x 516 -> 1032 39 / 43; with few of them 8192 x 516 -> 1032 15.8 / 15.0
//   128 x 128, 64 x 64    by whether the larger fill the card (4096 x 258 -> 516, fp32: 64 x 64 6.2, 128 x 128 8.3)
template <typename T, bool CF> static int launch_int8(const Int8Args& a, long batch, hipStream_t st) {
    const long few = (a.N + 15) / 16 * ((a.O + 15) / 16), few2 = (a.N + 31) / 32 * ((a.O + 15) / 16);
    if (a.N <= FEW_MAX || few2 <= 320) {
        if (a.N <= 16 || few <= 256) launch_few<int8_t, T, CF, 1>(a, st);
        else if (a.N <= 32 || few2 <= 320) launch_few<int8_t, T, CF, 2>(a, st);
        else launch_few<int8_t, T, CF, 4>(a, st);
        return 0;
    }
    // m: outputs (y [N][O]) or pixels (y [B][O][P])
    const long M = CF ? a.P : a.O, N = CF ? a.O : a.N, B = CF ? batch : 1;
    const long t256 = ((M + 255) / 256) * ((N + 255) / 256) * B, t128 = ((M + 127) / 128) * ((N + 127) / 128) * B;
    constexpr int WM = CF ? 4 : 1, WN = CF ? 1 : 4;
    if (a.O <= 32) return launch_tile<T, CF, WM, WN, 1, 1, 3>(a, batch, st);
    if (a.O <= 64) return launch_tile<T, CF, WM, WN, CF ? 1 : 2, CF ? 2 : 1, 3>(a, batch, st);
    if (a.K >= 512 && t256 >= 256 && t256 * 65536 / 17 <= M * N * B / 16) return launch_tile<T, CF, 4, 2, 2, 4, 4>(a, batch, st);
    if constexpr (!CF)
        if (a.K >= 512 && (M + 127) / 128 * ((N + 255) / 256) >= 400) return launch_tile<T, CF, 2, 2, 2, 4, 3>(a, batch, st);
    if (t128 >= 256) return launch_tile<T, CF, 2, 2, 2, 2, 3>(a, batch, st);
    return launch_tile<T, CF, 2, 2, 1, 1, 4>(a, batch, st);
}
template <typename X, typename T, bool CF, int NMT> static void launch_fused_tile(const Int8Args& a, long batch, hipStream_t st) {
    int span;
    const long P = CF ? a.P : a.N, tiles = (P + 32 * NMT - 1) / (32 * NMT), parts = fused_parts(a.O, NMT, &span), blocks = (CF ? tiles * batch : tiles) * parts;
    hipLaunchKernelGGL((int8_fused_kernel<X, T, CF, NMT>), dim3((unsigned)blocks), dim3(256), 32 * NMT * fused_ld(a.K) + 4 * 4096, st, a, (unsigned)tiles,
                       (unsigned)parts, span);
}
template <typename X, typename T> static void launch_fused_type(const Int8Args& a, long batch, bool cf, int how, hipStream_t st) {
    if (how == FUSE_FEW) launch_few<X, T, false, 1>(a, st);
    else if (how == 1) cf ? launch_fused_tile<X, T, true, 1>(a, batch, st) : launch_fused_tile<X, T, false, 1>(a, batch, st);
    else if (how == 2) cf ? launch_fused_tile<X, T, true, 2>(a, batch, st) : launch_fused_tile<X, T, false, 2>(a, batch, st);
    else cf ? launch_fused_tile<X, T, true, 4>(a, batch, st) : launch_fused_tile<X, T, false, 4>(a, batch, st);
}
template <typename X> static void launch_fused(const Int8Args& a, int y_type, long batch, bool cf, int how, hipStream_t st) {
    if (y_type == GNR_F32) launch_fused_type<X, float>(a, batch, cf, how, st);
    else if (y_type == GNR_BF16) launch_fused_type<X, __bf16>(a, batch, cf, how, st);
    else launch_fused_type<X, _Float16>(a, batch, cf, how, st);
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
    } else if (const int how = int8_fuse(p)) {
        const bool cf = p->y_channels_first != 0;
        a.xf = p->x; a.xf_batch = p->x_batch; a.xf_pitch = p->x_stride;
        if (p->x_type == GNR_F32) launch_fused<float>(a, p->y_type, p->batch, cf, how, st);
        else if (p->x_type == GNR_BF16) launch_fused<__bf16>(a, p->y_type, p->batch, cf, how, st);
        else launch_fused<_Float16>(a, p->y_type, p->batch, cf, how, st);
        const hipError_t e = hipGetLastError();
        return e == hipSuccess ? 0 : fail("gnr_int8_linear: launch failed: %s", hipGetErrorString(e));
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
    const bool cf = p->y_channels_first != 0;
    a.flat = !a.slots && (p->batch == 1 || (a.x_batch == a.P * a.x_pitch && a.xs_batch == a.P));
    if (p->y_type == GNR_F32) rc = cf ? launch_int8<float, true>(a, p->batch, st) : launch_int8<float, false>(a, p->batch, st);
    else if (p->y_type == GNR_BF16) rc = cf ? launch_int8<__bf16, true>(a, p->batch, st) : launch_int8<__bf16, false>(a, p->batch, st);
    else rc = cf ? launch_int8<_Float16, true>(a, p->batch, st) : launch_int8<_Float16, false>(a, p->batch, st);
    if (rc) return 1;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("gnr_int8_linear: launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // extern "C"
