// HIP kernels of the descriptor heads (gfx950): matrix product with bias, activation and residual in its
// epilogue, and unit rows.
//
//   linear     y[m][n] = round(act(sum_k x[m][k] w[n][k] + b[n]) + r[m][n]),  products of fp16 / bf16 values summed in fp32
//   unit rows  y[m][c] = fp16(x[m][c] / |x[m]|),  the sum of squares in 64 bits, the norm rounded to fp32
//
// Weights are laid out once, when a layer is created, in the order the matrix instruction takes them:
//   fragment (p, s) = 1 KiB holding, for lane l and e = 0..7, w[chan(p, l & 15)][32 s + 8 (l >> 4) + e],
//   the two fragments of a 64-deep step back to back, then the next panel of 16 channels, then the next step: what a tile
//   reads for one step is one contiguous piece, and the tiles of a launch spread over all memory channels.  Zeros beyond N and K.
// A pair of panels 2u, 2u+1 covers 32 channels, interleaved so that the accumulators of the pair give every
// lane 8 CONSECUTIVE channels (16-byte fp16 stores):  chan(2u + c, 4 g + j) = 32 u + 8 g + 4 c + j.
#include <hip/hip_runtime.h>
#include <math.h>
#include "frhot_kernels.h"

namespace frhot {

typedef _Float16 half_t;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

#define FR_DEV __device__ __forceinline__

namespace {

FR_DEV void glds16(const void* g, void* lds_wave_base) {
    // 64 lanes x 16 B: lane i's bytes land at lds_wave_base + 16*i.
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

FR_DEV int xcd_remap(int bid, int n) {      // every XCD gets a contiguous run of logical tiles (blocks b and b+8 share one)
    const int q = n >> 3, r = n & 7, x = bid & 7, i = bid >> 3;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

template <bool BF>
FR_DEV float4v mfma(uint4v a, uint4v b, float4v c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

FR_DEV float load1(const void* p, size_t i, int type) {
    if (type == kF32) return ((const float*)p)[i];
    if (type == kBF16) return (float)((const __bf16*)p)[i];
    return (float)((const half_t*)p)[i];
}

FR_DEV void store1(void* p, size_t i, int type, float v) {
    if (type == kF32) ((float*)p)[i] = v;
    else if (type == kBF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((half_t*)p)[i] = (half_t)v;
}

// exp(x + lo) for x <= 0 as exp2 of the rounded product, the product's rounding put back to first order: within 3 units of
// 2^-24 of its value down to fp32's normal range (x > -87), below that zero.
FR_DEV float exp_neg(float x, float lo) {
    const float t = x * 1.44269504f;
    float r = __builtin_fmaf(x, 1.44269504f, -t);
    r = __builtin_fmaf(x, 1.92596299e-8f, r);
    r = __builtin_fmaf(lo, 1.44269504f, r);
    const float p = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(p, r * 0.693147181f, p);
}
// v / (1 + exp(-x)), from h = exp(-|x| / 2) so that nothing overflows, and far left, where the answer is v h h, not before v has met
// the first h: v exp(x) is a normal number for longer than exp(x) is.  The hardware's reciprocal is off by at most one unit.
FR_DEV float gated(float v, float x) {
    const float m = fmaxf(-fabsf(x), -400.f);
    const float t = m * 0.721347520f;
    const float r = __builtin_fmaf(m, 9.62981495e-9f, __builtin_fmaf(m, 0.721347520f, -t));
    const float p = __builtin_amdgcn_exp2f(t);
    const float h = __builtin_fmaf(p, r * 0.693147181f, p);
    const float s = x < 0.f ? h : 1.f;
    return v * s * (s * __builtin_amdgcn_rcpf(__builtin_fmaf(h, h, 1.f)));
}
// The normal distribution's function: erfc(z) = exp(-z^2) erfcx(z) with erfcx(z) = t P(t), t = 1 / (1 + z / 2), z = |v| / sqrt 2; P of
// degree 9 is a least-squares fit to scipy's erfcx over z = 0..10, reweighted towards an even relative error (2e-8; 2.9e-7 as
// evaluated in fp32).  v^2 is carried with its rounding.
FR_DEV float normal_cdf(float v) {
    constexpr float C[10] = {0.282064497f, 0.282857031f, 0.238644838f, 0.22554186f, -0.0983176306f, 0.421274275f, -0.670022488f, 0.428928405f, -0.123254694f, 0.0122838775f};
    const float a = fminf(fabsf(v), 100.f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.353553391f, 1.f));
    float p = C[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) p = __builtin_fmaf(p, t, C[i]);
    const float s = a * a, lo = __builtin_fmaf(a, a, -s);
    const float h = 0.5f * p * t * exp_neg(-0.5f * s, -0.5f * lo);      // erfc(z) / 2
    return v < 0.f ? h : 1.f - h;
}
// The activations in fp32.  Each keeps its relative accuracy as long as its value is a normal number, and NaN stays NaN (a maximum with zero would turn it into
// zero).  With the library's expf and erfcf and an IEEE division, silu / gelu / tanh gelu of 21,888 x 1568 values cost 22 / 38 / 25 us
// on top of the product; these forms 9.7 / 18.9 / 11.5 (K = 64 to fp16, 31.2 us without one).
template <int W>
FR_DEV void activate(float (&v)[W], int act) {
    if (act == kActRelu) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];
    } else if (act == kActSilu) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = gated(v[j], v[j]);
    } else if (act == kActGelu) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = v[j] * normal_cdf(v[j]);
    } else if (act == kActGeluTanh) {       // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = gated(v[j], 1.59576912f * __builtin_fmaf(0.044715f * v[j] * v[j], v[j], v[j]));
    }
}

// W elements at any address their type may have: this memory takes 16-byte accesses at such addresses, so odd widths and row
// distances need no code of their own (21,897 x 24 x 1561 to fp32: 109 us with a store per element).
template <typename T, int W> struct vect { typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T)))); };

// W consecutive channels n .. n+W-1 of row m: bias, activation, residual.
template <int W>
FR_DEV void load_bias(const float* __restrict__ bias, int n, float (&b)[W]) {      // (padded with zeros to whole panels)
#pragma unroll
    for (int j = 0; j < W; j += 4) {
        const float4v t = *(const float4v*)(bias + n + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[j + i] = t[i];
    }
}
template <int W>
FR_DEV void epilogue(const LinearOut& o, const float (&b)[W], size_t m, int n, float (&v)[W]) {
    const float c = o.scale ? o.scale[m] : 1.f;     // (a power of two: the product is exact)
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = __builtin_fmaf(v[j], c, b[j]);
    activate<W>(v, o.act);
    if (o.res) {
        const size_t at = m * (size_t)o.ldr + n;
        if (n + W <= o.N) {
            if (o.rtype == kF32) {
                const auto r = *(const typename vect<float, W>::type*)((const float*)o.res + at);
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] += r[j];
            } else if (o.rtype == kBF16) {
                const auto r = *(const typename vect<__bf16, W>::type*)((const __bf16*)o.res + at);
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] += (float)r[j];
            } else {
                const auto r = *(const typename vect<half_t, W>::type*)((const half_t*)o.res + at);
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] += (float)r[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (n + j < o.N) v[j] += load1(o.res, at + j, o.rtype);
        }
    }
}

// The same, then ONE rounding and the store.  Columns from N on are not written.
template <int W>
FR_DEV void finish(const LinearOut& o, const float (&b)[W], size_t m, int n, float (&v)[W]) {
    if (n >= o.N) return;
    epilogue<W>(o, b, m, n, v);
    const size_t at = m * (size_t)o.ldo + n;
    if (n + W <= o.N) {
        if (o.otype == kF32) {
#pragma unroll
            for (int j = 0; j < W; j += 4) *(typename vect<float, 4>::type*)((float*)o.out + at + j) = typename vect<float, 4>::type{v[j], v[j + 1], v[j + 2], v[j + 3]};
        } else if (o.otype == kBF16) {
            typename vect<__bf16, W>::type t;
#pragma unroll
            for (int j = 0; j < W; ++j) t[j] = (__bf16)v[j];
            *(typename vect<__bf16, W>::type*)((__bf16*)o.out + at) = t;
        } else {
            typename vect<half_t, W>::type t;
#pragma unroll
            for (int j = 0; j < W; ++j) t[j] = (half_t)v[j];
            *(typename vect<half_t, W>::type*)((half_t*)o.out + at) = t;
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (n + j < o.N) store1(o.out, at + j, o.otype, v[j]);
    }
}

// Elements k0 .. k0+7 of a row of K at any address, zeros from the K-th on (nothing outside the row is read): where the row ends
// inside or in front of them, the row's last eight are loaded and shifted down.
FR_DEV uint4v load_chunk(const uint16_t* row, int k0, int K) {
    if (K < 8) {
        uint4v o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned lo = k0 + 2 * e < K ? row[k0 + 2 * e] : 0u, hi = k0 + 2 * e + 1 < K ? row[k0 + 2 * e + 1] : 0u;
            o[e] = lo | (hi << 16);
        }
        return o;
    }
    typedef unsigned long long ulong2v __attribute__((ext_vector_type(2)));
    const int at = min(k0, K - 8), b = (k0 - at) * 16;         // (b: 0 .. 16 * (k0 - K + 8))
    const ulong2v v = __builtin_bit_cast(ulong2v, *(const vect<uint16_t, 8>::type*)(row + at));
    ulong2v o;
    o[0] = b == 0 ? v[0] : b < 64 ? (v[0] >> (b & 63)) | (v[1] << (64 - b & 63)) : b < 128 ? v[1] >> (b & 63) : 0ull;
    o[1] = b < 64 ? v[1] >> (b & 63) : 0ull;
    return __builtin_bit_cast(uint4v, o);
}

// w [N][K] -> fragments (see the head of the file); thread = one lane's 16 bytes of one fragment
__global__ __launch_bounds__(256) void linear_layout_kernel(const uint16_t* __restrict__ w, uint16_t* __restrict__ wt, int N, int K,
                                                            int panels, int ksteps) {
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)panels * ksteps * 64) return;
    const int lane = (int)(t & 63);
    const int kk = (int)(t >> 6) & 1, p = (int)((t >> 7) % panels), s = (int)((t >> 7) / panels) * 2 + kk;
    const int r = lane & 15;
    const int ch = (p >> 1) * 32 + (r >> 2) * 8 + (p & 1) * 4 + (r & 3);
    const int k0 = s * 32 + (lane >> 4) * 8;
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (ch < N && k0 + e < K) ? w[(size_t)ch * K + k0 + e] : (uint16_t)0;
    uint4v o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (unsigned)v[2 * e] | ((unsigned)v[2 * e + 1] << 16);
    *(uint4v*)(wt + t * 8) = o;
}

// Rows whose addresses LDS-DMA cannot take (odd strides, K not a multiple of 8), brought into rows of `kpad` elements with zeros
// behind the K-th: where a wide layer would read them many times (plan_linear).  Bound by its bytes, 4.5 TB/s in cache.
__global__ __launch_bounds__(256) void linear_pack_kernel(const uint16_t* __restrict__ x, int64_t ldx, int K, int kpad,
                                                          uint16_t* __restrict__ out, int rows) {
    const int per_row = kpad >> 3;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)rows * per_row) return;
    const int r = (int)(t / per_row), k0 = (int)(t % per_row) * 8;
    *(uint4v*)(out + t * 8) = load_chunk(x + (size_t)r * ldx, k0, K);
}

// The rows between two layers of a head.  Their values are fp32 and the matrix instruction takes fp16 (its fp32 form runs at a
// sixteenth of the rate): each value goes in as the sum of two fp16 numbers, hi the value rounded and lo what that left, so the next
// layer is one product of twice the depth.  Its weights are laid out twice in a row for that; going round in one copy inside the
// products' loops cost a call of one row 0.2 of 6.1 us.  A row is first brought by a power of two to a largest finite value in
// 2^14 .. 2^15, which fp16 holds whatever the row's own range; the epilogue takes the power back.  Lost is half a step of lo: 2^-23 of
// the value at most, or 2^-39 of the row's largest where that is more.  (The power stops at 2^126, where that is less than half of
// fp32's smallest number.)  Infinities and NaN stay what they are in hi, with nothing in lo.
// A wave takes a row; rows of up to 512 R values are read once.  2011 x 1024: 5.6 us, mostly the launch.  With fp16 inner rows the whole
// of 2011 x 4096 -> 1024 -> 512 took 40.5 us and was 2.9e-4 off its 64-bit value (2-norm), with pairs 48.6 us and 2.1e-4, which is the
// unit rows' own rounding.
template <int R>
__global__ __launch_bounds__(256) void linear_split_kernel(const float* __restrict__ x, int64_t ldx, int N, int kpad,
                                                           half_t* __restrict__ out, float* __restrict__ scale, int rows) {
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= rows) return;
    const float* const row = x + (size_t)m * ldx;
    half_t* const o = out + (size_t)m * 2 * kpad;
    float v[R ? R : 1][8];
    float most = 0.f;
    auto load = [&](int c, float (&t)[8]) __attribute__((always_inline)) {
        const float4v a = *(const float4v*)(row + c), b = *(const float4v*)(row + c + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = c + j < N ? (j < 4 ? a[j & 3] : b[j & 3]) : 0.f;
    };
    auto largest = [&](const float (&t)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = fabsf(t[j]);
            if (f <= 3.402823466e38f) most = fmaxf(most, f);
        }
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * 512 + lane * 8 < kpad) { load(i * 512 + lane * 8, v[i]); largest(v[i]); }
    } else {
        for (int c = lane * 8; c < kpad; c += 512) { load(c, v[0]); largest(v[0]); }
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor(most, s));
    int e = 0;
    (void)frexpf(most, &e);                                         // most = f 2^e, f in [1/2, 1)
    const int up = most > 0.f ? min(15 - e, 126) : 0;
    const float by = ldexpf(1.f, up);
    if (lane == 0) scale[m] = ldexpf(1.f, -up);
    auto store = [&](int c, const float (&t)[8]) __attribute__((always_inline)) {
        half8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = t[j] * by;
            hi[j] = (half_t)f;
            lo[j] = fabsf(f) <= 3.402823466e38f ? (half_t)(f - (float)hi[j]) : (half_t)0.f;
        }
        *(half8*)(o + c) = hi;
        *(half8*)(o + kpad + c) = lo;
    };
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * 512 + lane * 8 < kpad) store(i * 512 + lane * 8, v[i]);
    } else {
        for (int c = lane * 8; c < kpad; c += 512) { load(c, v[0]); store(c, v[0]); }
    }
}

// The tile kernel: TM x TN of y (or of a K slice's partial sums) at a time, 64 K-elements per step.  X and W stages arrive by
// 16-byte LDS-DMA in rings of XS and WS stages, loads running XS-1 and WS-1 steps ahead, waited for with counted vmcnt so that
// the newest stages stay in flight across the step's one barrier.  X rows are 128 bytes in LDS, 16-byte chunk c of row
// r at position c ^ (r & 7) (applied to the source address, undone at the read); weight fragments lie as in memory and are
// read linearly: neither read has a bank conflict.  Waves WX x WY, each (TM/WX) x (TN/WY).  A step's MFMAs go in four units
// (32-deep half kk, half of the rows xh); a unit's fragments are read while the one before it computes, and the last unit of
// a step computes behind the barrier, under the next step's first reads.
// GATHER: rows that LDS-DMA cannot take go through registers, loaded one step before they are put into their stage.
// 65536 x 512 x 4096 with relu to fp32: 246 us, 1,118 TFLOP/s (1,420 is what a large library product reaches here); the matrix cores
// are busy 0.54 of the time, and a step's LDS traffic (192 KiB of fragments, 64 KiB of LDS-DMA) takes about as long as its MFMAs.  Four
// waves of 128 x 128 read a third less of it and took 293 us where eight took 267.
// Behind the last step the stages are free: every wave brings its accumulators through a part of them that is its own, half of
// its rows at a time, and finishes them row by row, eight consecutive channels a lane (whole cache lines per store, and one
// copy of the epilogue's code instead of one per accumulator).
template <bool BF, int TM, int TN, int WX, int WY, int XS, int WS>
struct TileCore {
    static constexpr int NW = WX * WY, TX = TM / WX, TY = TN / WY, NX = TX / 16, NY = TY / 16, NXH = NX / 2;
    static constexpr int XB = TM * 128, WB = TN * 128, LDS = XS * XB + WS * WB;
    static constexpr int NPX = TM / 8 / NW, NPW = TN / 8 / NW;
    static constexpr int DX = XS - 1, DW = WS - 1;
    // loads that may still be in flight when the next step's stages must have landed (issue order: W, then X)
    static constexpr int KEEP = DX == DW ? (DX - 1) * (NPX + NPW) : NPX;
    static_assert(TM % (8 * NW) == 0 && TN % (8 * NW) == 0 && TX % 32 == 0 && TY % 32 == 0, "tile shape");
    static_assert((DX == DW || (DX == 2 && DW == 1)) && KEEP <= 63 && LDS <= 163840, "ring shape");
    // the wave's part of LDS at the end: HR rows of TY fp32 values, 16 bytes of padding a row (no bank conflict)
    static constexpr int HR = TX / 2 > 64 ? 64 : TX / 2, ER = TY + 4;
    static_assert(NW * HR * ER * 4 <= LDS && HR % 16 == 0, "room for the epilogue");

    float4v acc[NY][NX];
    uint4v fw[2][NY], fx[2][NXH];

    FR_DEV void zero() {
#pragma unroll
        for (int y = 0; y < NY; ++y)
#pragma unroll
            for (int x = 0; x < NX; ++x) acc[y][x] = float4v{0.f, 0.f, 0.f, 0.f};
    }
    template <int U>
    FR_DEV void read(const char* xb, const char* wb, int lane, int wx, int wy) {
        constexpr int kk = U >> 1, xh = U & 1;
        const int coff = ((kk * 4 + (lane >> 4)) ^ (lane & 7)) << 4;
        if (xh == 0) {
#pragma unroll
            for (int y = 0; y < NY; ++y) fw[kk][y] = *(const uint4v*)(wb + ((wy * NY + y) * 2 + kk) * 1024 + lane * 16);
        }
#pragma unroll
        for (int x = 0; x < NXH; ++x) fx[xh][x] = *(const uint4v*)(xb + (wx * TX + (xh * NXH + x) * 16 + (lane & 15)) * 128 + coff);
    }
    template <int U>
    FR_DEV void mma() {
        constexpr int kk = U >> 1, xh = U & 1;
#pragma unroll
        for (int y = 0; y < NY; ++y)
#pragma unroll
            for (int x = 0; x < NXH; ++x) acc[y][xh * NXH + x] = mfma<BF>(fw[kk][y], fx[xh][x], acc[y][xh * NXH + x]);
    }
    FR_DEV static void wait_keep() {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(KEEP) : "memory");
    }
    FR_DEV static void wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
};

template <bool BF, int TM, int TN, int WX, int WY, int XS, int WS, bool GATHER>
__global__ __launch_bounds__(64 * WX * WY) void linear_tile_kernel(LinearIn a, LinearOut o) {
    using Core = TileCore<BF, TM, TN, WX, WY, XS, WS>;
    constexpr int NW = Core::NW, NPX = Core::NPX, NPW = Core::NPW, NY = Core::NY;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const xs = smem;
    char* const ws = smem + XS * Core::XB;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wx = wave / WY, wy = wave % WY;
    const int l15 = lane & 15, g0 = lane >> 4;

    const int tiles = a.mtiles * a.ntiles;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int z = id / tiles, t = id % tiles;
    const int m0 = (a.m_fast ? t % a.mtiles : t / a.ntiles) * TM, n0 = (a.m_fast ? t / a.mtiles : t % a.ntiles) * TN;
    const int k_lo = z * a.ksteps_per_split, S = min(a.ksteps, k_lo + a.ksteps_per_split) - k_lo;

    const int c = (lane & 7) ^ (lane >> 3);             // the 16-byte chunk this lane fetches of its row
    const char* xp[NPX];
#pragma unroll
    for (int i = 0; i < NPX; ++i) {
        int m = m0 + 8 * (wave + NW * i) + (lane >> 3);
        m = m < a.M ? m : a.M - 1;
        xp[i] = (const char*)a.x + (a.tiled ? (size_t)(m >> 8) * a.xtile + (size_t)(m & 255) * 128 : (size_t)m * a.ldx * 2) + c * 16 +
                (size_t)k_lo * a.xstep;
    }
    const int wpanel = n0 >> 4;
    int xk = k_lo, wk = k_lo;                           // what the next issue brings
    uint4v gx[GATHER ? NPX : 1];                        // GATHER: a stage of X on its way through registers
    auto next_x = [&](int slot) __attribute__((always_inline)) {
        char* const st = xs + slot * Core::XB;
        if (xk * 64 + 64 <= a.K) {
#pragma unroll
            for (int i = 0; i < NPX; ++i) {
                if constexpr (GATHER) gx[i] = __builtin_bit_cast(uint4v, *(const typename vect<uint16_t, 8>::type*)xp[i]);
                else glds16(xp[i], st + (wave + NW * i) * 1024);
                xp[i] += a.xstep;
            }
        } else if constexpr (GATHER) {
#pragma unroll
            for (int i = 0; i < NPX; ++i) gx[i] = load_chunk((const uint16_t*)xp[i] - xk * 64 - c * 8, xk * 64 + c * 8, a.K);
        } else {                                        // chunks behind the K-th element: zeros (K is a multiple of 8 here)
            const bool tail = xk * 64 + c * 8 >= a.K;
#pragma unroll
            for (int i = 0; i < NPX; ++i) glds16(tail ? (const char*)a.zeros + c * 16 : xp[i], st + (wave + NW * i) * 1024);
        }
        ++xk;
    };
    // What is counted by vmcnt stays in the order written: loads into registers are not moved across.
    auto order = [&]() __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto put_x = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NPX; ++i) *(uint4v*)(xs + slot * Core::XB + (wave + NW * i) * 1024 + lane * 16) = gx[i];
    };
    auto next_w = [&](int slot) {
        char* const st = ws + slot * Core::WB;
#pragma unroll
        for (int i = 0; i < NPW; ++i) {
            const int piece = wave + NW * i;
            const int p = min(wpanel + (piece >> 1), a.panels - 1);     // (columns beyond N: computed from the last panel and dropped)
            const char* src = (const char*)a.wt + ((size_t)wk * a.panels + p) * 2048 + (piece & 1) * 1024;
            glds16(src + lane * 16, st + piece * 1024);
        }
        ++wk;
    };

    Core core;
    core.zero();
    // prologue: stages 0 .. D-1
    if constexpr (GATHER) {
        next_w(0);
        if (Core::DW > 1 && S > 1) next_w(1);
        next_x(0);
        put_x(0);
        if (S > 1) next_x(1);                           // (put into its stage by the first step)
        Core::wait_all();
        __builtin_amdgcn_s_waitcnt(0xC07F);             // lgkmcnt(0)
    } else if constexpr (Core::DX == Core::DW) {
        for (int d = 0; d < Core::DX; ++d)
            if (d < S) { next_w(d); next_x(d); }
        if (S >= Core::DX) Core::wait_keep(); else Core::wait_all();
    } else {
        next_w(0);
        next_x(0);
        if (S > 1) { next_x(1); Core::wait_keep(); } else { Core::wait_all(); }
    }
    __builtin_amdgcn_s_barrier();

    int xslot = 0, wslot = 0;
    auto fence = [&]() __attribute__((always_inline)) { __builtin_amdgcn_sched_barrier(0); };
    auto reads_done = [&]() __attribute__((always_inline)) {
        fence(); __builtin_amdgcn_s_waitcnt(0xC07F); fence();       // lgkmcnt(0)
    };
    for (int s = 0; s < S; ++s) {
        const char* const xb = xs + xslot * Core::XB;
        const char* const wb = ws + wslot * Core::WB;
        core.template read<0>(xb, wb, lane, wx, wy);
        fence();
        if (s > 0) {
            core.template mma<3>();
            fence();
        }
        // the stages that the barrier behind the previous step has freed
        if (s + Core::DW < S) next_w(wslot == 0 ? WS - 1 : wslot - 1);
        if constexpr (GATHER) {
            order();
            if (s + 1 < S) put_x(xslot == XS - 1 ? 0 : xslot + 1);
        }
        if (s + Core::DX < S) next_x(xslot == 0 ? XS - 1 : xslot - 1);
        reads_done();
        core.template read<1>(xb, wb, lane, wx, wy);
        fence();
        core.template mma<0>();
        reads_done();
        core.template read<2>(xb, wb, lane, wx, wy);
        fence();
        core.template mma<1>();
        reads_done();
        core.template read<3>(xb, wb, lane, wx, wy);
        fence();
        core.template mma<2>();
        reads_done();       // every read of this step's stages has returned: they may be refilled behind the barrier
        if (s + Core::DX < S) Core::wait_keep(); else Core::wait_all();
        __builtin_amdgcn_s_barrier();
        fence();
        xslot = xslot == XS - 1 ? 0 : xslot + 1;
        wslot = wslot == WS - 1 ? 0 : wslot + 1;
    }
    core.template mma<3>();

    // (all stages have been read by all waves: the barrier above)
    constexpr int HR = Core::HR, ER = Core::ER, LR = Core::TY / 8, RI = 64 / LR;    // LR lanes a row, RI rows an iteration
    float* const eb = (float*)smem + wave * HR * ER;
    const int n = n0 + wy * Core::TY + (lane % LR) * 8;
    float bv[8];
    load_bias<8>(a.bias, n < a.npad ? n : 0, bv);
#pragma unroll
    for (int h = 0; h < Core::TX / HR; ++h) {
#pragma unroll
        for (int x = 0; x < HR / 16; ++x)
#pragma unroll
            for (int y = 0; y < NY; ++y)
                *(float4v*)(eb + (x * 16 + l15) * ER + (y >> 1) * 32 + g0 * 8 + (y & 1) * 4) = core.acc[y][h * (HR / 16) + x];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int r = lane / LR; r < HR; r += RI) {
            const int m = m0 + wx * Core::TX + h * HR + r;
            const float4v v0 = *(const float4v*)(eb + r * ER + (lane % LR) * 8), v1 = *(const float4v*)(eb + r * ER + (lane % LR) * 8 + 4);
            if (m >= a.M || n >= a.npad) continue;
            if (a.slab) {
                float* d = a.slab + ((size_t)z * a.M + m) * a.npad + n;
                *(float4v*)d = v0;
                *(float4v*)(d + 4) = v1;
            } else {
                float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                finish<8>(o, bv, m, n, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The wave kernel, for calls of few tiles: a block is one 16 FX x 16 FW tile, and its NW waves share out K, 64 elements at a
// time in turn.  Each wave multiplies its own slices of both operands for the whole tile, with a pipeline of its own: every
// byte enters the CU once, as it would with a shared stage, but no wave ever waits for another until the sums are joined, in
// wave order, through LDS.  Weight fragments (1 KiB of consecutive bytes) are loaded straight into registers; X goes through
// LDS by LDS-DMA, eight rows of 128 bytes an instruction: in fragment order consecutive lanes read different rows, which the
// load path serves 16 bytes a clock (38 GB/s per CU measured, against 110-145 for whole lines).
// What bounds it is the CU's load path: 256 x 4096 x 4096 moves 1 MiB into every CU in 14 us, 74 GB/s; one row of 4096 to 512 channels
// takes 6.1 us on 16 CUs, an empty launch 3.9.  Deeper rings for the weights changed neither.
// GATHER: rows that LDS-DMA cannot take (not 16-byte aligned, K not a multiple of 8) go through registers into the stage, whole lines
// of a row by consecutive lanes as well (41 x 429 x 3647: 7.6 us, 16 in fragment order straight into registers).
template <int FX, int FW, int NW, int ST>
struct WaveShape {
    static constexpr int TM = 16 * FX, TN = 16 * FW, ER = TN + 4;
    static constexpr int XB = TM * 128, STAGES = NW * ST * XB, PART = NW * TM * ER * 4;
    static constexpr int LDS = STAGES > PART ? STAGES : PART;
    static_assert(LDS <= 163840 && (ST - 1) * 2 * (FX + FW) <= 63, "stages");
};
template <bool BF, int FX, int FW, int NW, int ST, bool GATHER>
__global__ __launch_bounds__(64 * NW) void linear_wave_kernel(LinearIn a, LinearOut o) {
    using Shape = WaveShape<FX, FW, NW, ST>;
    constexpr int TM = Shape::TM, TN = Shape::TN, ER = Shape::ER;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l15 = lane & 15, g0 = lane >> 4;
    const int tiles = a.mtiles * a.ntiles;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int z = id / tiles, t = id % tiles;
    const int m0 = (a.m_fast ? t % a.mtiles : t / a.ntiles) * TM, n0 = (a.m_fast ? t / a.mtiles : t % a.ntiles) * TN;
    const int k_lo = z * a.ksteps_per_split, k_hi = min(a.ksteps, k_lo + a.ksteps_per_split);

    const char* wp[FW];
#pragma unroll
    for (int y = 0; y < FW; ++y) wp[y] = (const char*)a.wt + (size_t)min((n0 >> 4) + y, a.panels - 1) * 2048 + lane * 16;
    const size_t wstep = (size_t)a.panels * 2048;
    auto row_at = [&](int r) __attribute__((always_inline)) {
        int m = m0 + r;
        m = m < a.M ? m : a.M - 1;
        return (const char*)a.x + (a.tiled ? (size_t)(m >> 8) * a.xtile + (size_t)(m & 255) * 128 : (size_t)m * a.ldx * 2);
    };
    float4v acc[FW][FX];
#pragma unroll
    for (int y = 0; y < FW; ++y)
#pragma unroll
        for (int x = 0; x < FX; ++x) acc[y][x] = float4v{0.f, 0.f, 0.f, 0.f};

    char* const st0 = smem + wave * ((GATHER ? 1 : ST) * Shape::XB);
    const int c = (lane & 7) ^ (lane >> 3);             // the 16-byte chunk this lane fetches of its row
    const char* xp[2 * FX];
#pragma unroll
    for (int i = 0; i < 2 * FX; ++i) xp[i] = row_at(8 * i + (lane >> 3)) + c * 16;
    const char* const zeros = (const char*)a.zeros + c * 16;
    uint4v bw[GATHER ? 2 : ST][2][FW], bx[2 * FX];
    // slice i -> X stage p (GATHER: registers) and weight registers
    auto issue = [&](int i, int p, uint4v (&vw)[2][FW]) __attribute__((always_inline)) {
        const int ks = k_lo + wave + NW * i;
        char* const st = st0 + p * Shape::XB;
        if constexpr (GATHER) {
#pragma unroll
            for (int x = 0; x < 2 * FX; ++x) bx[x] = __builtin_bit_cast(uint4v, *(const typename vect<uint16_t, 8>::type*)(xp[x] + ks * 128));
        } else if (ks * 64 + 64 <= a.K) {
#pragma unroll
            for (int x = 0; x < 2 * FX; ++x) glds16(xp[x] + (size_t)ks * a.xstep, st + x * 1024);
        } else {                                        // chunks behind the K-th element: zeros (K is a multiple of 8 here)
            const bool tail = ks * 64 + c * 8 >= a.K;
#pragma unroll
            for (int x = 0; x < 2 * FX; ++x) glds16(tail ? zeros : xp[x] + (size_t)ks * a.xstep, st + x * 1024);
        }
#pragma unroll
        for (int y = 0; y < FW; ++y)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) vw[kk][y] = *(const uint4v*)(wp[y] + (size_t)ks * wstep + kk * 1024);
    };
    auto mma = [&](int p, const uint4v (&vw)[2][FW]) __attribute__((always_inline)) {
        const char* const st = st0 + p * Shape::XB;
        uint4v vx[2][FX];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int x = 0; x < FX; ++x)
                vx[kk][x] = *(const uint4v*)(st + (x * 16 + l15) * 128 + (((kk * 4 + g0) ^ (lane & 7)) << 4));
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xC07F);             // lgkmcnt(0): the stage has been read and may be refilled
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int x = 0; x < FX; ++x)
#pragma unroll
                for (int y = 0; y < FW; ++y) acc[y][x] = mfma<BF>(vw[kk][y], vx[kk][x], acc[y][x]);
        __builtin_amdgcn_sched_barrier(0);
    };
    const int slices = (k_hi - k_lo - wave + NW - 1) / NW;  // of this wave: k_lo + wave, + NW, ...
    int i = 0;
    if constexpr (GATHER) {
        // The slice after next comes into registers while one is multiplied; the slice that the row ends in is the last, by itself.
        auto fence = [&]() __attribute__((always_inline)) { asm volatile("" ::: "memory"); __builtin_amdgcn_wave_barrier(); };
        auto put = [&]() __attribute__((always_inline)) {   // (the stage is the wave's own: no other wave reads it)
#pragma unroll
            for (int x = 0; x < 2 * FX; ++x) *(uint4v*)(st0 + x * 1024 + lane * 16) = bx[x];
            fence();
        };
        const bool cut = slices > 0 && (k_lo + wave + NW * (slices - 1)) * 64 + 64 > a.K;
        const int n = cut ? slices - 1 : slices;
        if (n > 0) issue(0, 0, bw[0]);
        for (; i + 3 <= n; i += 2) {                    // nothing in here branches: the compiler can count what is in flight
            put();
            issue(i + 1, 0, bw[1]);
            mma(0, bw[0]);
            put();
            issue(i + 2, 0, bw[0]);
            mma(0, bw[1]);
        }
        if (i < n) {
            put();
            if (i + 1 < n) issue(i + 1, 0, bw[1]);
            mma(0, bw[0]);
            if (i + 1 < n) {
                put();
                mma(0, bw[1]);
            }
        }
        if (cut) {
            const int ks = k_lo + wave + NW * n;
#pragma unroll
            for (int y = 0; y < FW; ++y)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) bw[0][kk][y] = *(const uint4v*)(wp[y] + (size_t)ks * wstep + kk * 1024);
#pragma unroll 1
            for (int x = 0; x < 2 * FX; ++x)
                *(uint4v*)(st0 + x * 1024 + lane * 16) = load_chunk((const uint16_t*)row_at(8 * x + (lane >> 3)), ks * 64 + c * 8, a.K);
            fence();
            mma(0, bw[0]);
        }
    } else {
        const int n = slices;
#pragma unroll
        for (int p = 0; p < ST - 1; ++p)
            if (p < n) issue(p, p, bw[p]);
        for (; i + 2 * ST - 1 <= n; i += ST) {          // nothing in here branches: the compiler can count what is in flight
#pragma unroll
            for (int p = 0; p < ST; ++p) {
                issue(i + p + ST - 1, (p + ST - 1) % ST, bw[(p + ST - 1) % ST]);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * 2 * (FX + FW)) : "memory");
                mma(p, bw[p]);
            }
        }
#pragma unroll
        for (int q = 0; q < 2 * ST - 2; ++q) {
            if (i + q < n) {
                if (i + q + ST - 1 < n) {
                    issue(i + q + ST - 1, (q + ST - 1) % ST, bw[(q + ST - 1) % ST]);
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * 2 * (FX + FW)) : "memory");
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                }
                mma(q % ST, bw[q % ST]);
            }
        }
    }
    __syncthreads();                                    // the sums take the stages' place

    float* const part = (float*)smem;
    float* const mine = part + wave * TM * ER;
#pragma unroll
    for (int x = 0; x < FX; ++x)
#pragma unroll
        for (int y = 0; y < FW; ++y) *(float4v*)(mine + (x * 16 + l15) * ER + (y >> 1) * 32 + g0 * 8 + (y & 1) * 4) = acc[y][x];
    __syncthreads();
    for (int i = tid; i < TM * (TN / 8); i += 64 * NW) {
        const int r = i / (TN / 8), m = m0 + r, cn = (i % (TN / 8)) * 8, ch = n0 + cn;
        if (m >= a.M || ch >= a.npad) continue;
        float bv[8], v[8] = {};
        load_bias<8>(a.bias, ch, bv);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* p = part + w * TM * ER + r * ER + cn;
            const float4v p0 = *(const float4v*)p, p1 = *(const float4v*)(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] += p0[j]; v[4 + j] += p1[j]; }
        }
        if (a.slab) {
            float* d = a.slab + ((size_t)z * a.M + m) * a.npad + ch;
            *(float4v*)d = float4v{v[0], v[1], v[2], v[3]};
            *(float4v*)(d + 4) = float4v{v[4], v[5], v[6], v[7]};
        } else {
            finish<8>(o, bv, m, ch, v);
        }
    }
}

// Joins the K slices in slice order and finishes the rows; thread = 8 channels of one row.
__global__ __launch_bounds__(256) void linear_join_kernel(LinearIn a, LinearOut o, int splits) {
    const int per_row = a.npad >> 3;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)a.M * per_row) return;
    const int m = (int)(t / per_row), n = (int)(t % per_row) * 8;
    float bv[8], v[8] = {};
    load_bias<8>(a.bias, n, bv);
    const float* p = a.slab + (size_t)m * a.npad + n;
    const size_t step = (size_t)a.M * a.npad;
    for (int z = 0; z < splits; z += 4) {           // four slices in flight, added in slice order
        float4v q[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (z + i < splits) { q[i][0] = *(const float4v*)(p + (z + i) * step); q[i][1] = *(const float4v*)(p + (z + i) * step + 4); }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (z + i < splits) {
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[j] += q[i][0][j]; v[4 + j] += q[i][1][j]; }
            }
    }
    finish<8>(o, bv, m, n, v);
}

// ------------------------------------------------------------- unit rows ---
// The norm comes from a 64-bit sum of squares rounded to fp32, then one IEEE division per element: the stored row is the same
// whatever the summation order, and the same as the library's own upload makes of it (gallery_upsert_kernel).  A row
// shorter than 1e-30 is divided by one.
// Bound by HBM: 262144 x 512 fp32, 805 MB, 135-140 us = 5.8 TB/s (with a second read of x in place of registers 347).
// L lanes a row, each R vectors of V consecutive elements (16 bytes, at any address) in registers: x is read once.  R = 0: rows too
// long for that are read twice, the second time out of the cache.
// TAIL: V does not divide the row.  Its last vector then begins at N - V and shares elements with the one before it: they count once
// in the sum and are stored twice, with the same value (1,375,152 rows of 22 fp16: 44 us element by element).  Rows shorter than V
// go element by element.
template <typename T, int V, bool TAIL>
FR_DEV void load_row(const T* row, int c, int N, float (&v)[V]) {
    if (!TAIL || N >= V) {
        const auto t = *(const typename vect<T, V>::type*)(row + (TAIL ? min(c, N - V) : c));
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < N ? (float)row[j] : 0.f;
    }
}
template <int V, bool TAIL>
FR_DEV void add_squares(double& ss, int c, int N, const float (&v)[V]) {
    const int shared = TAIL && N >= V ? max(0, c + V - N) : 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (!TAIL || j >= shared) ss += (double)v[j] * (double)v[j];
}
template <int V, bool TAIL>
FR_DEV void store_unit(const UnitOut& o, int N, int m, int c, const float (&v)[V], float nrm) {
    half_t* d;
    if (o.gallery) {                        // (N is a multiple of 64 here)
        const int64_t r = o.row0 + m;       // (the order of a gallery's rows in memory: see gal_index)
        d = (half_t*)o.out + ((((size_t)(r >> 8) * (N >> 6) + (c >> 6)) << 8) + (r & 255)) * 64 + (c & 63);
    } else {
        d = (half_t*)o.out + (size_t)m * o.ldo + (TAIL && N >= V ? min(c, N - V) : c);
    }
    half_t t[V];
#pragma unroll
    for (int j = 0; j < V; ++j) t[j] = (half_t)__fdiv_rn(v[j], nrm);
    if (!TAIL || N >= V) {
        typename vect<half_t, V>::type u;
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = t[j];
        *(typename vect<half_t, V>::type*)d = u;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < N) d[j] = t[j];
    }
}
template <typename T, int L, int R, bool TAIL>
__global__ __launch_bounds__(256) void unit_rows_kernel(const T* __restrict__ x, int64_t ldx, int M, int N, UnitOut o) {
    constexpr int V = 16 / sizeof(T), RB = 256 / L;             // RB rows a block
    const int m = blockIdx.x * RB + threadIdx.x / L, l = threadIdx.x % L;
    if (m >= M) return;                     // (the lanes of a row leave together)
    const T* const row = x + (size_t)m * ldx;
    double ss = 0.0;
    float v[R ? R : 1][V];
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * L + l) * V;
            if (c < N) load_row<T, V, TAIL>(row, c, N, v[i]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * L + l) * V;
            if (c < N) add_squares<V, TAIL>(ss, c, N, v[i]);
        }
    } else {
        for (int c = l * V; c < N; c += L * V) {
            load_row<T, V, TAIL>(row, c, N, v[0]);
            add_squares<V, TAIL>(ss, c, N, v[0]);
        }
    }
#pragma unroll
    for (int s = L / 2; s > 0; s >>= 1) ss += __shfl_xor(ss, s);
    float nrm = (float)sqrt(ss);
    nrm = nrm < 1e-30f ? 1.0f : nrm;
    if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int c = (i * L + l) * V;
            if (c < N) store_unit<V, TAIL>(o, N, m, c, v[i], nrm);
        }
    } else {
        for (int c = l * V; c < N; c += L * V) {
            load_row<T, V, TAIL>(row, c, N, v[0]);
            store_unit<V, TAIL>(o, N, m, c, v[0], nrm);
        }
    }
    if (l == 0 && o.keys_dst) o.keys_dst[o.row0 + m] = o.keys_src[o.row0 + m];
}

constexpr int64_t kRunRows = 1 << 22;       // rows of one launch

template <typename T, int L, int R>
hipError_t launch_unit(const void* x, int64_t ldx, int64_t M, int N, const UnitOut& o, hipStream_t s) {
    const int64_t rb = 256 / L;
    const auto kern = N % (16 / (int)sizeof(T)) ? unit_rows_kernel<T, L, R, true> : unit_rows_kernel<T, L, R, false>;
    for (int64_t m0 = 0; m0 < M; m0 += kRunRows) {
        const int64_t n = M - m0 < kRunRows ? M - m0 : kRunRows;
        UnitOut u = o;
        if (o.gallery) u.row0 = o.row0 + m0;
        else u.out = (half_t*)o.out + (size_t)m0 * o.ldo;
        hipLaunchKernelGGL(kern, dim3((unsigned)((n + rb - 1) / rb)), dim3(256), 0, s, (const T*)x + (size_t)m0 * ldx, ldx, (int)n, N, u);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
template <typename T>
hipError_t unit_by_width(const void* x, int64_t ldx, int64_t M, int N, const UnitOut& o, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (N <= 16 * V) return launch_unit<T, 4, 4>(x, ldx, M, N, o, s);
    if (N <= 64 * V) return launch_unit<T, 16, 4>(x, ldx, M, N, o, s);
    if (N <= 256 * V) return launch_unit<T, 64, 4>(x, ldx, M, N, o, s);
    if (N <= 1024 * V) return launch_unit<T, 64, 16>(x, ldx, M, N, o, s);
    return launch_unit<T, 64, 0>(x, ldx, M, N, o, s);
}

template <bool BF, int TM, int TN, int WX, int WY, int XS, int WS>
hipError_t launch_tile(LinearIn a, const LinearOut& o, int splits, bool gather, hipStream_t s, bool attr) {
    using Core = TileCore<BF, TM, TN, WX, WY, XS, WS>;
    const auto whole = linear_tile_kernel<BF, TM, TN, WX, WY, XS, WS, false>;
    const auto pieces = linear_tile_kernel<BF, TM, TN, WX, WY, XS, WS, true>;
    if (attr) {
        const hipError_t e = hipFuncSetAttribute((const void*)whole, hipFuncAttributeMaxDynamicSharedMemorySize, Core::LDS);
        return e != hipSuccess ? e : hipFuncSetAttribute((const void*)pieces, hipFuncAttributeMaxDynamicSharedMemorySize, Core::LDS);
    }
    a.mtiles = (a.M + TM - 1) / TM;
    a.ntiles = (a.npad + TN - 1) / TN;
    a.m_fast = a.mtiles < a.ntiles;
    a.splits = splits;
    a.ksteps_per_split = (a.ksteps + splits - 1) / splits;
    hipLaunchKernelGGL(gather ? pieces : whole, dim3((unsigned)(a.mtiles * a.ntiles * splits)), dim3(64 * WX * WY), Core::LDS, s, a, o);
    return hipGetLastError();
}

template <bool BF, int FX, int FW, int NW, int ST>
hipError_t launch_wave(LinearIn a, const LinearOut& o, int splits, bool gather, hipStream_t s, bool attr) {
    using Shape = WaveShape<FX, FW, NW, ST>;
    const auto whole = linear_wave_kernel<BF, FX, FW, NW, ST, false>;
    const auto pieces = linear_wave_kernel<BF, FX, FW, NW, ST, true>;
    if (attr) {
        const hipError_t e = hipFuncSetAttribute((const void*)whole, hipFuncAttributeMaxDynamicSharedMemorySize, Shape::LDS);
        return e != hipSuccess ? e : hipFuncSetAttribute((const void*)pieces, hipFuncAttributeMaxDynamicSharedMemorySize, Shape::LDS);
    }
    a.mtiles = (a.M + Shape::TM - 1) / Shape::TM;
    a.ntiles = (a.npad + Shape::TN - 1) / Shape::TN;
    a.m_fast = a.mtiles < a.ntiles;
    a.splits = splits;
    a.ksteps_per_split = (a.ksteps + splits - 1) / splits;
    hipLaunchKernelGGL(gather ? pieces : whole, dim3((unsigned)(a.mtiles * a.ntiles * splits)), dim3(64 * NW), Shape::LDS, s, a, o);
    return hipGetLastError();
}

// The tile shapes and what their tiles take, in microseconds: the first round (256 tiles, one a CU, with the launch) first + steps *
// first_step, each further one more + steps * more_step.  Fitted to some 590 calls of 32 to 4096 tiles, K = 64 to 4096, N = 32 to 2048
// (7 to 15 % rms).  The wave kernel's small tiles have a batch done in one round; the tile kernel's 128-row tiles run two to a CU,
// which hides their beginnings and ends (short K: 6533 x 1504 x 128 12.9 us, 28 with the wave kernel); per value the 256-row tiles are
// the cheapest.
struct Shape { int tm, tn; float first, first_step, more, more_step, slow; };   // slow: a step of rows that LDS-DMA cannot take, against this
constexpr Shape kShapes[] = {
    {16, 32, 4.0f, 0.040f, 2.45f, 0.059f, 1.2f},       // wave kernel, 16 waves:  256 x 512 x 4096    8.1 us
    {32, 32, 3.6f, 0.070f, 0.82f, 0.081f, 1.3f},       // wave kernel,  8 waves:  64 x 4096 x 4096    9.8 us
    {64, 64, 4.8f, 0.165f, 3.05f, 0.22f, 1.3f},         // wave kernel,  8 waves:  256 x 4096 x 4096  17 us
    {64, 128, 6.0f, 0.26f, 4.8f, 0.31f, 1.3f},         // wave kernel,  4 waves:  2011 x 1024 x 4096 24 us (128 x 64, more through LDS: 27)
    {128, 32, 3.2f, 0.33f, 0.63f, 0.57f, 1.7f},         // tile kernel, two a CU:  115728 x 32 x 2496 106 us (32 x 32 wave tiles: 121)
    {128, 64, 3.9f, 0.36f, 1.3f, 0.27f, 1.7f},          // tile kernel, two a CU:  13373 x 224 x 1024 14 us (256 x 128: 18)
    {256, 128, 6.7f, 0.76f, 4.9f, 0.97f, 1.7f},         // tile kernel:            16384 x 512 x 4096 70 us
    {256, 256, 10.6f, 1.23f, 8.6f, 1.57f, 1.7f},        // tile kernel:            65536 x 512 x 4096 242 us
};
constexpr int kNumShapes = sizeof kShapes / sizeof kShapes[0];
template <bool BF>
hipError_t launch_shape(int t, const LinearIn& a, const LinearOut& o, int splits, bool gather, hipStream_t s, bool attr) {
    switch (t) {
        case 0: return launch_wave<BF, 1, 2, 16, 3>(a, o, splits, gather, s, attr);
        case 1: return launch_wave<BF, 2, 2, 8, 2>(a, o, splits, gather, s, attr);
        case 2: return launch_wave<BF, 4, 4, 8, 2>(a, o, splits, gather, s, attr);
        case 3: return launch_wave<BF, 4, 8, 4, 2>(a, o, splits, gather, s, attr);
        case 4: return launch_tile<BF, 128, 32, 4, 1, 3, 3>(a, o, splits, gather, s, attr);
        case 5: return launch_tile<BF, 128, 64, 2, 2, 3, 3>(a, o, splits, gather, s, attr);
        case 6: return launch_tile<BF, 256, 128, 4, 2, 3, 3>(a, o, splits, gather, s, attr);
        default: return launch_tile<BF, 256, 256, 2, 4, 3, 2>(a, o, splits, gather, s, attr);
    }
}

// What a call runs as: the shape, the number of K slices and the way unaligned rows go in, whichever an estimate of the
// time puts first.  K slices divide the steps and add the join (a launch, and every slice's sums written and read once: 3.5 us +
// the bytes at 4 TB/s).  Rows that LDS-DMA cannot take go through registers (16384 x 512 x 4095: 106 us, 200 packed) or, where
// wide layers read them many times and the workspace holds them, are packed by a pass of their own, 2 us + the bytes at 4.5 TB/s
// (800 x 4096 x 4095: 47 us, 60 through registers).
LinearPlan plan_linear(int M, int npad, int ksteps, bool whole, int64_t pack_rows, size_t slab_bytes) {
    LinearPlan best;
    float best_t = 1e30f;
    auto consider = [&](float t, int shape, int splits, bool gather) {
        if (t < best_t) { best_t = t; best.shape = shape; best.splits = splits; best.gather = gather; }
    };
    const float sums = (float)M * (float)npad * 4e-6f;          // MB of a slice's sums
    auto shapes = [&](float extra, bool gather) {
        for (int i = 0; i < kNumShapes; ++i) {
            const Shape& sh = kShapes[i];
            const float slow = gather ? sh.slow : 1.f;
            const int tiles = (M + sh.tm - 1) / sh.tm * ((npad + sh.tn - 1) / sh.tn);       // (at most 2^18 x 2^11)
            const float steps = (float)ksteps * slow;
            consider(extra + sh.first + steps * sh.first_step + (float)((tiles - 1) >> 8) * (sh.more + steps * sh.more_step), i, 1, gather);
            if (tiles > 256) continue;
            for (int splits : {2, 3, 4, 6, 8, 12, 16}) {
                if (splits > ksteps || tiles * splits > 512 || splits * sums * 1e6f > (float)slab_bytes) break;
                const float part = (float)((ksteps + splits - 1) / splits) * slow;
                consider(extra + sh.first + part * sh.first_step + (float)((tiles * splits - 1) >> 8) * (sh.more + part * sh.more_step) + 3.5f +
                             splits * sums * 0.5f, i, splits, gather);
            }
        }
    };
    if (whole) shapes(0.f, false);
    else shapes(0.f, true);
    if (!whole && M <= pack_rows) shapes(2.f + (float)M * (float)ksteps * 256e-6f / 4.5f, false);
    return best;
}

}  // namespace

size_t linear_layout_bytes(int N, int K) { return (size_t)linear_npad(N) * linear_kpad(K) * 2; }

hipError_t launch_linear_layout(const void* w, void* wt, int N, int K, hipStream_t s) {
    if (!w || !wt || N <= 0 || K <= 0) return hipErrorInvalidValue;
    const int panels = linear_npad(N) / 16, ksteps = linear_kpad(K) / 32;
    const size_t n = (size_t)panels * ksteps * 64;
    hipLaunchKernelGGL(linear_layout_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (const uint16_t*)w, (uint16_t*)wt, N, K,
                       panels, ksteps);
    return hipGetLastError();
}

LinearPlan linear_plan(int64_t M, int npad, int ksteps, bool whole, size_t row_bytes, const LinearWork& ws) {
    LinearPlan p = plan_linear((int)(M < kRunRows ? M : kRunRows), npad, ksteps, whole, (int64_t)(ws.pack_bytes / row_bytes), ws.slab_bytes);
    const int per = (ksteps + p.splits - 1) / p.splits;
    p.splits = (ksteps + per - 1) / per;                        // (no empty slice)
    p.M = M;
    p.whole = whole;
    return p;
}

hipError_t launch_linear(const LinearCall& q, const LinearWork& ws, hipStream_t s) {
    if (q.M <= 0 || q.N <= 0 || q.K <= 0 || !q.x || !q.wt || !q.bias || !q.out.out || !ws.slabs || !ws.pack || !ws.zeros || !q.plan)
        return hipErrorInvalidValue;
    LinearIn a{};
    a.wt = q.wt; a.bias = q.bias; a.zeros = ws.zeros;
    const int parts = q.pair ? 2 : 1;
    a.K = q.pair ? 2 * linear_kpad(q.K) : q.K; a.npad = linear_npad(q.N); a.panels = a.npad / 16; a.ksteps = parts * (linear_kpad(q.K) / 64);
    if (q.pair && (q.tiled || q.ldx != a.K || (size_t)q.x % 16)) return hipErrorInvalidValue;
    // can LDS-DMA take the rows?
    const bool whole = q.tiled || (a.K % 8 == 0 && q.ldx % 8 == 0 && (size_t)q.x % 16 == 0);
    const size_t row_bytes = (size_t)linear_kpad(q.K) * 2;
    if (q.plan->M != q.M || q.plan->whole != whole) *q.plan = linear_plan(q.M, a.npad, a.ksteps, whole, row_bytes, ws);
    const LinearPlan& plan = *q.plan;
    const bool pack = !whole && !plan.gather;
    for (int64_t m0 = 0; m0 < q.M; m0 += kRunRows) {        // (a launch has fewer than 2^32 threads)
        const int rows = (int)(q.M - m0 < kRunRows ? q.M - m0 : kRunRows);
        a.M = rows;
        if (!pack) {
            a.ldx = q.ldx; a.tiled = q.tiled; a.xtile = (size_t)(q.K / 64) * 32768; a.xstep = q.tiled ? 32768 : 128;
            a.x = (const char*)q.x + (q.tiled ? (size_t)(m0 / 256) * a.xtile : (size_t)m0 * q.ldx * 2);
        } else {                                            // (M <= pack_rows: one run)
            const size_t n = (size_t)rows * (row_bytes / 16);
            hipLaunchKernelGGL(linear_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (const uint16_t*)q.x, q.ldx, q.K,
                               (int)(row_bytes / 2), (uint16_t*)ws.pack, rows);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            a.x = ws.pack; a.ldx = (int64_t)(row_bytes / 2); a.tiled = 0; a.xtile = 0; a.xstep = 128;
        }
        LinearOut o = q.out;
        const size_t osz = o.otype == kF32 ? 4 : 2, rsz = o.rtype == kF32 ? 4 : 2;
        o.out = (char*)o.out + (size_t)m0 * o.ldo * osz;
        if (o.res) o.res = (const char*)o.res + (size_t)m0 * o.ldr * rsz;
        if (o.scale) o.scale += m0;
        o.N = q.N;
        const int splits = plan.splits;
        a.slab = splits > 1 ? ws.slabs : nullptr;
        hipError_t e = q.bf16 ? launch_shape<true>(plan.shape, a, o, splits, plan.gather, s, false)
                              : launch_shape<false>(plan.shape, a, o, splits, plan.gather, s, false);
        if (e != hipSuccess) return e;
        if (splits > 1) {
            const size_t n = (size_t)rows * (a.npad / 8);
            hipLaunchKernelGGL(linear_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a, o, splits);
            e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

hipError_t launch_linear_split(const float* x, int64_t ldx, int64_t M, int N, void* out, float* scale, hipStream_t s) {
    const int kpad = linear_kpad(N);
    if (!x || !out || !scale || M <= 0 || M > kRunRows || N <= 0 || ldx < kpad || ldx % 64 || (size_t)x % 16 || (size_t)out % 16)
        return hipErrorInvalidValue;
    const auto kern = kpad <= 512 ? linear_split_kernel<1> : kpad <= 2048 ? linear_split_kernel<4> : linear_split_kernel<0>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, x, ldx, N, kpad, (half_t*)out, scale, (int)M);
    return hipGetLastError();
}

hipError_t launch_unit_rows(const void* x, int type, int64_t ldx, int64_t M, int N, const UnitOut& o, hipStream_t s) {
    if (!x || !o.out || M <= 0 || N <= 0 || (o.gallery && N % 64)) return hipErrorInvalidValue;
    if (type == kF32) return unit_by_width<float>(x, ldx, M, N, o, s);
    if (type == kBF16) return unit_by_width<__bf16>(x, ldx, M, N, o, s);
    return unit_by_width<half_t>(x, ldx, M, N, o, s);
}

hipError_t linear_kernels_init() {
    for (int t = 0; t < kNumShapes; ++t) {
        hipError_t e = launch_shape<false>(t, LinearIn{}, LinearOut{}, 1, false, nullptr, true);
        if (e == hipSuccess) e = launch_shape<true>(t, LinearIn{}, LinearOut{}, 1, false, nullptr, true);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace frhot
