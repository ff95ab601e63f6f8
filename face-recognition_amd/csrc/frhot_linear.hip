// HIP kernels of the descriptor heads (gfx950): matrix product with bias, activation and residual in its
// epilogue, and unit rows.
//
//   linear     y[m][n] = round(act(sum_k x[m][k] w[n][k] + b[n]) + r[m][n]),  products of fp16 / bf16 values summed in fp32
//   unit rows  y[m][c] = fp16(x[m][c] / |x[m]|),  the sum of squares in 64 bits, the norm rounded to fp32
//
// Weights are laid out once, when a layer is created, in the order the matrix instruction takes them:
//   fragment (p, s) = 1 KiB holding, for lane l and e = 0..7, w[chan(p, l & 15)][32 s + 8 (l >> 4) + e],
//   fragments of one panel p of 16 channels back to back over s, zeros beyond N and K.
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

// The activation in fp32.  Written so that each keeps its relative accuracy far out (gelu through erfc, the tanh form
// through its logistic equivalent) and NaN stays NaN (a maximum with zero would turn it into zero).
FR_DEV float activate(float v, int act) {
    switch (act) {
        case kActRelu: return v < 0.f ? 0.f : v;
        case kActSilu: return v / (1.f + expf(-v));
        case kActGelu: return 0.5f * v * erfcf(v * -0.70710678118654752f);
        case kActGeluTanh: return v / (1.f + expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
        default: return v;
    }
}

// Eight consecutive channels n .. n+7 of row m: bias, activation, residual, ONE rounding, store.  Columns from N on are not
// written.
FR_DEV void finish8(const LinearOut& o, const float* __restrict__ bias, size_t m, int n, float (&v)[8]) {
    if (n >= o.N) return;
    const float4v b0 = *(const float4v*)(bias + n), b1 = *(const float4v*)(bias + n + 4);     // (padded with zeros)
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] += b0[j]; v[4 + j] += b1[j]; }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = activate(v[j], o.act);
    const bool whole = n + 8 <= o.N;
    if (o.res) {
        const size_t at = m * (size_t)o.ldr + n;
        if (whole && o.vec_res) {
            if (o.rtype == kF32) {
                const float4v r0 = *(const float4v*)((const float*)o.res + at), r1 = *(const float4v*)((const float*)o.res + at + 4);
#pragma unroll
                for (int j = 0; j < 4; ++j) { v[j] += r0[j]; v[4 + j] += r1[j]; }
            } else if (o.rtype == kBF16) {
                const bf8 r = *(const bf8*)((const __bf16*)o.res + at);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += (float)r[j];
            } else {
                const half8 r = *(const half8*)((const half_t*)o.res + at);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += (float)r[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (n + j < o.N) v[j] += load1(o.res, at + j, o.rtype);
        }
    }
    const size_t at = m * (size_t)o.ldo + n;
    if (whole && o.vec_out) {
        if (o.otype == kF32) {
            *(float4v*)((float*)o.out + at) = float4v{v[0], v[1], v[2], v[3]};
            *(float4v*)((float*)o.out + at + 4) = float4v{v[4], v[5], v[6], v[7]};
        } else if (o.otype == kBF16) {
            bf8 t;
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = (__bf16)v[j];
            *(bf8*)((__bf16*)o.out + at) = t;
        } else {
            half8 t;
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = (half_t)v[j];
            *(half8*)((half_t*)o.out + at) = t;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j < o.N) store1(o.out, at + j, o.otype, v[j]);
    }
}

// w [N][K] -> fragments (see the head of the file); thread = one lane's 16 bytes of one fragment
__global__ __launch_bounds__(256) void linear_layout_kernel(const uint16_t* __restrict__ w, uint16_t* __restrict__ wt, int N, int K,
                                                            int panels, int ksteps) {
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)panels * ksteps * 64) return;
    const int lane = (int)(t & 63);
    const int s = (int)((t >> 6) % ksteps), p = (int)((t >> 6) / ksteps);
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

// Rows whose addresses the 16-byte loads cannot take (odd strides, K not a multiple of 8) are first brought into rows of
// `kpad` elements with zeros behind the K-th.
__global__ __launch_bounds__(256) void linear_pack_kernel(const uint16_t* __restrict__ x, int64_t ldx, int K, int kpad,
                                                          uint16_t* __restrict__ out, int rows) {
    const int per_row = kpad >> 3;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)rows * per_row) return;
    const int r = (int)(t / per_row), k0 = (int)(t % per_row) * 8;
    const uint16_t* src = x + (size_t)r * ldx + k0;
    uint4v o;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const unsigned lo = k0 + 2 * e < K ? src[2 * e] : 0u, hi = k0 + 2 * e + 1 < K ? src[2 * e + 1] : 0u;
        o[e] = lo | (hi << 16);
    }
    *(uint4v*)(out + t * 8) = o;
}

// One TM x TN tile of y (or of a K slice's partial sums) per block, 64 K-elements per step through two LDS stages filled by
// 16-byte LDS-DMA.  X rows are 128 bytes in LDS, 16-byte chunk c of row r at position c ^ (r & 7) (applied to the
// source address, undone at the read); weight fragments lie as in memory and are read linearly: neither read has a bank
// conflict.  Waves WX x WY, each (TM/WX) x (TN/WY).
template <bool BF, int TM, int TN, int WX, int WY>
__global__ __launch_bounds__(64 * WX * WY) void linear_tile_kernel(LinearIn a, LinearOut o) {
    constexpr int NW = WX * WY, TX = TM / WX, TY = TN / WY, NX = TX / 16, NY = TY / 16;
    constexpr int XB = TM * 128, WB = TN * 128, SB = XB + WB;
    constexpr int NPX = TM / 8 / NW, NPW = TN / 8 / NW;
    static_assert(TM % (8 * NW) == 0 && TN % (8 * NW) == 0 && TX % 16 == 0 && TY % 32 == 0, "tile shape");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wx = wave / WY, wy = wave % WY;
    const int l15 = lane & 15, g0 = lane >> 4, l7 = lane & 7;

    const int tiles = a.mtiles * a.ntiles;
    const int id = xcd_remap(blockIdx.x, gridDim.x);
    const int z = id / tiles, t = id % tiles;
    const int mt = a.m_fast ? t % a.mtiles : t / a.ntiles, nt = a.m_fast ? t / a.mtiles : t % a.ntiles;
    const int m0 = mt * TM, n0 = nt * TN;
    const int k_lo = z * a.ksteps_per_split, k_hi = min(a.ksteps, k_lo + a.ksteps_per_split);

    const int c = l7 ^ (lane >> 3);                 // the 16-byte chunk this lane fetches of its row
    const char* xp[NPX];
#pragma unroll
    for (int i = 0; i < NPX; ++i) {
        int m = m0 + 8 * (wave + NW * i) + (lane >> 3);
        m = m < a.M ? m : a.M - 1;
        xp[i] = (const char*)a.x + (a.tiled ? (size_t)(m >> 8) * a.xtile + (size_t)(m & 255) * 128 : (size_t)m * a.ldx * 2) + c * 16;
    }
    const char* wp[NPW];
#pragma unroll
    for (int i = 0; i < NPW; ++i) {
        const int piece = wave + NW * i;
        int p = (n0 >> 4) + (piece >> 1);
        p = p < a.panels ? p : a.panels - 1;        // (columns beyond N: computed from the last panel and dropped)
        wp[i] = (const char*)a.wt + ((size_t)p * (2 * a.ksteps) + (piece & 1)) * 1024 + lane * 16;
    }
    auto issue = [&](int ks, char* st) {
        const bool tail = ks * 64 + c * 8 >= a.K;   // chunks behind the K-th element: zeros (K is a multiple of 8 here)
#pragma unroll
        for (int i = 0; i < NPX; ++i) {
            const char* src = xp[i] + (size_t)ks * a.xstep;
            glds16(tail ? (const char*)a.zeros + c * 16 : src, st + (wave + NW * i) * 1024);
        }
#pragma unroll
        for (int i = 0; i < NPW; ++i) glds16(wp[i] + (size_t)ks * 2048, st + XB + (wave + NW * i) * 1024);
    };

    float4v acc[NY][NX];
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
        for (int x = 0; x < NX; ++x) acc[y][x] = float4v{0.f, 0.f, 0.f, 0.f};

    issue(k_lo, smem);
    __syncthreads();
    for (int ks = k_lo; ks < k_hi; ++ks) {
        char* const st = smem + ((ks - k_lo) & 1) * SB;
        if (ks + 1 < k_hi) issue(ks + 1, smem + (((ks - k_lo) & 1) ^ 1) * SB);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int coff = ((kk * 4 + g0) ^ l7) << 4;
            uint4v fx[NX], fw[NY];
#pragma unroll
            for (int x = 0; x < NX; ++x) fx[x] = *(const uint4v*)(st + (wx * TX + x * 16 + l15) * 128 + coff);
#pragma unroll
            for (int y = 0; y < NY; ++y) fw[y] = *(const uint4v*)(st + XB + ((wy * NY + y) * 2 + kk) * 1024 + lane * 16);
#pragma unroll
            for (int y = 0; y < NY; ++y)
#pragma unroll
                for (int x = 0; x < NX; ++x) acc[y][x] = mfma<BF>(fw[y], fx[x], acc[y][x]);
        }
        __syncthreads();
    }

#pragma unroll
    for (int x = 0; x < NX; ++x) {
        const int m = m0 + wx * TX + x * 16 + l15;
        if (m >= a.M) continue;
#pragma unroll
        for (int u = 0; u < NY / 2; ++u) {
            const int n = n0 + wy * TY + u * 32 + g0 * 8;
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = acc[2 * u][x][j]; v[4 + j] = acc[2 * u + 1][x][j]; }
            if (a.slab) {
                if (n < a.npad) {
                    float* d = a.slab + ((size_t)z * a.M + m) * a.npad + n;
                    *(float4v*)d = float4v{v[0], v[1], v[2], v[3]};
                    *(float4v*)(d + 4) = float4v{v[4], v[5], v[6], v[7]};
                }
            } else {
                finish8(o, a.bias, m, n, v);
            }
        }
    }
}

// Joins the K slices in slice order and finishes the rows; thread = 8 channels of one row.
__global__ __launch_bounds__(256) void linear_join_kernel(LinearIn a, LinearOut o, int splits) {
    const int per_row = a.npad >> 3;
    const size_t t = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= (size_t)a.M * per_row) return;
    const int m = (int)(t / per_row), n = (int)(t % per_row) * 8;
    float v[8] = {};
    for (int z = 0; z < splits; ++z) {
        const float* p = a.slab + ((size_t)z * a.M + m) * a.npad + n;
        const float4v p0 = *(const float4v*)p, p1 = *(const float4v*)(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[j] += p0[j]; v[4 + j] += p1[j]; }
    }
    finish8(o, a.bias, m, n, v);
}

// ------------------------------------------------------------- unit rows ---
// One wave per row.  The norm comes from a 64-bit sum of squares rounded to fp32, then one IEEE division per
// element: the stored row is the same whatever the summation order, and the same as the library's own upload makes of
// it (gallery_upsert_kernel).  A row shorter than 1e-30 is divided by one.
__global__ __launch_bounds__(256) void unit_rows_kernel(const void* __restrict__ x, int type, int64_t ldx, int M, int N,
                                                        UnitOut o) {
    const int m = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= M) return;
    const size_t at = (size_t)m * ldx;
    double ss = 0.0;
    for (int c = lane; c < N; c += 64) {
        const double v = load1(x, at + c, type);
        ss += v * v;
    }
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) ss += __shfl_xor(ss, s);
    float nrm = (float)sqrt(ss);
    nrm = nrm < 1e-30f ? 1.0f : nrm;
    for (int c = lane; c < N; c += 64) {
        const half_t v = (half_t)__fdiv_rn(load1(x, at + c, type), nrm);
        if (o.gallery) {
            const int64_t r = o.row0 + m;       // (the order of a gallery's rows in memory: see gal_index)
            ((half_t*)o.out)[((((size_t)(r >> 8) * (N >> 6) + (c >> 6)) << 8) + (r & 255)) * 64 + (c & 63)] = v;
        } else {
            ((half_t*)o.out)[(size_t)m * o.ldo + c] = v;
        }
    }
    if (lane == 0 && o.keys_dst) o.keys_dst[o.row0 + m] = o.keys_src[o.row0 + m];
}

template <bool BF, int TM, int TN, int WX, int WY>
hipError_t launch_tile(LinearIn a, const LinearOut& o, int splits, hipStream_t s) {
    constexpr int SB = (TM + TN) * 128;
    a.mtiles = (a.M + TM - 1) / TM;
    a.ntiles = (a.npad + TN - 1) / TN;
    a.m_fast = a.mtiles < a.ntiles;
    a.ksteps_per_split = (a.ksteps + splits - 1) / splits;
    hipLaunchKernelGGL((linear_tile_kernel<BF, TM, TN, WX, WY>), dim3((unsigned)(a.mtiles * a.ntiles * splits)), dim3(64 * WX * WY),
                       2 * SB, s, a, o);
    return hipGetLastError();
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

hipError_t launch_linear(const LinearCall& q, const LinearWork& ws, hipStream_t s) {
    if (q.M <= 0 || q.N <= 0 || q.K <= 0 || !q.x || !q.wt || !q.bias || !q.out.out || !ws.slabs || !ws.pack || !ws.zeros)
        return hipErrorInvalidValue;
    LinearIn a{};
    a.wt = q.wt; a.bias = q.bias; a.zeros = ws.zeros;
    a.K = q.K; a.npad = linear_npad(q.N); a.panels = a.npad / 16; a.ksteps = linear_kpad(q.K) / 64;
    const bool direct = q.tiled || (q.K % 8 == 0 && q.ldx % 8 == 0 && (size_t)q.x % 16 == 0);
    const size_t row_bytes = (size_t)linear_kpad(q.K) * 2;
    // rows that must be packed first go through the workspace in runs of whole tiles
    const int64_t run = direct ? q.M : (int64_t)(ws.pack_bytes / row_bytes) / 256 * 256;
    if (run <= 0) return hipErrorInvalidValue;
    for (int64_t m0 = 0; m0 < q.M; m0 += run) {
        const int rows = (int)(q.M - m0 < run ? q.M - m0 : run);
        a.M = rows;
        if (direct) {
            a.x = q.x; a.ldx = q.ldx; a.tiled = q.tiled; a.xtile = (size_t)(q.K / 64) * 32768; a.xstep = q.tiled ? 32768 : 128;
        } else {
            const size_t n = (size_t)rows * (row_bytes / 16);
            hipLaunchKernelGGL(linear_pack_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
                               (const uint16_t*)q.x + (size_t)m0 * q.ldx, q.ldx, q.K, (int)(row_bytes / 2), (uint16_t*)ws.pack, rows);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            a.x = ws.pack; a.ldx = (int64_t)(row_bytes / 2); a.tiled = 0; a.xtile = 0; a.xstep = 128;
        }
        LinearOut o = q.out;
        const size_t osz = o.otype == kF32 ? 4 : 2, rsz = o.rtype == kF32 ? 4 : 2;
        o.out = (char*)o.out + (size_t)m0 * o.ldo * osz;
        if (o.res) o.res = (const char*)o.res + (size_t)m0 * o.ldr * rsz;
        o.N = q.N;
        o.vec_out = (size_t)o.out % 16 == 0 && (size_t)o.ldo * osz % 16 == 0;
        o.vec_res = o.res && (size_t)o.res % 16 == 0 && (size_t)o.ldr * rsz % 16 == 0;
        // Few tiles leave CUs idle: K is then cut into slices whose partial sums meet in the workspace.
        const int tiles = ((rows + 127) / 128) * ((a.npad + 127) / 128);
        int splits = 256 / tiles;
        if (splits > a.ksteps) splits = a.ksteps;
        const size_t slab = (size_t)rows * a.npad * 4;
        if ((size_t)splits * slab > ws.slab_bytes) splits = (int)(ws.slab_bytes / slab);
        if (splits < 1) splits = 1;
        splits = (a.ksteps + (a.ksteps + splits - 1) / splits - 1) / ((a.ksteps + splits - 1) / splits);
        a.slab = splits > 1 ? ws.slabs : nullptr;
        hipError_t e = q.bf16 ? launch_tile<true, 128, 128, 2, 2>(a, o, splits, s) : launch_tile<false, 128, 128, 2, 2>(a, o, splits, s);
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

hipError_t launch_unit_rows(const void* x, int type, int64_t ldx, int64_t M, int N, const UnitOut& o, hipStream_t s) {
    if (!x || !o.out || M <= 0 || N <= 0 || (o.gallery && N % 64)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(unit_rows_kernel, dim3((unsigned)((M + 3) / 4)), dim3(256), 0, s, x, type, ldx, (int)M, N, o);
    return hipGetLastError();
}

hipError_t linear_kernels_init() {
    hipError_t e = hipFuncSetAttribute((const void*)linear_tile_kernel<false, 128, 128, 2, 2>, hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
    if (e == hipSuccess)
        e = hipFuncSetAttribute((const void*)linear_tile_kernel<true, 128, 128, 2, 2>, hipFuncAttributeMaxDynamicSharedMemorySize, 65536);
    return e;
}

}  // namespace frhot
