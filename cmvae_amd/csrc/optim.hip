// AdamW over many tensors in one launch, with states in 32 or in 8 bits: cmvae_adamw_step, cmvae_adamw_state_values.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// The tensors' addresses and sizes travel in the launch's own arguments (nothing is uploaded, nothing is kept between
// calls, and a captured launch carries them): a workgroup takes one piece of 4096 values and finds its tensor by one
// vector read of the pieces' starts and a ballot.
//
// Bound by memory.  States in 32 bits beside bf16 parameters (22 bytes a value): 123 M values of 44 tensors in 505 us, 5.4 TB/s;
// 1.1 M fp32 values of 58 tensors in 8 us.  States in 8 bits beside fp32 (16 bytes a value): 98.8 M values in 327 us, 4.8 TB/s;
// what they stand for, as fp32: 156 us, 6.3 TB/s.
//
// 8-bit states: 256 consecutive values of a tensor share one fp32 scale per moment.
//   m: OCP e4m3 of m / s, s = max|m| / 448, to nearest, ties to even;
//   v: 5 exponent and 3 mantissa bits, no sign, of v / s, s = max v / 1.75: code c stands for s 2^((c >> 3) - 31) (1 +
//      (c & 7) / 8), 0 for zero; to nearest, ties to even, but a positive v never becomes 0 (the next step divides by
//      its root).  31 octaves below the block's largest, and a root to 3 %, where e4m3 would hold 18.
//   A moment beyond fp32 (its gradient was not finite, or its square is not) becomes e4m3's NaN / code 255, read as
//   infinity, and stays out of its block's scale: its neighbours keep theirs.
// The step itself uses the moments before they are rounded, in fp32: its few roundings, 2^-24 of the step each, are far under
// the parameter's own, and a root and a reciprocal in fp64 are not.  Moments and the choice between two neighbouring codes are
// computed in fp64, which costs no more than fp32 here (the card does 128 fp64 operations per cycle and compute unit, and
// the kernel waits for memory): a code is then the nearest one of the exact moment, not of a rounded one.
#include "common.h"

#include <cmath>
#include <type_traits>

namespace cmvae {
namespace opt {

constexpr int PIECE = 4096, BLOCK = 256;        // values per workgroup; values per scale
constexpr int MAX_T = 96;                       // tensors per launch: 3.2 KB of arguments

struct Table {
    void* p[MAX_T];
    const void* g[MAX_T];
    long n[MAX_T];
    int first[MAX_T];                           // first piece of the tensor in this launch
    int block[MAX_T];                           // its states begin at BLOCK * block
    uint8_t kind[MAX_T];                        // dtype | 4 if its rows of four values are not aligned
    int count;
};
static_assert(sizeof(Table) + 128 <= 4096, "launch arguments");

struct Hyper {
    double lr, b1, b2, eps, wd;
    double c1, c2;                              // 1 - b1^t, 1 - b2^t
    const long long* step_dev;                  // != NULL: t from device memory
};

struct Consts {
    float decay, step, rc2, eps;                // 1 - lr wd, lr / c1, 1 / sqrt(c2)
};

__device__ __forceinline__ Consts consts_of(const Hyper& h) {
    double c1 = h.c1, c2 = h.c2;
    if (h.step_dev) {
        __shared__ double s[2];
        if (threadIdx.x == 0) {
            const double t = (double)h.step_dev[0];
            s[0] = 1.0 - pow(h.b1, t);
            s[1] = 1.0 - pow(h.b2, t);
        }
        __syncthreads();
        c1 = s[0];
        c2 = s[1];
    }
    return {(float)(1.0 - h.lr * h.wd), (float)(h.lr / c1), (float)(1.0 / sqrt(c2)), (float)h.eps};
}

__device__ __forceinline__ int find(const Table& t) {
    const int lane = threadIdx.x & 63, b = (int)blockIdx.x;
    int k = 0;
#pragma unroll
    for (int i = 0; i < MAX_T; i += 64) {
        const int at = i + lane;
        k += __popcll(__ballot(at < t.count && t.first[at < MAX_T ? at : 0] <= b));
    }
    return __builtin_amdgcn_readfirstlane(k) - 1;
}

template <typename T>
__device__ __forceinline__ void get4(const void* base, long i, long n, bool whole, float (&x)[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T* p = (const T*)base + i;
    if (whole) {
        const T4 v = *reinterpret_cast<const T4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = i + j < n ? (float)p[j] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void put4(void* base, long i, long n, bool whole, const float (&x)[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T* p = (T*)base + i;
    if (whole) {
        *reinterpret_cast<T4*>(p) = T4{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) p[j] = (T)x[j];
    }
}

__device__ __forceinline__ float update(float p, float m, float v, const Consts& c) {
    return p * c.decay - c.step * (m * __builtin_amdgcn_rcpf(sqrtf(v) * c.rc2 + c.eps));      // the reciprocal to 1 ulp
}

// ------------------------------------------------------------------------------------------------ states in 32 bits
template <typename T>
__device__ __forceinline__ void step32(const Table& t, int k, const Hyper& h, float* m0, float* v0) {
    const Consts c = consts_of(h);
    const float b1 = (float)h.b1, b2 = (float)h.b2, a1 = (float)(1.0 - h.b1), a2 = (float)(1.0 - h.b2);
    const long n = t.n[k];
    const bool al = !(t.kind[k] & 4);
    float* m = m0 + (long)t.block[k] * BLOCK;
    float* v = v0 + (long)t.block[k] * BLOCK;
    const long i0 = (long)((int)blockIdx.x - t.first[k]) * PIECE + threadIdx.x * 4;
#pragma unroll
    for (int r = 0; r < PIECE / 1024; ++r) {
        const long i = i0 + r * 1024;
        if (i >= n) break;
        const bool whole = al && i + 4 <= n;
        float p[4], g[4];
        get4<T>(t.p[k], i, n, whole, p);
        get4<T>(t.g[k], i, n, whole, g);
        float4 mm = *reinterpret_cast<const float4*>(m + i), vv = *reinterpret_cast<const float4*>(v + i);
        float* mp = &mm.x;
        float* vp = &vv.x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mp[j] = b1 * mp[j] + a1 * g[j];
            vp[j] = b2 * vp[j] + a2 * g[j] * g[j];
            p[j] = update(p[j], mp[j], vp[j], c);
        }
        *reinterpret_cast<float4*>(m + i) = mm;
        *reinterpret_cast<float4*>(v + i) = vv;
        put4<T>(t.p[k], i, n, whole, p);
    }
}

__global__ __launch_bounds__(256) void adamw32_kernel(Table t, Hyper h, float* m, float* v) {
    const int k = find(t);
    switch (t.kind[k] & 3) {
        case CMVAE_F32: step32<float>(t, k, h, m, v); break;
        case CMVAE_BF16: step32<__bf16>(t, k, h, m, v); break;
        default: step32<_Float16>(t, k, h, m, v); break;
    }
}

// ------------------------------------------------------------------------------------------------ states in 8 bits
// over the 16 lanes of a block of 256 values: lane ^ 1, lane ^ 2, the other four of eight, the other eight
template <int CTRL>
__device__ __forceinline__ double max_dpp(double x) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, 0xf, 0xf, false);
    return fmax(x, __hiloint2double(hi, lo));
}
__device__ __forceinline__ double max16(double x) {
    return max_dpp<0x140>(max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(x))));
}

__device__ __forceinline__ float decode_v(int code) {
    float x = __int_as_float((code + 768) << 20);
    x = code == 0 ? 0.f : x;
    return code == 255 ? INFINITY : x;
}

// x rounded to e4m3's grid (quantum 2^(e - 3), e the exponent, at least -6), as a float: adding 1.5 * 2^52 quanta makes
// the fp64 adder round there
__device__ __forceinline__ float round_m(double x) {
    const int hi = __double2hiint(x);
    const int e = max((hi >> 20) & 0x7ff, 1023 - 6);
    const double c = __hiloint2double(((e - 3 + 52) << 20) | 0x80000, 0);
    const float r = (float)((x + c) - c);
    return (hi & 0x7ff00000) == 0x7ff00000 ? __int_as_float(0x7fc00000) : r;
}

// x >= 0 -> code, to nearest even on the fp64 bits (the low word only as "more than a tie"); no branch here nor where it is
// used: sixteen of them per thread cost more than what they skip
__device__ __forceinline__ int round_v(double x, bool finite) {
    const int hi = __double2hiint(x) | (__double2loint(x) != 0 ? 1 : 0);
    int r = ((hi + 0xffff + ((hi >> 17) & 1)) >> 17) - (1023 - 31) * 8;
    r = min(max(r, 1), 254);
    r = x > 0.0 ? r : 0;
    return finite ? r : 255;
}

__device__ __forceinline__ double moment(double b, double x, double y) {
#pragma clang fp contract(off)
    return b * x + y;
}

// x / s from i = 1 / s, corrected once: of 10^8 moments about one lies exactly between two codes, where the plain
// product x i may fall on either side
__device__ __forceinline__ double over(double x, double s, double i) {
    const double q = x * i;
    return fma(fma(-q, s, x), i, q);
}

template <typename T>
__device__ __forceinline__ void step8(const Table& t, int k, const Hyper& h, int* m0, int* v0, float* sm0, float* sv0) {
    const Consts c = consts_of(h);
    const double b1 = h.b1, b2 = h.b2, a1 = 1.0 - h.b1, a2 = 1.0 - h.b2;
    const long n = t.n[k];
    const bool al = !(t.kind[k] & 4);
    const int blk = ((int)blockIdx.x - t.first[k]) * (PIECE / BLOCK) + (threadIdx.x >> 4);       // block of the tensor
    const long i0 = (long)blk * BLOCK + (threadIdx.x & 15) * 4;
    if ((long)blk * BLOCK >= n) return;
    const long b = (long)t.block[k] + blk, s0 = (b * BLOCK + (threadIdx.x & 15) * 4) / 4;
    const double sm = (double)sm0[b], sv = (double)sv0[b];
    float p[4][4];
    double m[4][4], v[4][4];
    double am = 0.0, av = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const long i = i0 + q * 64;
        const bool whole = al && i + 4 <= n;
        float g[4];
        get4<T>(t.p[k], i, n, whole, p[q]);
        get4<T>(t.g[k], i, n, whole, g);
        const int mc = m0[s0 + q * 16], vc = v0[s0 + q * 16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float mf = j == 0 ? __builtin_amdgcn_cvt_f32_fp8(mc, 0) : j == 1 ? __builtin_amdgcn_cvt_f32_fp8(mc, 1)
                             : j == 2 ? __builtin_amdgcn_cvt_f32_fp8(mc, 2) : __builtin_amdgcn_cvt_f32_fp8(mc, 3);
            const float vf = decode_v((vc >> (8 * j)) & 255);
            const double gd = (double)g[j];
            // products rounded on their own, as written: with b1 = 0.9 a block's largest moment lies exactly between two
            // fp32 scales about once in 4480 blocks of bf16 gradients, and the same fp64 products then decide the same
            double mm = moment(b1, (double)mf * sm, a1 * gd), vv = moment(b2, (double)vf * sv, a2 * gd * gd);
            if (i + j >= n) mm = vv = 0.0;
            m[q][j] = mm;
            v[q][j] = vv;
            const double x = fabs(mm);
            am = fmax(am, x <= 3.4028234663852886e38 ? x : 0.0);
            av = fmax(av, vv <= 3.4028234663852886e38 ? vv : 0.0);
        }
    }
    am = max16(am);
    av = max16(av);
    const float nm = fmaxf((float)(am * (1.0 / 448.0)), 0x1p-126f), nv = fmaxf((float)(av * (1.0 / 1.75)), 0x1p-126f);
    const double im = 1.0 / (double)nm, iv = 1.0 / (double)nv;
    if ((threadIdx.x & 15) == 0) {
        sm0[b] = nm;
        sv0[b] = nv;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const long i = i0 + q * 64;
        float r[4];
        int vc = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            r[j] = round_m(over(m[q][j], nm, im));                // not finite: over() makes NaN of it
            const double vv = v[q][j];
            vc |= round_v(over(vv, nv, iv), vv <= 3.4028234663852886e38) << (8 * j);
            p[q][j] = update(p[q][j], (float)m[q][j], (float)vv, c);
        }
        int mc = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
        mc = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], mc, true);
        m0[s0 + q * 16] = mc;
        v0[s0 + q * 16] = vc;
        put4<T>(t.p[k], i, n, al && i + 4 <= n, p[q]);
    }
}

__global__ __launch_bounds__(256) void adamw8_kernel(Table t, Hyper h, int* m, int* v, float* sm, float* sv) {
    const int k = find(t);
    switch (t.kind[k] & 3) {
        case CMVAE_F32: step8<float>(t, k, h, m, v, sm, sv); break;
        case CMVAE_BF16: step8<__bf16>(t, k, h, m, v, sm, sv); break;
        default: step8<_Float16>(t, k, h, m, v, sm, sv); break;
    }
}

// what 8-bit states stand for, four values per thread
__global__ __launch_bounds__(256) void values_kernel(const int* m, const int* v, const float* sm, const float* sv, long n4,
                                                     float4* mo, float4* vo) {
    const long i = blockIdx.x * 256L + threadIdx.x;
    if (i >= n4) return;
    const int mc = m[i], vc = v[i];
    const float a = sm[i / (BLOCK / 4)], b = sv[i / (BLOCK / 4)];
    mo[i] = make_float4(__builtin_amdgcn_cvt_f32_fp8(mc, 0) * a, __builtin_amdgcn_cvt_f32_fp8(mc, 1) * a,
                        __builtin_amdgcn_cvt_f32_fp8(mc, 2) * a, __builtin_amdgcn_cvt_f32_fp8(mc, 3) * a);
    vo[i] = make_float4(decode_v(vc & 255) * b, decode_v((vc >> 8) & 255) * b, decode_v((vc >> 16) & 255) * b,
                        decode_v((vc >> 24) & 255) * b);
}

}  // namespace opt
}  // namespace cmvae

using namespace cmvae;

extern "C" int cmvae_adamw_step(const cmvae_adamw_tensor* tensors_host, int count, int state_bits, void* exp_avg,
                                void* exp_avg_sq, float* scales, int64_t state_len, int64_t step, const int64_t* step_dev,
                                double lr, double beta1, double beta2, double eps, double weight_decay, void* stream) {
    cmvae::clear_stale_error();
    CMVAE_REQUIRE(count >= 0 && (count == 0 || (tensors_host && exp_avg && exp_avg_sq)), "cmvae_adamw_step: NULL argument");
    CMVAE_REQUIRE(state_bits == 32 || (state_bits == 8 && scales), "cmvae_adamw_step: states of %d bits (32, or 8 with scales)",
                  state_bits);
    CMVAE_REQUIRE(state_len >= 0 && state_len % opt::BLOCK == 0 && state_len / opt::BLOCK < (1L << 31),
                  "cmvae_adamw_step: %ld state values (a multiple of %d)", (long)state_len, opt::BLOCK);
    CMVAE_REQUIRE((((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0, "cmvae_adamw_step: states must be 16-byte aligned");
    CMVAE_REQUIRE(step_dev || step >= 1, "cmvae_adamw_step: steps count from 1");
    CMVAE_REQUIRE(std::isfinite(lr) && std::isfinite(weight_decay) && eps >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1,
                  "cmvae_adamw_step: lr %g, betas (%g, %g), eps %g, weight decay %g", lr, beta1, beta2, eps, weight_decay);
    for (int i = 0; i < count; ++i) {
        const cmvae_adamw_tensor& d = tensors_host[i];
        CMVAE_REQUIRE(d.n >= 0 && d.state >= 0 && d.state % opt::BLOCK == 0 && d.state <= state_len && d.n <= state_len - d.state &&
                          (d.n == 0 || (d.param && d.grad)) && d.dtype >= CMVAE_F32 && d.dtype <= CMVAE_F16,
                      "cmvae_adamw_step: tensor %d (n %ld, state %ld, dtype %ld)", i, (long)d.n, (long)d.state, (long)d.dtype);
        const uintptr_t size = d.dtype == CMVAE_F32 ? 4 : 2;
        CMVAE_REQUIRE((((uintptr_t)d.param | (uintptr_t)d.grad) & (size - 1)) == 0, "cmvae_adamw_step: tensor %d is not aligned", i);
    }
    opt::Hyper h = {lr, beta1, beta2, eps, weight_decay, 1.0, 1.0, (const long long*)step_dev};
    if (!step_dev) {
        h.c1 = 1.0 - std::pow(beta1, (double)step);
        h.c2 = 1.0 - std::pow(beta2, (double)step);
    }
    opt::Table t;
    t.count = 0;
    long pieces = 0;
    for (int i = 0; i <= count; ++i) {
        const long more = i < count ? (tensors_host[i].n + opt::PIECE - 1) / opt::PIECE : 0;
        if (t.count && (i == count || t.count == opt::MAX_T || pieces + more > (1L << 30))) {
            if (state_bits == 32)
                hipLaunchKernelGGL(opt::adamw32_kernel, dim3((unsigned)pieces), dim3(256), 0, (hipStream_t)stream, t, h,
                                   (float*)exp_avg, (float*)exp_avg_sq);
            else
                hipLaunchKernelGGL(opt::adamw8_kernel, dim3((unsigned)pieces), dim3(256), 0, (hipStream_t)stream, t, h,
                                   (int*)exp_avg, (int*)exp_avg_sq, scales, scales + state_len / opt::BLOCK);
            if (int e = check_launch("adamw_kernel")) return e;
            t.count = 0;
            pieces = 0;
        }
        if (more == 0) continue;
        const cmvae_adamw_tensor& d = tensors_host[i];
        CMVAE_REQUIRE(more <= (1L << 30), "cmvae_adamw_step: tensor %d has %ld values", i, (long)d.n);
        const int c = t.count++;
        const uintptr_t vec = d.dtype == CMVAE_F32 ? 15 : 7;
        t.p[c] = d.param;
        t.g[c] = d.grad;
        t.n[c] = d.n;
        t.first[c] = (int)pieces;
        t.block[c] = (int)(d.state / opt::BLOCK);
        t.kind[c] = (uint8_t)(d.dtype | ((((uintptr_t)d.param | (uintptr_t)d.grad) & vec) ? 4 : 0));
        pieces += more;
    }
    return 0;
}

extern "C" int cmvae_adamw_state_values(const void* exp_avg, const void* exp_avg_sq, const float* scales, int64_t state_len,
                                        float* exp_avg_out, float* exp_avg_sq_out, void* stream) {
    cmvae::clear_stale_error();
    CMVAE_REQUIRE(state_len >= 0 && state_len % opt::BLOCK == 0 && state_len / 1024 < (1L << 31) - 1,
                  "cmvae_adamw_state_values: %ld state values (a multiple of %d)", (long)state_len, opt::BLOCK);
    if (state_len == 0) return 0;
    CMVAE_REQUIRE(exp_avg && exp_avg_sq && scales && exp_avg_out && exp_avg_sq_out, "cmvae_adamw_state_values: NULL argument");
    CMVAE_REQUIRE((((uintptr_t)exp_avg_out | (uintptr_t)exp_avg_sq_out) & 15) == 0 && (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 3) == 0,
                  "cmvae_adamw_state_values: buffers must be 16-byte aligned");
    const long n4 = state_len / 4;
    hipLaunchKernelGGL(opt::values_kernel, dim3((unsigned)((n4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       (const int*)exp_avg, (const int*)exp_avg_sq, scales, scales + state_len / opt::BLOCK, n4,
                       (float4*)exp_avg_out, (float4*)exp_avg_sq_out);
    return check_launch("adamw values_kernel");
}
