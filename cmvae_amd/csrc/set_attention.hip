// Set attention and its backward pass, which recomputes the probabilities: cmvae_set_attention_{fwd,bwd}.
//
//   s_ij = scale q_i . k_j          valid (i, j): i < q_len, j < k_len and, if causal, j <= i + k_len - q_len
//   p_i  = softmax of s_i over its valid j (all zero if it has none),   o_i = sum_j p_ij v_j (+ q_i if residual)
//   dv_j = sum_i p_ij do_i,   ds_ij = p_ij (do_i . v_j - delta_i),   delta_i = do_i . sum_j p_ij v_j
//   dq_i = scale sum_j ds_ij k_j (+ do_i if residual),   dk_j = scale sum_i ds_ij q_i
//
// The G = H / Hkv query heads that share a key head are one list of rows — the G * q_len rows that count (row r = head
// r / q_len, position r % q_len), then the others, which only get zeros — so a tile of keys is read once for all of them and
// the gradients of shared heads are summed in registers, in a fixed order.
//
// Every product is a 32 x 32 matrix instruction with the contraction's second factor in registers.  The forward and the dq
// kernel hold 32 query rows per wave and form S^T (keys x queries): a lane then has 16 keys of ONE query, so the softmax
// reduces inside the lane plus one exchange between the wave's halves, and the accumulator is, as it stands, the
// second factor of the next product (o^T = V^T P^T, dq^T = K^T dS^T).  The dkv kernel holds 32 keys per wave and forms
// S (queries x keys) for dv^T = dO^T P and dk^T = Q^T dS.  No probability is ever stored.
//
// Element types: bf16 and fp16 on their 32x32x16 instructions; fp32 on the bf16 one, each value as the exact sum of three
// bf16 pieces (to nearest, 8 + 8 + 8 bits) and each product as the six piece products that reach above 2^-24 of it —
// fp32's own accuracy (test_gpu_set_attention.py holds it to fp32 tolerances) at 6/16 of the fp32 instruction's cycles.  An
// infinite fp32 input makes NaN of its rows.  Scores, softmax statistics, delta and every accumulator are fp32; in the
// 16-bit types P and dS are factors in two parts, each to nearest; fp16's are held times a power of two.
#include "common.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace cmvae {
namespace sa {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const char *q, *k, *v, *doo, *att, *att_low;
    char *o, *ocopy, *olow, *dq, *dk, *dv;
    float *lse, *delta, *part, *part_ml;
    const int *q_len, *k_len;
    long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, g_sb, g_ss, g_sh;   // strides in elements
    int B, Sq, Sk, H, Hkv, G, R, causal, residual, nsplit, ntiles, sg, fold, piece;
    float scale, c;                                                                // c = scale * log2(e)
};

// fp16 probabilities are held times 2^15 as factors: p <= 1 fits (32768 < 65504), and a row of many keys, whose p are
// under fp16's smallest normal 2^-14, keeps 11 bits of each.  The other types have fp32's exponents.
template <typename T> __device__ constexpr float p_shift() { return std::is_same<T, _Float16>::value ? 15.f : 0.f; }
// fp16's dS, whose size is that of the gradients, times p, is held times a power of two of its own, see fit_ds(): at first this
template <typename T> __device__ constexpr float ds_scale() { return std::is_same<T, _Float16>::value ? 0x1p48f : 1.f; }

template <typename T>
struct Vec8 {};
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

// What the matrix instructions take for a T: itself, or three bf16 planes for fp32.
template <typename T> struct Elem { typedef T type; static constexpr int P = 1; };
template <> struct Elem<float> { typedef __bf16 type; static constexpr int P = 3; };

// Second factor of a product over D channels, 32 columns: D / 2 values per lane.
template <typename T, int D>
struct Frag {
    u32x4 x[Elem<T>::P][D / 16];
};

// x - (one half of a packed bf16 pair) in one v_dot2c_f32_bf16 with (-1, 0) / (0, -1); the selectors are made once per kernel
// and kept in registers (as an inline constant the assembler's -1.0 is not the packed pattern).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
struct Sel {
    bf16x2 lo, hi;
};
__device__ __forceinline__ Sel make_sel() {
    unsigned a = 0x0000bf80u, b = 0xbf800000u;
    asm volatile("" : "+v"(a), "+v"(b));
    return Sel{__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b)};
}
__device__ __forceinline__ void split2(float x, float y, const Sel& q, unsigned (&p)[3]) {
    const bf16x2 a = __builtin_convertvector(f32x2{x, y}, bf16x2);
    const float rx = __builtin_amdgcn_fdot2_f32_bf16(a, q.lo, x, false), ry = __builtin_amdgcn_fdot2_f32_bf16(a, q.hi, y, false);
    const bf16x2 b = __builtin_convertvector(f32x2{rx, ry}, bf16x2);
    const float sx = __builtin_amdgcn_fdot2_f32_bf16(b, q.lo, rx, false), sy = __builtin_amdgcn_fdot2_f32_bf16(b, q.hi, ry, false);
    p[0] = __builtin_bit_cast(unsigned, a);
    p[1] = __builtin_bit_cast(unsigned, b);
    p[2] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{sx, sy}, bf16x2));
}
__device__ __forceinline__ void split8(const float (&v)[8], const Sel& q, u32x4 (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned t[3];
        split2(v[2 * i], v[2 * i + 1], q, t);
#pragma unroll
        for (int j = 0; j < 3; ++j) p[j][i] = t[j];
    }
}

template <typename T>
__device__ __forceinline__ f32x16 mma16(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (std::is_same<T, __bf16>::value)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// a product of P planes each, small terms first
template <typename T>
__device__ __forceinline__ f32x16 mma(const u32x4 (&a)[Elem<T>::P], const u32x4 (&b)[Elem<T>::P], f32x16 c) {
    typedef typename Elem<T>::type E;
    if constexpr (Elem<T>::P == 3) {
        c = mma16<E>(a[2], b[0], c);
        c = mma16<E>(a[0], b[2], c);
        c = mma16<E>(a[1], b[1], c);
        c = mma16<E>(a[1], b[0], c);
        c = mma16<E>(a[0], b[1], c);
    }
    return mma16<E>(a[0], b[0], c);
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// 2^x, results under 2^-126 as 0 (a weight that small adds nothing to a sum that holds a 1)
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// the value of the lane 32 places away
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// row of accumulator register r in a 32 x 32 tile, for lane half h
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

// The LDS pitch of a tile row: 16 bytes more than the row, so that the 32 rows of a fragment read start in different banks.
template <int D> __host__ __device__ constexpr int pitch() { return D * 2 + 16; }

// ---- first factor = 32 rows of an LDS tile of ROWS rows (P planes), contraction over the D channels ------------------
// The contraction's order is free as long as both factors agree: lane half h takes channels 16c + 8h .. + 7, one 16-byte
// read per plane.
template <typename T, int D, int ROWS>
__device__ __forceinline__ f32x16 mul_rows(const char* tile, int row0, const Frag<T, D>& b, f32x16 acc) {
    constexpr int P = Elem<T>::P;
    const int lane = threadIdx.x & 63;
    const char* p = tile + (row0 + (lane & 31)) * pitch<D>() + (lane >> 5) * 16;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        u32x4 a[P], y[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            a[i] = *reinterpret_cast<const u32x4*>(p + i * ROWS * pitch<D>() + c * 32);
            y[i] = b.x[i][c];
        }
        acc = mma<T>(a, y, acc);
    }
    return acc;
}

// ---- first factor = 32 channels x 32 rows of an LDS tile (transposed), second factor = a 32 x 32 accumulator --------
// Register r of the accumulator is tile row acc_row(r, h), which fixes the contraction's order: registers 8s .. 8s + 7 are
// one instruction's eight; the matching first factor — four rows at one channel, twice — comes from the transposing LDS
// read (16 lanes name 4 rows x 16 channels, lane i receives channel i of the four rows).
//   16-bit types: the accumulator is a factor twice, as its rounding and as what that leaves.  Every result's error (2-norm,
// against float64) is then that of its own rounding, to three digits (fp16's dq and dk within 4 %); with one factor o's was 1.16
// to 1.31 times that, dq's 1.5 and dk's and dv's 1.42.  One factor (two for dq alone) against two, us: forward + backward of 2 x
// 4096 causal rows x 16 heads of 128 bf16 870 / 1005, of 8 x 777 against 2049 x 8 heads of 64 fp16 168 / 190; forward of one token
// x 32 heads of 128 against 16 lists of up to 8191 75.5 / 78.5; dense 8 x 4096 x 16 heads bf16, forward 805 / 1060 (heads of 64)
// and 1524 / 1790 (128), dk dv 1500 / 1990 and 3720 / 4500.
template <typename T, int D, int ROWS>
__device__ __forceinline__ void mul_cols(const char* tile, int row0, const f32x16& w, const Sel& sel, f32x16 (&acc)[D / 32]) {
    constexpr int P = Elem<T>::P;
    typedef __attribute__((address_space(3))) s16x4 lds4;
    const int lane = threadIdx.x & 63, h = lane >> 5, i = lane & 15;
    const char* p = tile + (row0 + 4 * h + (i >> 2)) * pitch<D>() + (lane & 16) * 2 + (i & 3) * 8;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        u32x4 b[P], low[P];
        if constexpr (P == 3) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = w[8 * s + j];
            split8(v, sel, b);
        } else {
            typename Vec8<T>::type v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (T)w[8 * s + j];
            b[0] = __builtin_bit_cast(u32x4, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (T)(w[8 * s + j] - (float)v[j]);
            low[0] = __builtin_bit_cast(u32x4, v);
        }
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            u32x4 a[P];
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const char* at = p + (k * ROWS + 16 * s) * pitch<D>() + d * 64;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 8 * pitch<D>()));
                a[k] = __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
            acc[d] = mma<T>(a, b, acc[d]);
            if constexpr (P == 1) acc[d] = mma<T>(a, low, acc[d]);
        }
    }
}

// fp16: dS as a factor needs a scale.  Unscaled, values under 2^-25 were 0 and those over 65504 infinite — p of 1 / 4096 takes
// gradients of size 1e-3 to the one end (dq off by 0.5 %), a loss scale takes them to the other.  A lane's column (a query row in
// dq, a key in dk) holds dS f, f a power of two; where a tile brings a value over 2^15, f, that tile and the sums so far are
// scaled down until the largest is in [2^12, 2^13) (exactly: f starts at 2^48 and dS f is fp32's until it is rounded).  What is
// rounded as a subnormal is then 2^26 times smaller than the column's largest value, or under 2^-62.  The lane's other half has the
// rest of its column; the branch is the wave's, and taken for a column's first tile and a few more.  Forward + backward of 2 x
// 4096 causal rows x 16 heads of 128 920 -> 996 us, of dense 8 x 4096 x 16 heads of 64 3300 -> 3460; bf16 needs none of it
// (both before the factors' second parts).
template <int N>
__device__ __forceinline__ void fit_ds(f32x16& s, f32x16 (&acc)[N], float& f) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(s[i]));
    if (__ballot(mx > 0x1p15f) == 0) return;
    mx = fmaxf(mx, other_half(mx));
    const int down = mx > 0x1p15f && mx < INFINITY ? (__float_as_int(mx) >> 23) - (127 + 12) : 0;
    const float by = __int_as_float((127 - down) << 23);
    s *= by;
#pragma unroll
    for (int d = 0; d < N; ++d) acc[d] *= by;
    f *= by;
}

// eight channels of a row as fp32
template <typename T>
__device__ __forceinline__ void load8(const char* p, float (&v)[8]) {
    if constexpr (std::is_same<T, float>::value) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    } else {
        const typename Vec8<T>::type a = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
    }
}

// one row as a second factor (lane & 31 = column); rows that are not there are zero
template <typename T, int D>
__device__ __forceinline__ Frag<T, D> load_frag(const char* row, bool there, const Sel& sel) {
    const int h = (threadIdx.x & 63) >> 5;
    Frag<T, D> f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const char* p = row + (16 * c + 8 * h) * sizeof(T);
        if constexpr (Elem<T>::P == 3) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (there) load8<T>(p, v);
            u32x4 x[3];
            split8(v, sel, x);
#pragma unroll
            for (int i = 0; i < 3; ++i) f.x[i][c] = x[i];
        } else {
            f.x[0][c] = u32x4{0, 0, 0, 0};
            if (there) f.x[0][c] = *reinterpret_cast<const u32x4*>(p);
        }
    }
    return f;
}

// the product of two rows, each lane half over its half of the channels
template <typename T, int D>
__device__ __forceinline__ float dot_rows(const char* x, const char* y, bool there) {
    const int h = (threadIdx.x & 63) >> 5;
    float s = 0.f;
    if (there)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            float a[8], b[8];
            load8<T>(x + (16 * c + 8 * h) * sizeof(T), a);
            load8<T>(y + (16 * c + 8 * h) * sizeof(T), b);
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf(a[j], b[j], s);
        }
    return s + other_half(s);
}

// four channels of a row, fp32 -> T
template <typename T>
__device__ __forceinline__ void store4(char* p, float a, float b, float c, float d) {
    if constexpr (std::is_same<T, float>::value) {
        *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    } else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 v = {(T)a, (T)b, (T)c, (T)d};
        *reinterpret_cast<T4*>(p) = v;
    }
}
template <typename T>
__device__ __forceinline__ f32x4 load4(const char* p) {
    if constexpr (std::is_same<T, float>::value) {
        return *reinterpret_cast<const f32x4*>(p);
    } else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const T4 v = *reinterpret_cast<const T4*>(p);
        return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    }
}

// one piece of a result row: o without the residual (16-bit types: and what its rounding leaves, so that the backward's delta is
// not that of a rounded o, which would leave dq's error at 1.07 to 1.11 times its own rounding's and dk's at up to 1.05), and o
template <typename T>
__device__ __forceinline__ void store_o(const Args& a, long at, const char* residual, f32x4 o) {
    if (a.ocopy) store4<T>(a.ocopy + at, o[0], o[1], o[2], o[3]);
    if (!std::is_same<T, float>::value && a.olow)
        store4<T>(a.olow + at, o[0] - (float)(T)o[0], o[1] - (float)(T)o[1], o[2] - (float)(T)o[2], o[3] - (float)(T)o[3]);
    if (residual) o += load4<T>(residual);
    store4<T>(a.o + at, o[0], o[1], o[2], o[3]);
}

// ---- tiles of ROWS rows through registers into LDS: requested while the previous tile is used -----------------------
// A thread's pieces lie STEP rows apart, so their addresses are one 32-bit offset per thread on top of a scalar base (with a
// 64-bit product per piece and tile instead, and a division per piece on the key side, dk and dv of dense 8 x 4096 x 16 heads
// of 64 bf16 took 1579 us for 1380).
template <typename T, int D, int ROWS, int THREADS>
struct Stage {
    static constexpr int CPR = D * sizeof(T) / 16;               // 16-byte pieces per row
    static constexpr int N = ROWS * CPR / THREADS, STEP = THREADS / CPR;
    static_assert(ROWS * CPR % THREADS == 0 && THREADS % CPR == 0, "whole pieces per thread");
    u32x4 x[N];
    __device__ __forceinline__ static int tid() { return (int)threadIdx.x % THREADS; }
    __device__ __forceinline__ static unsigned offset(long stride) {
        return (unsigned)(tid() / CPR * (int)stride + tid() % CPR * 16);
    }
    // `left` rows from `base` on, the others are zeros
    __device__ __forceinline__ void load(const char* base, long stride, unsigned off, int left) {
        if (left >= ROWS) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = *reinterpret_cast<const u32x4*>(base + i * STEP * stride + off);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[i] = u32x4{0, 0, 0, 0};
                if (i * STEP + tid() / CPR < left) x[i] = *reinterpret_cast<const u32x4*>(base + i * STEP * stride + off);
            }
        }
    }
    // rows of a key head's list from (g, pos) on, `left` of them to the list's end, through more than one head
    __device__ __forceinline__ void load_across(const char* base, long ss, long sh, int g, int pos, int left, int ql) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = i * STEP + tid() / CPR;
            x[i] = u32x4{0, 0, 0, 0};
            if (j < left) {
                const int q = (pos + j) / ql;
                x[i] = *reinterpret_cast<const u32x4*>(base + (pos + j - q * ql) * ss + (g + q) * sh + tid() % CPR * 16);
            }
        }
    }
    __device__ __forceinline__ void put(char* tile, const Sel& sel) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = i * THREADS + tid();
            char* at = tile + (id / CPR) * pitch<D>() + (id % CPR) * (Elem<T>::P == 3 ? 8 : 16);
            if constexpr (Elem<T>::P == 3) {
                const f32x4 v = __builtin_bit_cast(f32x4, x[i]);
                unsigned a[3], b[3];
                split2(v[0], v[1], sel, a);
                split2(v[2], v[3], sel, b);
#pragma unroll
                for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2*>(at + k * ROWS * pitch<D>()) = make_uint2(a[k], b[k]);
            } else {
                *reinterpret_cast<u32x4*>(at) = x[i];
            }
        }
    }
};

__device__ __forceinline__ void lens(const Args& a, int b, int& ql, int& kl) {
    ql = a.Sq;
    kl = a.Sk;
    if (a.q_len) ql = min(max(a.q_len[b], 0), a.Sq);
    if (a.k_len) kl = min(max(a.k_len[b], 0), a.Sk);
}

struct Place {           // what a workgroup works on
    int b, kh, tile, split, ql, kl;
};

// Which piece of work a workgroup takes.  A compute unit holds few workgroups, each of them long, so what matters is that its
// sum is near the others'.
//   Lengths given (and up to 64 batch entries): every workgroup ranks the entries by the length that its side walks, one lane
//   per entry, and the tiles are dealt longest first, those without a valid row last.
//   Otherwise: (batch, key head) runs fastest — with a multiple of 8 of them each stays on one XCD, whose L2 then holds its
//   keys — and the causal order's longest tiles come first.
// With one to two workgroups per compute unit the second ones are dealt shortest first: each joins a long one.
// Measured on 16 padded sets of 383 to 1531 rows, fp32, against plain order: forward 371 -> 229 us, dq 522 -> 312, dk and dv
// 690 -> 484.
template <int ROWS, bool KEYS>
__device__ __forceinline__ Place place(const Args& a) {
    Place p;
    int id = blockIdx.x;
    const int lane = threadIdx.x & 63;
    // one to two workgroups per compute unit, both resident: the second ones are dealt shortest first, each joins a long one
    auto fold = [&](int jobs) {
        if (jobs > a.fold && jobs <= 2 * a.fold && id >= a.fold && id < jobs) id = a.fold + jobs - 1 - id;
    };
    // the causal order's longest tiles first: of a list of n tiles that runs through G heads, every head's last one, then every
    // head's last but one ...
    auto longest_first = [&](int i, int n) {
        if (!a.causal || KEYS) return i;
        const int per = n / a.G, more = n - per * a.G;             // the first `more` heads have per + 1 tiles
        int round = i / a.G, g = i - round * a.G;
        return (g + 1) * per + min(g + 1, more) - 1 - round;
    };
    if ((a.q_len || a.k_len) && a.B <= 64) {
        int ql, kl, nt = 0, w = 0;
        lens(a, lane < a.B ? lane : 0, ql, kl);
        if (lane < a.B) {
            nt = KEYS ? (kl + ROWS - 1) / ROWS : (a.G * ql + ROWS - 1) / ROWS;
            w = KEYS ? ql : kl;
        }
        int start = 0, zeros = 0, total = 0;               // tiles before this lane's entry's, tiles without a row before them
        for (int i = 0; i < a.B; ++i) {
            const int wi = __builtin_amdgcn_readlane(w, i), ni = __builtin_amdgcn_readlane(nt, i);
            start += wi > w || (wi == w && i < lane) ? ni : 0;
            zeros += i < lane ? a.ntiles - ni : 0;
            total += ni;
        }
        fold(total * a.Hkv * a.nsplit);
        p.split = id % a.nsplit;
        id /= a.nsplit;
        p.kh = id % a.Hkv;
        id /= a.Hkv;
        const bool some = id < total;
        const int at = some ? id - start : id - total - zeros;
        const unsigned long long mine = __ballot(lane < a.B && at >= 0 && at < (some ? nt : a.ntiles - nt));
        p.b = __ffsll((long long)mine) - 1;
        const int t = __builtin_amdgcn_readlane(at, p.b), n = __builtin_amdgcn_readlane(nt, p.b);
        p.tile = some ? longest_first(t, n) : n + t;
        p.ql = __builtin_amdgcn_readlane(ql, p.b);
        p.kl = __builtin_amdgcn_readlane(kl, p.b);
        return p;
    }
    const int nbh = a.B * a.Hkv;
    if (a.causal) fold(nbh * a.ntiles * a.nsplit);
    const int bh = id % nbh;
    id /= nbh;
    p.split = id % a.nsplit;
    id /= a.nsplit;
    p.tile = longest_first(id, a.ntiles);
    p.b = bh / a.Hkv;
    p.kh = bh - p.b * a.Hkv;
    lens(a, p.b, p.ql, p.kl);
    return p;
}

// row r of a key head's list: its head in the group and its position; whether it counts
struct Row {
    int g, pos;
    bool ok;
};
__device__ __forceinline__ Row row_of(const Args& a, int ql, int r) {
    const int valid = a.G * ql;
    Row w;
    w.ok = r < valid;
    const int x = w.ok ? r : r - valid, n = w.ok ? ql : a.Sq - ql;
    w.g = n > 0 ? x / n : 0;
    w.pos = x - w.g * n + (w.ok ? 0 : ql);
    return w;
}

// positions [lo, hi] that the valid rows r0 .. r1 - 1 of a key head's list cover
__device__ __forceinline__ void span(int ql, int r0, int r1, int& lo, int& hi) {
    const int g0 = r0 / ql, g1 = (r1 - 1) / ql;
    lo = g0 == g1 ? r0 - g0 * ql : 0;
    hi = g0 == g1 ? r1 - 1 - g0 * ql : ql - 1;
}

// Waves of a workgroup: NW waves of 32 own rows that share the tiles they walk (two buffers, one barrier per tile) — or, where
// there are few rows, WS waves that share the same 32 own rows and walk every WS-th tile, each in a buffer of its own without
// a barrier, and meet at the end: one launch where pieces of the walk would need a second one to join them.
template <typename T, int D>
constexpr int walkers() { return sizeof(T) * D > 256 ? 2 : 4; }      // fp32 heads of 128: 52 KB of planes per wave

// orders a wave's own LDS accesses across its lanes (the hardware runs them in order; this keeps the compiler to it)
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// wave w > 0 hands an accumulator to wave 0 (the buffers are free: all waves are through)
template <int WS, int N>
__device__ __forceinline__ void hand_over(char* smem, int w, const f32x16 (&acc)[N]) {
    __syncthreads();
    if (w > 0)
#pragma unroll
        for (int d = 0; d < N; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                reinterpret_cast<f32x4*>(smem)[(((w - 1) * N + d) * 4 + q) * 64 + (threadIdx.x & 63)] =
                    f32x4{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]};
    __syncthreads();
}
template <int N>
__device__ __forceinline__ void take_over(const char* smem, int w, float f, f32x16 (&acc)[N]) {
#pragma unroll
    for (int d = 0; d < N; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 x = reinterpret_cast<const f32x4*>(smem)[(((w - 1) * N + d) * 4 + q) * 64 + (threadIdx.x & 63)];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[d][4 * q + j] = fmaf(x[j], f, acc[d][4 * q + j]);
        }
}

// ------------------------------------------------------------------------------------------------ forward
// Keys in tiles of KT through LDS.  Running maximum m (log2 units) and sum l per row.  nsplit > 1: a workgroup covers one
// piece of the tiles and leaves (acc, m, l) for the joining kernel.
//   Bound by the matrix instructions and, between them, the exponentials and the LDS reads that feed them: with two workgroups
// per unit one computes while the other waits.  Dense 8 x 4096 x 16 heads, bf16: 520 TFLOP/s with 64 channels, 610 with 128, P's
// second part, half as much again, not counted (a large library product reaches 1390); fp32 (six bf16 products each), 8 x 2048 x
// 8 heads: 173 and 150 (the library's fp32 product 153).
template <typename T, int D, int NW, int KT, int WS>
__global__ __launch_bounds__(NW * WS * 64, NW == 4 && sizeof(T) * D <= 256 ? 2 : 1) void fwd_kernel(Args a) {
    extern __shared__ __align__(16) char smem[];
    constexpr int TB = Elem<T>::P * KT * pitch<D>();
    const Place pl = place<NW * 32, false>(a);
    const Sel sel = make_sel();
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
    const int ql = pl.ql, kl = pl.kl, rv = a.G * ql;
    const int r0 = pl.tile * NW * 32, r = r0 + (WS > 1 ? 0 : w) * 32 + (lane & 31);
    const Row me = row_of(a, ql, r);
    const int g = me.g, pos = me.pos;
    const bool row_ok = me.ok;
    const int off = kl - ql;
    int lo = 0, kend = 0;
    if (r0 < rv) {
        int hi;
        span(ql, r0, min(r0 + NW * 32, rv), lo, hi);
        kend = a.causal ? min(kl, hi + off + 1) : kl;
    }
    int t0 = 0, t1 = (max(kend, 0) + KT - 1) / KT;
    if (a.nsplit > 1) {                           // the pieces follow the keys that there are
        const int per = (t1 + a.nsplit - 1) / a.nsplit;
        t0 = pl.split * per;
        t1 = min(t1, t0 + per);
    }
    const long es = sizeof(T);
    const char* kb = a.k + (pl.b * a.k_sb + pl.kh * a.k_sh) * es;
    const char* vb = a.v + (pl.b * a.v_sb + pl.kh * a.v_sh) * es;
    const char* qrow = a.q + (pl.b * a.q_sb + pos * a.q_ss + (pl.kh * a.G + g) * a.q_sh) * es;
    const Frag<T, D> qf = load_frag<T, D>(qrow, row_ok, sel);
    f32x16 acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;
    const int klast = a.causal ? min(kl, pos + off + 1) : kl;      // this row's keys end here

    typedef Stage<T, D, KT, NW * 64> St;
    St ks, vs;
    const long ksb = a.k_ss * es, vsb = a.v_ss * es;
    const unsigned ko = St::offset(ksb), vo = St::offset(vsb);
    auto request = [&](int t) {
        ks.load(kb + (long)t * KT * ksb, ksb, ko, kl - t * KT);
        vs.load(vb + (long)t * KT * vsb, vsb, vo, kl - t * KT);
    };
    auto use = [&](int t, const char* kt, const char* vt) {
        f32x16 s[KT / 32];
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) s[u] = mul_rows<T, D, KT>(kt, u * 32, qf, zero16());
        const int k0 = t * KT;
        if (k0 + KT > kl || (a.causal && k0 + KT > lo + off + 1)) {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + u * 32 + acc_row(i, h) >= klast) s[u][i] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
        mx = fmaxf(mx, other_half(mx));
        const float mn = fmaxf(m, mx * a.c);
        const float mu = mn == -INFINITY ? 0.f : mn;               // a row without a valid key so far: every p is 0
        const float al = exp2_raw(m - mu), sub = mu - p_shift<T>();
        m = mn;
        float ps = 0.f;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = exp2_raw(fmaf(s[u][i], a.c, -sub));
                ps += s[u][i];
            }
        l = fmaf(l, al, ps);
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] *= al;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) mul_cols<T, D, KT>(vt, u * 32, s[u], sel, acc);
    };
    if constexpr (WS > 1) {
        char* my = smem + w * 2 * TB;
        int t = t0 + w;
        if (t < t1) request(t);
        for (; t < t1; t += WS) {
            ks.put(my, sel);
            vs.put(my + TB, sel);
            wave_sync();
            if (t + WS < t1) request(t + WS);
            use(t, my, my + TB);
            wave_sync();
        }
    } else {
        if (t0 < t1) {
            request(t0);
            ks.put(smem, sel);
            vs.put(smem + TB, sel);
        }
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            const char* kt = smem + ((t - t0) & 1) * 2 * TB;
            if (t + 1 < t1) request(t + 1);
            use(t, kt, kt + TB);
            if (t + 1 < t1) {
                char* nx = smem + ((t + 1 - t0) & 1) * 2 * TB;
                ks.put(nx, sel);
                vs.put(nx + TB, sel);
            }
            __syncthreads();
        }
    }
    l += other_half(l);
    if constexpr (WS > 1) {
        __shared__ float sm[WS][64], sl[WS][64];
        sm[w][lane] = m;
        sl[w][lane] = l;
        hand_over<WS>(smem, w, acc);
        if (w > 0) return;
        float mx = m;
#pragma unroll
        for (int i = 1; i < WS; ++i) mx = fmaxf(mx, sm[i][lane]);
        const float mu = mx == -INFINITY ? 0.f : mx, f0 = exp2_raw(m - mu);
        l *= f0;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] *= f0;
#pragma unroll
        for (int i = 1; i < WS; ++i) {
            const float fi = exp2_raw(sm[i][lane] - mu);
            l = fmaf(sl[i][lane], fi, l);
            take_over(smem, i, fi, acc);
        }
        m = mx;
    }
    if (r >= a.R) return;
    const long hrow = ((long)pl.b * a.H + pl.kh * a.G + g) * a.Sq + pos;
    if (a.nsplit > 1) {
        const long prow = (long)pl.split * a.B * a.Hkv * a.R + hrow;
        float* po = a.part + prow * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<float4*>(po + d * 32 + 8 * q4 + 4 * h) =
                    make_float4(acc[d][4 * q4], acc[d][4 * q4 + 1], acc[d][4 * q4 + 2], acc[d][4 * q4 + 3]);
        if (h == 0) {
            a.part_ml[prow * 2] = m;
            a.part_ml[prow * 2 + 1] = l;
        }
        return;
    }
    const float inv = row_ok && l != 0.f ? 1.f / l : 0.f;
    if (h == 0 && a.lse) a.lse[hrow] = row_ok && l != 0.f ? m - p_shift<T>() + log2f(l) : INFINITY;
    const long orow = (((long)pl.b * a.Sq + pos) * a.H + pl.kh * a.G + g) * D * es;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const long at = (d * 32 + 8 * q4 + 4 * h) * es;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            if (row_ok && l != 0.f)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = acc[d][4 * q4 + j] * inv;
            store_o<T>(a, orow + at, a.residual && row_ok ? qrow + at : nullptr, o);
        }
}

// ------------------------------------------------------------------------------------------------ forward of few rows
// A key head's list of a few rows (one new token, a set's summary by one query; most_rows()) against many keys: the
// keys and values are read once, and that is the time.  No LDS, no matrix instruction (32 columns of which 1 .. 8 count):
// a row of keys lies over CL lanes, 16 bytes each, 64 / CL keys per wave and step, U steps' loads in flight; a score is the
// sum over the CL lanes, a lane keeps its channels' sums for its keys and its own running maximum, and the waves join at the
// end.  16-bit values meet in v_dot2 (two products per instruction): scores over channel pairs, sums over pairs of keys.
// A workgroup takes `piece` keys; pieces of a list are joined by fwd_join_kernel.  Reads 5.3 TB/s at 16 lists of 8191 keys x 8 heads
// of 128 (bf16 and fp32), 4.7 at 4 of 6400 x 4 heads of 64 fp32 (11 us).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}
template <int CL>
__device__ __forceinline__ float sum_lanes(float x) {
    x += dpp<0xB1>(x);                            // lane ^ 1
    x += dpp<0x4E>(x);                            // lane ^ 2
    x += dpp<0x141>(x);                           // the other four of eight
    if constexpr (CL >= 16) x += dpp<0x140>(x);   // the other eight of sixteen
    if constexpr (CL >= 32) x += __shfl_xor(x, 16);
    return x;
}
__device__ __forceinline__ float dot2(unsigned a, unsigned b, float c, __bf16) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a), __builtin_bit_cast(bf16x2, b), c, false);
}
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float dot2(unsigned a, unsigned b, float c, _Float16) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, a), __builtin_bit_cast(f16x2, b), c, false);
}
// two values as their roundings and as what those leave
template <typename T>
__device__ __forceinline__ void two_parts(float x, float y, unsigned (&p)[2]) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    const T2 a = __builtin_convertvector(f32x2{x, y}, T2);
    p[0] = __builtin_bit_cast(unsigned, a);
    p[1] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x - (float)a[0], y - (float)a[1]}, T2));
}

template <typename T, int D, int R>
__global__ __launch_bounds__(256) void fwd_rows_kernel(Args a) {
    constexpr int CL = D * sizeof(T) / 16, KP = 64 / CL, E = 16 / sizeof(T), U = 4;
    constexpr int STEP = U * KP;                                    // keys per wave and round
    __shared__ float sm[4][R], sl[4][R];
    __shared__ float so[4][R][D];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, ch = lane % CL, kg = lane / CL;
    const int nbh = a.B * a.Hkv, bh = (int)blockIdx.x % nbh, split = (int)blockIdx.x / nbh;
    const int b = bh / a.Hkv, kh = bh - b * a.Hkv;
    int ql, kl;
    lens(a, b, ql, kl);
    const int rv = a.G * ql, off = kl - ql;
    const long es = sizeof(T);
    const int k0 = split * a.piece, k1 = min(kl, k0 + a.piece);
    const char* kb = a.k + (b * a.k_sb + kh * a.k_sh) * es + ch * 16;
    const char* vb = a.v + (b * a.v_sb + kh * a.v_sh) * es + ch * 16;
    u32x4 q[R];
    int last[R];                                                    // row r's keys end here
    float m[R], l[R], acc[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        q[r] = u32x4{0, 0, 0, 0};
        last[r] = 0;
        if (r < rv) {
            const int g = r / ql, pos = r - g * ql;
            q[r] = *reinterpret_cast<const u32x4*>(a.q + (b * a.q_sb + pos * a.q_ss + (kh * a.G + g) * a.q_sh) * es + ch * 16);
            last[r] = a.causal ? min(kl, pos + off + 1) : kl;
        }
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.f;
    }
    for (int kc = k0 + w * STEP; kc < k1; kc += 4 * STEP) {
        u32x4 kv[U], vv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = kc + u * KP + kg;
            kv[u] = vv[u] = u32x4{0, 0, 0, 0};
            if (key < k1) {
                kv[u] = *reinterpret_cast<const u32x4*>(kb + key * a.k_ss * es);
                vv[u] = *reinterpret_cast<const u32x4*>(vb + key * a.v_ss * es);
            }
        }
        float p[R][U];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float s = 0.f;
                if constexpr (std::is_same<T, float>::value) {
                    const f32x4 x = __builtin_bit_cast(f32x4, q[r]), y = __builtin_bit_cast(f32x4, kv[u]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s = fmaf(x[e], y[e], s);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s = dot2(q[r][e], kv[u][e], s, T());
                }
                s = sum_lanes<CL>(s);
                p[r][u] = kc + u * KP + kg < last[r] ? s : -INFINITY;
                mx = fmaxf(mx, p[r][u] * a.c);
            }
            const float mu = mx == -INFINITY ? 0.f : mx, al = exp2_raw(m[r] - mu), sub = mu - p_shift<T>();
            m[r] = mx;
            float ps = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                p[r][u] = exp2_raw(fmaf(p[r][u], a.c, -sub));
                ps += p[r][u];
            }
            l[r] = fmaf(l[r], al, ps);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] *= al;
        }
        if constexpr (std::is_same<T, float>::value) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const f32x4 y = __builtin_bit_cast(f32x4, vv[u]);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r][e] = fmaf(p[r][u], y[e], acc[r][e]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; u += 2) {                        // two keys' values at one channel beside each other
                unsigned y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[2 * e] = __builtin_amdgcn_perm(vv[u + 1][e], vv[u][e], 0x05040100);
                    y[2 * e + 1] = __builtin_amdgcn_perm(vv[u + 1][e], vv[u][e], 0x07060302);
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    unsigned pp[2];                                 // as in mul_cols(): p's rounding and what that leaves
                    two_parts<T>(p[r][u], p[r][u + 1], pp);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[r][e] = dot2(pp[0], y[e], dot2(pp[1], y[e], acc[r][e], T()), T());
                }
            }
        }
    }
    // the wave's key groups meet, then the waves
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float mx = m[r];
#pragma unroll
        for (int o = CL; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        const float f = exp2_raw(m[r] - (mx == -INFINITY ? 0.f : mx));
        float ls = l[r] * f;
#pragma unroll
        for (int o = CL; o < 64; o <<= 1) ls += __shfl_xor(ls, o);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float x = acc[r][e] * f;
#pragma unroll
            for (int o = CL; o < 64; o <<= 1) x += __shfl_xor(x, o);
            if (kg == 0) so[w][r][ch * E + e] = x;
        }
        if (lane == 0) {
            sm[w][r] = mx;
            sl[w][r] = ls;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.R * (D / 4); i += 256) {
        const int r = i / (D / 4), d4 = i - r * (D / 4);
        const Row me = row_of(a, ql, r);
        float mx = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        const float mu = mx == -INFINITY ? 0.f : mx;
        float ls = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float f = exp2_raw(sm[j][r] - mu);
            ls = fmaf(sl[j][r], f, ls);
            const f32x4 x = *reinterpret_cast<const f32x4*>(&so[j][r][d4 * 4]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
        }
        const long hrow = ((long)b * a.H + kh * a.G + me.g) * a.Sq + me.pos;
        if (a.nsplit > 1) {
            const long prow = (long)split * nbh * a.R + hrow;
            if (d4 == 0) {
                a.part_ml[prow * 2] = mx;
                a.part_ml[prow * 2 + 1] = ls;
            }
            if (mx != -INFINITY) *reinterpret_cast<f32x4*>(a.part + prow * D + d4 * 4) = o;
            continue;
        }
        const bool ok = me.ok && ls != 0.f;
        if (d4 == 0 && a.lse) a.lse[hrow] = ok ? mx - p_shift<T>() + log2f(ls) : INFINITY;
        const float inv = ok ? 1.f / ls : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = ok ? o[e] * inv : 0.f;
        const long at = ((((long)b * a.Sq + me.pos) * a.H + kh * a.G + me.g) * D + d4 * 4) * es;
        store_o<T>(a, at, a.residual && me.ok ? a.q + (b * a.q_sb + me.pos * a.q_ss + (kh * a.G + me.g) * a.q_sh + d4 * 4) * es : nullptr,
                   o);
    }
}

// Joins the splits of a row: D / 4 lanes per row times SG groups that share its splits out (SG from the host: few rows of
// many splits would otherwise be a long walk on a handful of lanes; 16 rows of 50 splits took 24 us that way).  One pass with a
// running maximum, its loads ahead of it: 4.7 us there, 6.0 with a pass of its own for the maximum.
template <typename T, int D>
__global__ __launch_bounds__(256) void fwd_join_kernel(Args a) {
    constexpr int LPR = D / 4;
    __shared__ float sm[256], sl[256];
    __shared__ f32x4 so[256];
    const long rows = (long)a.B * a.Hkv * a.R;
    const int rpb = 256 / LPR / a.sg, lr = (int)threadIdx.x / (LPR * a.sg);
    const int d4 = threadIdx.x % LPR, sg = (int)threadIdx.x / LPR % a.sg;
    const long row = (long)blockIdx.x * rpb + lr;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (row < rows) {
#pragma unroll 4
        for (int s = sg; s < a.nsplit; s += a.sg) {
            const long at = s * rows + row;
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
            f32x4 p = *reinterpret_cast<const f32x4*>(a.part + at * D + d4 * 4);
            const float mx = fmaxf(m, ml.x), mu = mx == -INFINITY ? 0.f : mx;
            const float f = exp2_raw(m - mu), wgt = exp2_raw(ml.x - mu);
            if (ml.x == -INFINITY) p = f32x4{0.f, 0.f, 0.f, 0.f};   // a piece without a valid key: its sums may not have been written
            m = mx;
            l = fmaf(wgt, ml.y, l * f);
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(wgt, p[j], o[j] * f);
        }
    }
    if (a.sg > 1) {
        sm[threadIdx.x] = m;
        sl[threadIdx.x] = l;
        so[threadIdx.x] = o;
        __syncthreads();
        if (sg != 0) return;
        for (int i = 1; i < a.sg; ++i) m = fmaxf(m, sm[threadIdx.x + i * LPR]);
        const float mu = m == -INFINITY ? 0.f : m;
        l = 0.f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < a.sg; ++i) {
            const float wgt = exp2_raw(sm[threadIdx.x + i * LPR] - mu);
            l = fmaf(wgt, sl[threadIdx.x + i * LPR], l);
            const f32x4 p = so[threadIdx.x + i * LPR];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = fmaf(wgt, p[j], o[j]);
        }
    }
    if (row >= rows) return;
    const int b = (int)(row / ((long)a.H * a.Sq));
    const int rest = (int)(row - (long)b * a.H * a.Sq), head = rest / a.Sq, pos = rest - head * a.Sq;
    int ql, kl;
    lens(a, b, ql, kl);
    const bool ok = pos < ql && l != 0.f;
    if (d4 == 0 && a.lse) a.lse[row] = ok ? m - p_shift<T>() + log2f(l) : INFINITY;
    const float inv = ok ? 1.f / l : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = ok ? o[j] * inv : 0.f;
    const long es = sizeof(T), at = ((((long)b * a.Sq + pos) * a.H + head) * D + d4 * 4) * es;
    store_o<T>(a, at, a.residual && pos < ql ? a.q + (b * a.q_sb + pos * a.q_ss + head * a.q_sh + d4 * 4) * es : nullptr, o);
}

// sum over the splits of the 4 values at `e` of n4, shared out over SG groups of 256 / SG threads; true in the group that
// has the sum
__device__ __forceinline__ bool join_sum(const Args& a, const float* part, long n4, long e, int sg, f32x4& x) {
    __shared__ f32x4 red[256];
    x = f32x4{0.f, 0.f, 0.f, 0.f};
    const int per = 256 / a.sg;
    if (e < n4)
        for (int s = sg; s < a.nsplit; s += a.sg) x += reinterpret_cast<const f32x4*>(part)[s * n4 + e];
    if (a.sg == 1) return true;
    __syncthreads();
    red[threadIdx.x] = x;
    __syncthreads();
    if (sg != 0) return false;
    for (int i = 1; i < a.sg; ++i) x += red[threadIdx.x + i * per];
    return true;
}

// ------------------------------------------------------------------------------------------------ backward, query side
// The forward's shape; delta_i from the saved o, kept for the key side.  Bound as the forward; at its dense sizes, counting three
// products, bf16 670 TFLOP/s with 64 channels and 710 with 128 (a fourth, of what dS's rounding leaves, not counted),
// fp32 203 and 175.
template <typename T, int D, int NW, int KT, int WS>
__global__ __launch_bounds__(NW * WS * 64, NW == 4 && sizeof(T) * D <= 256 ? 2 : 1) void dq_kernel(Args a) {
    extern __shared__ __align__(16) char smem[];
    constexpr int TB = Elem<T>::P * KT * pitch<D>();
    const Place pl = place<NW * 32, false>(a);
    const Sel sel = make_sel();
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
    const int ql = pl.ql, kl = pl.kl, rv = a.G * ql;
    const int r0 = pl.tile * NW * 32, r = r0 + (WS > 1 ? 0 : w) * 32 + (lane & 31);
    const Row me = row_of(a, ql, r);
    const int g = me.g, pos = me.pos;
    const bool row_ok = me.ok;
    const int off = kl - ql;
    int lo = 0, kend = 0;
    if (r0 < rv) {
        int hi;
        span(ql, r0, min(r0 + NW * 32, rv), lo, hi);
        kend = a.causal ? min(kl, hi + off + 1) : kl;
    }
    int t0 = 0, t1 = (max(kend, 0) + KT - 1) / KT;
    if (a.nsplit > 1) {                           // the pieces follow the keys that there are
        const int per = (t1 + a.nsplit - 1) / a.nsplit;
        t0 = pl.split * per;
        t1 = min(t1, t0 + per);
    }
    const long es = sizeof(T);
    const int head = pl.kh * a.G + g;
    const char* kb = a.k + (pl.b * a.k_sb + pl.kh * a.k_sh) * es;
    const char* vb = a.v + (pl.b * a.v_sb + pl.kh * a.v_sh) * es;
    const char* grow = a.doo + (pl.b * a.g_sb + pos * a.g_ss + head * a.g_sh) * es;
    const Frag<T, D> qf = load_frag<T, D>(a.q + (pl.b * a.q_sb + pos * a.q_ss + head * a.q_sh) * es, row_ok, sel);
    const Frag<T, D> gf = load_frag<T, D>(grow, row_ok, sel);
    const long hrow = ((long)pl.b * a.H + head) * a.Sq + pos;
    const long orow = (((long)pl.b * a.Sq + pos) * a.H + head) * D * es;
    float dl, lse = INFINITY, f = ds_scale<T>();
    {
        dl = dot_rows<T, D>(grow, a.att + orow, row_ok);
        if (a.att_low) dl += dot_rows<T, D>(grow, a.att_low + orow, row_ok);
        if (row_ok) lse = a.lse[hrow];
        if (h == 0 && r < a.R && pl.split == 0 && (WS == 1 || w == 0)) a.delta[hrow] = dl;
    }
    f32x16 acc[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) acc[d] = zero16();
    const int klast = a.causal ? min(kl, pos + off + 1) : kl;

    typedef Stage<T, D, KT, NW * 64> St;
    St ks, vs;
    const long ksb = a.k_ss * es, vsb = a.v_ss * es;
    const unsigned ko = St::offset(ksb), vo = St::offset(vsb);
    auto request = [&](int t) {
        ks.load(kb + (long)t * KT * ksb, ksb, ko, kl - t * KT);
        vs.load(vb + (long)t * KT * vsb, vsb, vo, kl - t * KT);
    };
    auto use = [&](int t, const char* kt, const char* vt) {
        const int k0 = t * KT;
        const bool edge = k0 + KT > kl || (a.causal && k0 + KT > lo + off + 1);
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
            f32x16 s = mul_rows<T, D, KT>(kt, u * 32, qf, zero16());
            f32x16 dp = mul_rows<T, D, KT>(vt, u * 32, gf, zero16());
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float d = std::is_same<T, _Float16>::value ? fmaf(dp[i], f, -dl * f) : dp[i] - dl;      // f: exact
                s[i] = exp2_raw(fmaf(s[i], a.c, -lse)) * d;
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (k0 + u * 32 + acc_row(i, h) >= klast) s[i] = 0.f;
            }
            if constexpr (std::is_same<T, _Float16>::value) fit_ds(s, acc, f);
            mul_cols<T, D, KT>(kt, u * 32, s, sel, acc);
        }
    };
    auto unscale = [&](f32x16 (&x)[D / 32]) {
        if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) x[d] *= 1.f / f;
    };
    if constexpr (WS > 1) {
        char* my = smem + w * 2 * TB;
        int t = t0 + w;
        if (t < t1) request(t);
        for (; t < t1; t += WS) {
            ks.put(my, sel);
            vs.put(my + TB, sel);
            wave_sync();
            if (t + WS < t1) request(t + WS);
            use(t, my, my + TB);
            wave_sync();
        }
        unscale(acc);
        hand_over<WS>(smem, w, acc);
        if (w > 0) return;
#pragma unroll
        for (int i = 1; i < WS; ++i) take_over(smem, i, 1.f, acc);
    } else {
        if (t0 < t1) {
            request(t0);
            ks.put(smem, sel);
            vs.put(smem + TB, sel);
        }
        __syncthreads();
        for (int t = t0; t < t1; ++t) {
            const char* kt = smem + ((t - t0) & 1) * 2 * TB;
            if (t + 1 < t1) request(t + 1);
            use(t, kt, kt + TB);
            if (t + 1 < t1) {
                char* nx = smem + ((t + 1 - t0) & 1) * 2 * TB;
                ks.put(nx, sel);
                vs.put(nx + TB, sel);
            }
            __syncthreads();
        }
        unscale(acc);
    }
    if (r >= a.R) return;
    float* po = a.nsplit > 1 ? a.part + ((long)pl.split * a.B * a.Hkv * a.R + hrow) * D : nullptr;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int ch = d * 32 + 8 * q4 + 4 * h;
            f32x4 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = row_ok ? acc[d][4 * q4 + j] * a.scale : 0.f;
            if (po) {
                *reinterpret_cast<f32x4*>(po + ch) = o;
            } else {
                if (a.residual && row_ok) o += load4<T>(grow + ch * es);
                store4<T>(a.dq + orow + ch * es, o[0], o[1], o[2], o[3]);
            }
        }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void dq_join_kernel(Args a) {
    constexpr int LPR = D / 4;
    const long rows = (long)a.B * a.Hkv * a.R;
    const int per = 256 / a.sg, sg = (int)threadIdx.x / per;
    const long e = (long)blockIdx.x * per + threadIdx.x - sg * per, row = e / LPR;
    const int d4 = (int)(e - row * LPR);
    f32x4 o;
    if (!join_sum(a, a.part, rows * LPR, e, sg, o) || row >= rows) return;
    const int b = (int)(row / ((long)a.H * a.Sq));
    const int rest = (int)(row - (long)b * a.H * a.Sq), head = rest / a.Sq, pos = rest - head * a.Sq;
    int ql, kl;
    lens(a, b, ql, kl);
    const long es = sizeof(T);
    if (a.residual && pos < ql) o += load4<T>(a.doo + (b * a.g_sb + pos * a.g_ss + head * a.g_sh + d4 * 4) * es);
    store4<T>(a.dq + ((((long)b * a.Sq + pos) * a.H + head) * D + d4 * 4) * es, o[0], o[1], o[2], o[3]);
}

// ------------------------------------------------------------------------------------------------ backward, key side
// 32 keys per wave; query rows of the key head's list in tiles of RT through LDS, with their lse and delta.  Bound as the
// others, and with 128 channels by its registers: 128 accumulators and 128 of fragments leave one wave per SIMD, which waits out
// its LDS reads itself (bf16, dense 8 x 4096 x 16 heads, four products counted of six: 550 TFLOP/s with 64 channels, 490 with 128;
// fp32, 8 x 2048 x 8: 205 and 170).  Not faster with 128 channels, when four products were all and took 600 TFLOP/s: fragments
// requested a step ahead (618, but 64 channels lose as much), tiles without padding in a swizzled order (a third fewer bank
// conflicts, same time), dk and dv in workgroups of their own (548).
template <typename T, int D, int NW, int RT, int WS>
__global__ __launch_bounds__(NW * WS * 64, NW == 4 && (sizeof(T) * D <= 128 || (sizeof(T) == 4 && D == 64)) ? 2 : 1) void dkv_kernel(Args a) {
    extern __shared__ __align__(16) char smem[];
    constexpr int TB = Elem<T>::P * RT * pitch<D>(), BUF = 2 * TB + RT * 8;
    const Place pl = place<NW * 32, true>(a);
    const Sel sel = make_sel();
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
    const int ql = pl.ql, kl = pl.kl, off = kl - ql, rv = a.G * ql;
    const int key0 = pl.tile * NW * 32, key = key0 + (WS > 1 ? 0 : w) * 32 + (lane & 31);
    const bool key_ok = key < kl;
    const long es = sizeof(T);
    const Frag<T, D> kf = load_frag<T, D>(a.k + (pl.b * a.k_sb + key * a.k_ss + pl.kh * a.k_sh) * es, key_ok, sel);
    const Frag<T, D> vf = load_frag<T, D>(a.v + (pl.b * a.v_sb + key * a.v_ss + pl.kh * a.v_sh) * es, key_ok, sel);
    const char* qb = a.q + (pl.b * a.q_sb + (long)pl.kh * a.G * a.q_sh) * es;
    const char* gb = a.doo + (pl.b * a.g_sb + (long)pl.kh * a.G * a.g_sh) * es;
    const long hrow0 = ((long)pl.b * a.H + pl.kh * a.G) * a.Sq;
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d) dk[d] = dv[d] = zero16();

    int t1 = (rv + RT - 1) / RT, t = 0;
    if (a.nsplit > 1) {                           // the pieces follow the rows that there are
        const int per = (t1 + a.nsplit - 1) / a.nsplit;
        t = pl.split * per;
        t1 = min(t1, t + per);
    }
    if (key0 >= kl) t = t1;
    // a tile's place in the list: its first row's head and position; rows behind the head's last one are the next head's
    struct At {
        int t, g, pos;
    };
    auto step = [&](At x) {
        ++x.t;
        x.pos += RT;
        while (x.pos >= ql) {
            x.pos -= ql;
            ++x.g;
        }
        return x;
    };
    // the next tile of rows with a valid pair, from x on
    auto next = [&](At x) {
        if (a.causal)
            while (x.t < t1 && min(x.pos + RT, ql) - 1 + off < key0 && x.pos + RT <= ql) x = step(x);
        return x;
    };
    constexpr float unshift = std::is_same<T, _Float16>::value ? 0x1p-15f : 1.f;
    float f = ds_scale<T>();
    typedef Stage<T, D, RT, NW * 64> St;
    St qs, gs;
    const long qss = a.q_ss * es, qsh = a.q_sh * es, gss = a.g_ss * es, gsh = a.g_sh * es;
    const unsigned qo = St::offset(qss), go = St::offset(gss);
    float st_lse = 0.f, st_dl = 0.f;
    auto request = [&](At x) {
        const int left = rv - x.t * RT;
        const bool one = x.pos + min(left, RT) <= ql;             // all of one head
        if (one) {
            qs.load(qb + x.g * qsh + x.pos * qss, qss, qo, left);
            gs.load(gb + x.g * gsh + x.pos * gss, gss, go, left);
        } else {
            qs.load_across(qb, qss, qsh, x.g, x.pos, left, ql);
            gs.load_across(gb, gss, gsh, x.g, x.pos, left, ql);
        }
        if (St::tid() < RT) {
            const int j = St::tid();
            st_lse = INFINITY;
            st_dl = 0.f;
            if (j < left) {
                const int q = one ? 0 : (x.pos + j) / ql;
                const long at = hrow0 + (long)(x.g + q) * a.Sq + (x.pos + j - q * ql);
                st_lse = a.lse[at] - p_shift<T>();
                st_dl = a.delta[at];
            }
        }
    };
    auto put = [&](char* buf) {
        qs.put(buf, sel);
        gs.put(buf + TB, sel);
        if (St::tid() < RT) {
            reinterpret_cast<float*>(buf + 2 * TB)[St::tid()] = st_lse;
            reinterpret_cast<float*>(buf + 2 * TB)[RT + St::tid()] = st_dl;
        }
    };
    At x = {t, 0, 0};
    if (t < t1) {
        x.g = t * RT / ql;
        x.pos = t * RT - x.g * ql;
        x = next(x);
    }
    auto use = [&](const At& x, const char* buf) {
        const bool across = x.pos + RT > ql;
        const bool edge = a.causal && (across ? 0 : x.pos) + off < key0 + NW * 32 - 1;
#pragma unroll
        for (int u = 0; u < RT / 32; ++u) {
            f32x16 s = mul_rows<T, D, RT>(buf, u * 32, kf, zero16());
            f32x16 dp = mul_rows<T, D, RT>(buf + TB, u * 32, vf, zero16());
            const float* st = reinterpret_cast<const float*>(buf + 2 * TB) + u * 32 + 4 * h;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const f32x4 ls = *reinterpret_cast<const f32x4*>(st + 8 * q4);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * q4 + j] = exp2_raw(fmaf(s[4 * q4 + j], a.c, -ls[j]));
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    int p = x.pos + u * 32 + acc_row(i, h);
                    if (across) p -= p / ql * ql;
                    if (p + off < key) s[i] = 0.f;
                }
            }
            mul_cols<T, D, RT>(buf + TB, u * 32, s, sel, dv);
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const f32x4 dl = *reinterpret_cast<const f32x4*>(st + RT + 8 * q4);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[4 * q4 + j] *= dp[4 * q4 + j] - dl[j];
            }
            if constexpr (std::is_same<T, _Float16>::value) {
                s *= f * unshift;                                 // s was p times 2^15
                fit_ds(s, dk, f);
            }
            mul_cols<T, D, RT>(buf, u * 32, s, sel, dk);
        }
    };
    auto unscale = [&](f32x16 (&x)[D / 32]) {
        if constexpr (std::is_same<T, _Float16>::value)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) x[d] *= 1.f / f;
    };
    if constexpr (WS > 1) {
        char* my = smem + w * BUF;
        auto jump = [&](At x, int n) {                            // n tiles with a valid pair on
            for (; n > 0 && x.t < t1; --n) x = next(step(x));
            return x;
        };
        x = jump(x, w);
        if (x.t < t1) request(x);
        while (x.t < t1) {
            put(my);
            wave_sync();
            const At xn = jump(x, WS);
            if (xn.t < t1) request(xn);
            use(x, my);
            wave_sync();
            x = xn;
        }
        unscale(dk);
        hand_over<WS>(smem, w, dk);
        if (w == 0)
#pragma unroll
            for (int i = 1; i < WS; ++i) take_over(smem, i, 1.f, dk);
        hand_over<WS>(smem, w, dv);
        if (w > 0) return;
#pragma unroll
        for (int i = 1; i < WS; ++i) take_over(smem, i, 1.f, dv);
    } else {
        if (x.t < t1) {
            request(x);
            put(smem);
        }
        __syncthreads();
        int cur = 0;
        while (x.t < t1) {
            const At xn = next(step(x));
            if (xn.t < t1) request(xn);
            use(x, smem + cur * BUF);
            if (xn.t < t1) put(smem + (cur ^ 1) * BUF);
            __syncthreads();
            cur ^= 1;
            x = xn;
        }
        unscale(dk);
    }
    if (key >= a.Sk) return;
    const long krow = ((long)pl.b * a.Sk + key) * a.Hkv + pl.kh;
    const long part0 = (long)pl.split * a.B * a.Sk * a.Hkv + krow, total = (long)a.nsplit * a.B * a.Sk * a.Hkv;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            const int ch = d * 32 + 8 * q4 + 4 * h;
            f32x4 x, y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = key_ok ? dk[d][4 * q4 + j] * a.scale : 0.f;
                y[j] = key_ok ? dv[d][4 * q4 + j] * unshift : 0.f;
            }
            if (a.nsplit > 1) {
                if (!key_ok) continue;            // the joining kernel knows
                *reinterpret_cast<f32x4*>(a.part + part0 * D + ch) = x;
                *reinterpret_cast<f32x4*>(a.part + (total + part0) * D + ch) = y;
            } else {
                store4<T>(a.dk + (krow * D + ch) * es, x[0], x[1], x[2], x[3]);
                store4<T>(a.dv + (krow * D + ch) * es, y[0], y[1], y[2], y[3]);
            }
        }
}

template <typename T, int D>
__global__ __launch_bounds__(256) void dkv_join_kernel(Args a) {
    const long n4 = (long)a.B * a.Sk * a.Hkv * (D / 4);
    const int per = 256 / a.sg, sg = (int)threadIdx.x / per;
    const long e = (long)blockIdx.x * per + threadIdx.x - sg * per;
    const long row = e / ((D / 4) * a.Hkv);                        // b * Sk + key
    const int b = (int)(row / a.Sk);
    int ql = 0, kl = 0;
    if (e < n4) lens(a, b, ql, kl);
    const bool there = e < n4 && (int)(row - (long)b * a.Sk) < kl;
    f32x4 x, y;
    const bool mine = join_sum(a, a.part, n4, there ? e : n4, sg, x);
    join_sum(a, a.part + (size_t)a.nsplit * n4 * 4, n4, there ? e : n4, sg, y);
    if (!mine || e >= n4) return;
    store4<T>(a.dk + e * 4 * sizeof(T), x[0], x[1], x[2], x[3]);
    store4<T>(a.dv + e * 4 * sizeof(T), y[0], y[1], y[2], y[3]);
}

// ------------------------------------------------------------------------------------------------ launches
struct Plan {
    int nw, tile, ntiles, nsplit, occ, piece;       // waves per workgroup, contraction rows per tile, tiles of own rows
    size_t lds;
};

// One kernel's problem: `rows` own rows in tiles of 32 per (batch, key head), `len` rows to walk; `occ` workgroups of four
// waves fit on a compute unit; `key_side`: dk and dv.
struct Problem {
    int esize, D;
    long nbh;
    int rows, len;
    bool key_side;
    int occ;
    bool causal, ragged;
    int walkers() const { return esize * D > 256 ? 2 : 4; }
};

static Plan plan_with(const Problem& x, int nw, int nsplit) {
    Plan p;
    p.piece = 0;
    p.occ = x.occ;
    p.nw = nw;
    p.nsplit = nsplit;
    p.tile = nw == 4 && x.esize == 2 ? 64 : 32;
    p.ntiles = (x.rows + 32 * nw - 1) / (32 * nw);
    const size_t buf = (size_t)2 * (x.esize == 4 ? 3 : 1) * p.tile * (x.D * 2 + 16) + (x.key_side ? p.tile * 8 : 0);
    p.lds = (nw == 4 ? 2 : x.walkers()) * buf;
    return p;
}

// What a plan takes, in us, by single launches: a four-wave workgroup alone on its compute unit takes 1.4 us per tile (16-bit
// types, heads of 64) or 2 (fp32), twice that for heads of 128, and one tile's time for its ends; more workgroups on a unit add
// `more` of that each.  A round of waves that share out a walk takes `round` tiles, their ends and their meeting `ends`.  A
// joining launch: 4 us and the pieces' results, written and read at 4 TB/s.
static double cost(const Problem& x, const Plan& p) {
    const bool half = x.esize == 2;
    const double tau = (half ? 1.4 : 2.0) * (x.D / 64);
    const double more = p.nw == 1 ? (half && x.D == 64 ? 0.6 : 1.0) : p.occ == 1 ? 1.0 : half ? 0.55 : 0.78;
    const double round = half ? 0.65 : 1.0, ends = half ? 2.2 : 3.5;
    const int per = ((x.len + p.tile - 1) / p.tile + p.nsplit - 1) / p.nsplit;
    const double load = (double)(x.nbh * p.ntiles * p.nsplit) / compute_units();
    const double turns = more * (x.causal || x.ragged ? 0.6 * load + 0.4 : std::ceil(load));     // uneven ones fill each other's gaps
    const double one = p.nw == 4 ? per + 1 : (per + x.walkers() - 1) / x.walkers() * round + ends;
    const double bytes = 8.0 * p.nsplit * x.nbh * x.rows * x.D * (x.key_side ? 2 : 1);
    return tau * one * (turns > 1.0 ? turns : 1.0) + (p.nsplit > 1 ? 4.0 + bytes / 4e6 : 0.0);
}

// Four tiles of own rows per workgroup share what they walk; or one tile per workgroup, whose waves share out the walk.  The
// walk may be cut into pieces, which a second launch joins.
//   Where four tiles per workgroup fill the card: those, with pieces until there is a workgroup for every slot — twice that for
// the causal order at one workgroup per unit (two are dealt in pairs, see place()), half again as much where lengths will leave
// some without work — or, without lengths, whole, if that costs less (20 x 500 rows x 4 heads of 64 bf16, forward: 23 us whole, 31 in
// two; 8 x 512 against 2048 rows x 8 heads: 59, 51).
//   Else whatever costs least of both kinds, whole or in as many pieces as one, two or three turns of the card hold.  Forward +
//   backward in us, four tiles against one: fp32 4 x 200 rows x 4 heads of 64 67 / 43, 16 x 300 106 / 146, 400 against 8000
//   141 / 270, causal 4096 x 2 heads of 128 416 / 1261; bf16 35 / 25, 44 / 59, 74 / 78, 160 / 213.
static Plan make_plan(const Problem& x) {
    const long cus = compute_units();
    Plan best = plan_with(x, 4, 1);
    const long wg4 = x.nbh * best.ntiles;
    if (wg4 >= cus) {
        const int tiles = (x.len + best.tile - 1) / best.tile;
        const long slots = cus * x.occ, want = x.causal && x.occ == 1 ? 2 * slots : x.ragged ? slots + slots / 2 : slots;
        if (wg4 < want && tiles >= 8) {
            const Plan p = plan_with(x, 4, (int)std::min((want + wg4 - 1) / wg4, tiles / 4L));
            if (x.ragged || cost(x, p) < cost(x, best)) best = p;
        }
        return best;
    }
    if (wg4 == 0) return best;
    double least = cost(x, best);
    for (const int nw : {4, 1}) {
        Plan p = plan_with(x, nw, 1);
        const long wg = x.nbh * p.ntiles, tiles = (x.len + p.tile - 1) / p.tile;
        const long most = std::min(64L, nw == 4 ? tiles / 2 : tiles / (2 * x.walkers()));
        for (int turn = 0; turn <= 3; ++turn) {
            const long ns = turn == 0 ? 1 : std::min(most, turn * cus / wg);
            if (turn > 0 && ns <= p.nsplit) continue;
            p.nsplit = (int)ns;
            const double c = cost(x, p);
            if (c < least) {
                least = c;
                best = p;
            }
        }
    }
    return best;
}

// Rows per key head up to which fwd_rows_kernel takes a list: its arithmetic grows with the rows, the matrix instructions' does
// not.  Rows kernel / the other, us, for 16 lists of 8191 keys x 8 heads: bf16 heads of 128, 1 row 99 / 102, 2 102 / 104, 4 110 /
// 101, 8 167 / 105; fp16 heads of 64 50 / 51, 51 / 50, 55 / 50, 102 / 51; fp32 heads of 64, 4 rows 108 / 107 and for 16 of 2000
// 30 / 34 (6 rows 58 / 35); fp32 heads of 128, 1 row 193 / 332, 8 262 / 330; one list of 8192 keys x 8 heads of 128, 1 row, bf16 10 / 14.
constexpr int most_rows(int esize, int D) { return esize == 2 ? 2 : D == 64 ? 4 : 8; }

// Few rows: four waves per workgroup, at least two rounds of 16-byte loads each per piece, eight workgroups per unit (of padded
// lists some have no keys: 16 of up to 8191 keys x 8 heads of 128, 4 rows, 4 per unit 82 us, 8 76, 16 79).
static Plan rows_plan(int esize, int D, long nbh, int len) {
    Plan p = {4, 0, 1, 1, 4, 0, 0};
    const int round = 4 * 4 * (64 / (D * esize / 16));           // keys per round of a workgroup
    const long want = 8L * compute_units();
    long ns = (want + nbh - 1) / nbh;
    const long most = (len + 2 * round - 1) / (2 * round);
    if (ns > most) ns = most;
    if (ns < 1) ns = 1;
    if (ns > 64) ns = 64;
    p.piece = (int)((((len + ns - 1) / ns) + round - 1) / round * round);
    p.nsplit = len > 0 ? (len + p.piece - 1) / p.piece : 1;
    return p;
}

static size_t esize_of(int dtype) { return dtype == CMVAE_F32 ? 4 : 2; }

struct Sizes {
    Plan f, q, k;
    size_t fwd, bwd;
};
static Sizes sizes_of(const cmvae_set_attn& d) {
    Sizes z;
    const int es = (int)esize_of(d.dtype), G = d.H / d.Hkv;
    const long nbh = (long)d.B * d.Hkv;
    const int R = G * d.Sq;
    const bool causal = d.causal != 0, ragged = d.q_len || d.k_len;
    const Problem qside = {es, d.D, nbh, R, d.Sk, false, es * d.D > 256 ? 1 : 2, causal, ragged};
    z.f = R <= most_rows(es, d.D) ? rows_plan(es, d.D, nbh, d.Sk) : make_plan(qside);
    z.q = make_plan(qside);
    z.k = make_plan({es, d.D, nbh, d.Sk, R, true, d.D == 64 ? 2 : 1, causal, ragged});
    const size_t rows = (size_t)nbh * R, keys = (size_t)nbh * d.Sk;
    z.fwd = z.f.nsplit > 1 ? z.f.nsplit * rows * (d.D + 2) * 4 : 0;
    const size_t bq = z.q.nsplit > 1 ? z.q.nsplit * rows * d.D * 4 : 0;
    const size_t bk = z.k.nsplit > 1 ? (size_t)z.k.nsplit * 2 * keys * d.D * 4 : 0;
    z.bwd = bq > bk ? bq : bk;                    // the key side's launches follow the query side's on the same stream
    return z;
}

static void use(Args& a, const Plan& p) {
    a.ntiles = p.ntiles;
    a.nsplit = p.nsplit;
    a.piece = p.piece;
    a.fold = p.occ >= 2 ? compute_units() : 1 << 29;
}

// groups that share out the splits of one value in a joining kernel of n4 x 4 values: until the launch fills the card
static int join_groups(int nsplit, long n4, int most) {
    int sg = 1;
    while (sg < most && 2 * sg <= nsplit && n4 * sg < 256L * 1024) sg *= 2;
    return sg;
}

template <typename T, int D>
static int run_fwd(Args a, const Sizes& z, float* ws, void* stream) {
    constexpr int T4 = sizeof(T) == 2 ? 64 : 32, WS = walkers<T, D>();
    const long nbh = (long)a.B * a.Hkv, rows = nbh * a.R;
    use(a, z.f);
    a.part = ws;
    a.part_ml = ws + (size_t)a.nsplit * rows * D;
    const long blocks = nbh * a.ntiles * a.nsplit;
    constexpr int MOST = most_rows(sizeof(T), D);
    auto rows_of = [&](auto r) { return launch_kernel<fwd_rows_kernel<T, D, r>>(blocks, 256, 0, a, stream, "set_attention fwd_rows_kernel"); };
    int e;
    if (a.R <= MOST) {
        if (a.R == 1) e = rows_of(std::integral_constant<int, 1>());
        else if (a.R == 2) e = rows_of(std::integral_constant<int, 2>());
        else if (a.R <= 4) e = rows_of(std::integral_constant<int, std::min(4, MOST)>());
        else e = rows_of(std::integral_constant<int, MOST>());
    } else {
        e = z.f.nw == 4 ? launch_kernel<fwd_kernel<T, D, 4, T4, 1>>(blocks, 256, z.f.lds, a, stream, "set_attention fwd_kernel")
                        : launch_kernel<fwd_kernel<T, D, 1, 32, WS>>(blocks, WS * 64, z.f.lds, a, stream, "set_attention fwd_kernel");
    }
    if (e || a.nsplit == 1) return e;
    a.sg = join_groups(a.nsplit, rows * (D / 4), 256 / (D / 4));
    return launch_kernel<fwd_join_kernel<T, D>>((rows * (D / 4) * a.sg + 255) / 256, 256, 0, a, stream, "set_attention fwd_join_kernel");
}

template <typename T, int D>
static int run_bwd(Args a, const Sizes& z, float* ws, void* stream) {
    constexpr int T4 = sizeof(T) == 2 ? 64 : 32, WS = walkers<T, D>();
    const long nbh = (long)a.B * a.Hkv, rows = nbh * a.R, keys = nbh * a.Sk;
    a.part = ws;
    use(a, z.q);
    long blocks = nbh * a.ntiles * a.nsplit;
    int e = z.q.nw == 4 ? launch_kernel<dq_kernel<T, D, 4, T4, 1>>(blocks, 256, z.q.lds, a, stream, "set_attention dq_kernel")
                        : launch_kernel<dq_kernel<T, D, 1, 32, WS>>(blocks, WS * 64, z.q.lds, a, stream, "set_attention dq_kernel");
    if (e) return e;
    if (a.nsplit > 1) {
        a.sg = join_groups(a.nsplit, rows * (D / 4), 16);
        if ((e = launch_kernel<dq_join_kernel<T, D>>((rows * (D / 4) * a.sg + 255) / 256, 256, 0, a, stream, "set_attention dq_join_kernel")))
            return e;
    }
    use(a, z.k);
    blocks = nbh * a.ntiles * a.nsplit;
    e = z.k.nw == 4 ? launch_kernel<dkv_kernel<T, D, 4, T4, 1>>(blocks, 256, z.k.lds, a, stream, "set_attention dkv_kernel")
                    : launch_kernel<dkv_kernel<T, D, 1, 32, WS>>(blocks, WS * 64, z.k.lds, a, stream, "set_attention dkv_kernel");
    if (e || a.nsplit == 1) return e;
    const long n4 = keys * D / 4;
    a.sg = join_groups(a.nsplit, n4, 16);
    return launch_kernel<dkv_join_kernel<T, D>>((n4 * a.sg + 255) / 256, 256, 0, a, stream, "set_attention dkv_join_kernel");
}

static bool aligned(const void* p, const int64_t* s, int dtype) {
    const int m = 16 / (int)esize_of(dtype);
    for (int i = 0; i < 3; ++i)
        if (s[i] % m || s[i] < 0) return false;
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s[1] < (1 << 22);       // a tile's 64 rows: 31-bit offsets
}

static int check_desc(const char* who, const cmvae_set_attn* d) {
    CMVAE_REQUIRE(d != nullptr, "%s: NULL descriptor", who);
    CMVAE_REQUIRE(d->dtype == CMVAE_F32 || d->dtype == CMVAE_BF16 || d->dtype == CMVAE_F16, "%s: dtype %d", who, d->dtype);
    CMVAE_REQUIRE(d->D == 64 || d->D == 128, "%s: heads of %d channels (64 or 128 are supported)", who, d->D);
    CMVAE_REQUIRE(d->B >= 1 && d->Sq >= 1 && d->Sk >= 0 && d->H >= 1 && d->Hkv >= 1 && d->H % d->Hkv == 0,
                  "%s: B=%d Sq=%d Sk=%d heads=%d key heads=%d", who, d->B, d->Sq, d->Sk, d->H, d->Hkv);
    CMVAE_REQUIRE((long)d->H / d->Hkv * d->Sq < (1L << 30) && d->Sk < (1 << 30), "%s: more than 2^30 rows per key head", who);
    CMVAE_REQUIRE(d->scale >= 1e-30f && d->scale <= 1e30f, "%s: scale %g (a positive finite number)", who, (double)d->scale);
    const Sizes z = sizes_of(*d);
    const long nbh = (long)d->B * d->Hkv;
    CMVAE_REQUIRE(nbh * z.f.ntiles * z.f.nsplit < (1L << 31) && nbh * z.q.ntiles * z.q.nsplit < (1L << 31) && nbh * z.k.ntiles * z.k.nsplit < (1L << 31) &&
                      nbh * (d->H / d->Hkv) * d->Sq * (d->D / 4) / 256 < (1L << 31) - 1 &&
                      nbh * d->Sk * (d->D / 4) / 256 < (1L << 31) - 1,
                  "%s: the problem needs more than 2^31 workgroups", who);
    return 0;
}

static Args args_of(const cmvae_set_attn& d) {
    Args a = {};
    a.q = (const char*)d.q; a.k = (const char*)d.k; a.v = (const char*)d.v;
    a.doo = (const char*)d.dO;
    a.o = (char*)d.o; a.ocopy = (char*)d.attn; a.olow = (char*)d.attn_low;
    a.att_low = (const char*)d.attn_low;
    a.att = (const char*)(d.residual ? d.attn : d.o);
    a.dq = (char*)d.dq; a.dk = (char*)d.dk; a.dv = (char*)d.dv;
    a.lse = d.lse; a.delta = d.delta;
    a.q_len = d.q_len; a.k_len = d.k_len;
    a.q_sb = d.q_stride[0]; a.q_ss = d.q_stride[1]; a.q_sh = d.q_stride[2];
    a.k_sb = d.k_stride[0]; a.k_ss = d.k_stride[1]; a.k_sh = d.k_stride[2];
    a.v_sb = d.v_stride[0]; a.v_ss = d.v_stride[1]; a.v_sh = d.v_stride[2];
    a.g_sb = d.dO_stride[0]; a.g_ss = d.dO_stride[1]; a.g_sh = d.dO_stride[2];
    a.B = d.B; a.Sq = d.Sq; a.Sk = d.Sk; a.H = d.H; a.Hkv = d.Hkv;
    a.G = d.H / d.Hkv;
    a.R = a.G * d.Sq;
    a.causal = d.causal != 0;
    a.residual = d.residual != 0;
    a.scale = d.scale;
    a.c = d.scale * LOG2E;
    return a;
}

}  // namespace sa
}  // namespace cmvae

using namespace cmvae;

#define SA_DISPATCH(fn)                                                                        \
    switch (d->dtype * 1000 + d->D) {                                                          \
        case CMVAE_F32 * 1000 + 64: return sa::fn<float, 64>(a, z, (float*)workspace, stream);  \
        case CMVAE_F32 * 1000 + 128: return sa::fn<float, 128>(a, z, (float*)workspace, stream); \
        case CMVAE_BF16 * 1000 + 64: return sa::fn<__bf16, 64>(a, z, (float*)workspace, stream); \
        case CMVAE_BF16 * 1000 + 128: return sa::fn<__bf16, 128>(a, z, (float*)workspace, stream); \
        case CMVAE_F16 * 1000 + 64: return sa::fn<_Float16, 64>(a, z, (float*)workspace, stream); \
        default: return sa::fn<_Float16, 128>(a, z, (float*)workspace, stream);                 \
    }

extern "C" size_t cmvae_set_attention_workspace_bytes(const cmvae_set_attn* d, int backward) {
    cmvae::clear_stale_error();
    if (sa::check_desc("cmvae_set_attention_workspace_bytes", d)) return 0;
    const sa::Sizes z = sa::sizes_of(*d);
    return backward ? z.bwd : z.fwd;
}

extern "C" int cmvae_set_attention_fwd(const cmvae_set_attn* d, void* workspace, size_t workspace_bytes, void* stream) {
    cmvae::clear_stale_error();
    if (int e = sa::check_desc("cmvae_set_attention_fwd", d)) return e;
    CMVAE_REQUIRE(d->q && d->o && (d->Sk == 0 || (d->k && d->v)), "cmvae_set_attention_fwd: NULL tensor");
    CMVAE_REQUIRE(sa::aligned(d->q, d->q_stride, d->dtype) && sa::aligned(d->k, d->k_stride, d->dtype) &&
                      sa::aligned(d->v, d->v_stride, d->dtype) && (((uintptr_t)d->o | (uintptr_t)d->attn | (uintptr_t)d->attn_low) & 15) == 0,
                  "cmvae_set_attention_fwd: rows must start at multiples of 16 bytes and lie under 2^22 elements apart");
    const sa::Sizes z = sa::sizes_of(*d);
    CMVAE_REQUIRE(z.fwd == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= z.fwd),
                  "cmvae_set_attention_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, z.fwd);
    sa::Args a = sa::args_of(*d);
    SA_DISPATCH(run_fwd)
}

extern "C" int cmvae_set_attention_bwd(const cmvae_set_attn* d, void* workspace, size_t workspace_bytes, void* stream) {
    cmvae::clear_stale_error();
    if (int e = sa::check_desc("cmvae_set_attention_bwd", d)) return e;
    CMVAE_REQUIRE(d->q && d->dO && d->lse && d->delta && d->dq && (d->residual ? (const void*)d->attn : d->o) &&
                      (d->Sk == 0 || (d->k && d->v && d->dk && d->dv)),
                  "cmvae_set_attention_bwd: NULL tensor");
    CMVAE_REQUIRE(sa::aligned(d->q, d->q_stride, d->dtype) && sa::aligned(d->k, d->k_stride, d->dtype) &&
                      sa::aligned(d->v, d->v_stride, d->dtype) && sa::aligned(d->dO, d->dO_stride, d->dtype) &&
                      (((uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv | (uintptr_t)d->o | (uintptr_t)d->attn | (uintptr_t)d->attn_low) & 15) == 0,
                  "cmvae_set_attention_bwd: rows must start at multiples of 16 bytes and lie under 2^22 elements apart");
    const sa::Sizes z = sa::sizes_of(*d);
    CMVAE_REQUIRE(z.bwd == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= z.bwd),
                  "cmvae_set_attention_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, z.bwd);
    sa::Args a = sa::args_of(*d);
    SA_DISPATCH(run_bwd)
}
