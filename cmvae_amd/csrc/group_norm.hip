// Group norm with an activation on channels-last rows, and its backward pass: cmvae_group_norm_{fwd,bwd}.
//
//   per sample n and group g of C / G channels: mean and biased variance over the sample's P pixels x C / G channels,
//   xhat = (x - mean) rstd,  z = xhat w_c + b_c,  y = act(z)
//   dz = dy act'(z),  db_c = sum dz,  dw_c = sum dz xhat,
//   dx = rstd (dz w_c - m1 - xhat m2),   m1, m2 = means over the group of dz w_c and dz w_c xhat
//
// Both directions are bound by memory.  A sample whose rows fit in the registers of one workgroup is read once and written
// once (resident kernels; 800 x 196 x 64 fp32: 23 us forward, 31 backward, 3.5 and 3.9 TB/s; in 16 bits 19 and 25 for half
// the bytes, so what a value takes besides them shows); a larger one takes a pass for its sums, a small launch that finishes
// them, and a pass that applies them (16 x 9216 x 320 bf16: 60 us forward, 108 backward, 4.7 and 4.4 TB/s over what the passes
// move).  A thread's sums are per channel, so a group may end anywhere in its vector.
//
// The forward's sums are of d and d^2 in fp64, d = x - (the group's first value): no second pass, and what the variance loses to
// the mean is 2^-53 of the square of a difference, not of a value.  (Sums of x and x^2 leave 2^-52 x^2 where a group holds
// one value: at x = 10^5 more than eps, and rstd a third of what it is.  The difference costs the resident forward 4 %.)  The
// mean is kept as two fp32 numbers for the same reason.  The backward's sums are of mixed sign and fp32 in a thread, fp64 where
// threads meet.
// Sums are added in a fixed order: every run gives the same bits.
#include "common.h"

#include <cmath>
#include <type_traits>

namespace cmvae {
namespace gn {

struct Args {
    const void *x, *dy, *w, *b;
    void *y, *dx, *dw, *db;
    float4* stats;                              // [N, G]: mean (two parts), rstd
    double2* part;                              // forward sums [N, pc, C]
    float2* bpart;                              // backward sums [N, pc, C]
    float2* means;                              // m1, m2 [N, G]
    long x_sn, x_sp, g_sn, g_sp;                // strides in elements
    int N, P, C, G, Cg, CV, act, wtype, xtype;
    int pc, rows_per, cc, cw;                   // pixel pieces per sample, pixels per piece, channel pieces, vectors per one
    float eps;
};

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ void unpack(const typename Vec<T, V>::type& p, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = (float)p;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (float)p[j];
    }
}
template <typename T, int V>
__device__ __forceinline__ typename Vec<T, V>::type pack(const float (&x)[V]) {
    typename Vec<T, V>::type p;
    if constexpr (V == 1) {
        p = (T)x[0];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = (T)x[j];
    }
    return p;
}

__device__ __forceinline__ float value(const void* p, int type, long c) {
    if (type == CMVAE_F32) return ((const float*)p)[c];
    if (type == CMVAE_BF16) return (float)((const __bf16*)p)[c];
    return (float)((const _Float16*)p)[c];
}
__device__ __forceinline__ float param(const void* p, int type, int c, float none) { return p ? value(p, type, c) : none; }
__device__ __forceinline__ void put_param(void* p, int type, int c, double v) {
    if (!p) return;
    if (type == CMVAE_F32) ((float*)p)[c] = (float)v;
    else if (type == CMVAE_BF16) ((__bf16*)p)[c] = (__bf16)(float)v;
    else ((_Float16*)p)[c] = (_Float16)(float)v;
}

// 1 / (1 + e^-z); the reciprocal to 1 ulp (a division is ten instructions of the backward's forty per value)
__device__ __forceinline__ float sigmoid1(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

// z -> act(z) of a thread's vector: one branch per vector
template <int V>
__device__ __forceinline__ void activate(float (&z)[V], int act) {
    if (act == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = z[j] > 0.f ? z[j] : (z[j] != z[j] ? z[j] : 0.f);
    } else if (act == 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] = elu1(z[j]);
    } else if (act == 3) {
#pragma unroll
        for (int j = 0; j < V; ++j) z[j] *= sigmoid1(z[j]);
    }
}
// d -> d act'(z)
template <int V>
__device__ __forceinline__ void slope(const float (&z)[V], float (&d)[V], int act) {
    if (act == 1) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = z[j] > 0.f ? d[j] : 0.f;
    } else if (act == 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = z[j] > 0.f ? d[j] : d[j] * __expf(z[j]);
    } else if (act == 3) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float s = sigmoid1(z[j]);
            d[j] *= s * fmaf(z[j], 1.f - s, 1.f);
        }
    }
}

// from the sums of d = x - first and d^2 over m values
__device__ __forceinline__ float4 make_stats(double s1, double s2, float first, double m, float eps) {
    const double off = s1 / m, var = fmax(s2 / m - off * off, 0.0), mean = (double)first + off;
    const float hi = (float)mean;
    return make_float4(hi, (float)(mean - (double)hi), (float)(1.0 / sqrt(var + (double)eps)), 0.f);
}

// a thread's V channels: what normalises them
template <int V>
struct Channel {
    float mh[V], ml[V], rs[V], w[V], b[V];
};
template <int V>
__device__ __forceinline__ void load_params(const Args& a, int c0, Channel<V>& k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        k.w[j] = param(a.w, a.wtype, c0 + j, 1.f);
        k.b[j] = param(a.b, a.wtype, c0 + j, 0.f);
    }
}
template <int V>
__device__ __forceinline__ void load_stats(const Args& a, const float4* st, int c0, Channel<V>& k) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float4 s = st[(c0 + j) / a.Cg];
        k.mh[j] = s.x; k.ml[j] = s.y; k.rs[j] = s.z;
    }
}

// the first value of each of a thread's channels' groups; x: the sample
template <typename T, int V>
__device__ __forceinline__ void load_first(const Args& a, const T* x, int c0, double (&first)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) first[j] = (double)(float)x[(c0 + j) / a.Cg * a.Cg];
}
template <int V>
__device__ __forceinline__ void add_to(const float (&v)[V], const double (&first)[V], double (&s1)[V], double (&s2)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const double d = (double)v[j] - first[j];
        s1[j] += d;
        s2[j] = fma(d, d, s2[j]);
    }
}

// x -> xhat, d = dy -> dz
template <int V>
__device__ __forceinline__ void backward_of(const Channel<V>& k, int act, float (&x)[V], float (&d)[V]) {
    float z[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        x[j] = (x[j] - k.mh[j] - k.ml[j]) * k.rs[j];
        z[j] = fmaf(x[j], k.w[j], k.b[j]);
    }
    slope<V>(z, d, act);
}
template <int V>
__device__ __forceinline__ void forward_of(const Channel<V>& k, int act, float (&x)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = fmaf((x[j] - k.mh[j] - k.ml[j]) * k.rs[j], k.w[j], k.b[j]);
    activate<V>(x, act);
}

// ------------------------------------------------------------------------------------------------ sums where threads meet
__device__ __forceinline__ double2 add2(double2 a, double2 b) { return make_double2(a.x + b.x, a.y + b.y); }
__device__ __forceinline__ double2 wide(double2 a) { return a; }
__device__ __forceinline__ double2 wide(float2 a) { return make_double2((double)a.x, (double)a.y); }
__device__ __forceinline__ void narrow(double2 a, double2& b) { b = a; }
__device__ __forceinline__ void narrow(double2 a, float2& b) { b = make_float2((float)a.x, (float)a.y); }

// column sums of red[rows][cols] into put(c, sum); called by all THREADS threads.  Where there are fewer columns than threads,
// a column's rows are first shared out over `parts` threads, each of which leaves its sum in the first of its rows (one thread
// per column took 29.9 us of the forward for 800 samples of 196 x 64 bf16 values: 64 rows one after the other).
template <int THREADS, typename S, typename Put>
__device__ __forceinline__ void column_sums(S* red, int rows, int cols, Put&& put) {
    const int t = threadIdx.x;
    int parts = min(THREADS / cols, rows);
    if (parts > 1) {
        const int j = t / cols, c = t - j * cols;
        if (j < parts) {
            double2 s = wide(red[j * cols + c]);
            for (int r = j + parts; r < rows; r += parts) s = add2(s, wide(red[r * cols + c]));
            narrow(s, red[j * cols + c]);
        }
        __syncthreads();
    } else {
        parts = rows;
    }
    for (int c = t; c < cols; c += THREADS) {
        double2 s = wide(red[c]);
        for (int r = 1; r < parts; ++r) s = add2(s, wide(red[r * cols + c]));
        put(c, s);
    }
}

// put(g, sum over i < items of get(g, i)) for each group, by as many lanes per group as there are
template <int THREADS, typename Get, typename Put>
__device__ __forceinline__ void group_sums(int G, int items, Get&& get, Put&& put) {
    int L = 64;
    while (L > 1 && L * G > THREADS) L >>= 1;
    const int l = (int)threadIdx.x % L;
    for (int g = (int)threadIdx.x / L; g < G; g += THREADS / L) {
        double2 s = make_double2(0.0, 0.0);
        for (int i = l; i < items; i += L) s = add2(s, get(g, i));
        for (int o = L >> 1; o > 0; o >>= 1) s = add2(s, make_double2(__shfl_xor(s.x, o), __shfl_xor(s.y, o)));
        if (l == 0) put(g, s);
    }
}

// ------------------------------------------------------------------------------------------------ resident
// One workgroup per sample; thread t holds vectors t, t + A, t + 2A ... of the sample's P * CV, A = the largest multiple
// of CV up to the workgroup: its channels are the same in all of them.
template <typename T, int V, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void fwd_resident_kernel(Args a) {
    extern __shared__ __align__(16) char smem[];
    const bool one = a.Cg % V == 0;                                        // a thread's channels are of one group
    double2* red = reinterpret_cast<double2*>(smem);                       // [rows][CV or C]
    float4* st = reinterpret_cast<float4*>(smem + (size_t)THREADS * (one ? 1 : V) * sizeof(double2));
    typedef typename Vec<T, V>::type TV;
    const int n = blockIdx.x, t = threadIdx.x;
    const int rows = THREADS / a.CV, A = rows * a.CV;
    const int row = t / a.CV, c0 = (t - row * a.CV) * V;
    const bool on = t < A;
    const T* x = (const T*)a.x + n * a.x_sn + c0;
    TV hold[R];
    double first[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0;
    if (on) load_first<T, V>(a, x - c0, c0, first);
    for (int g = t; g < a.G; g += THREADS) st[g].x = (float)(x - c0)[g * a.Cg];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int p = row + i * rows;
        if (on && p < a.P) hold[i] = *reinterpret_cast<const TV*>(x + p * a.x_sp);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (on && row + i * rows < a.P) {
            float v[V];
            unpack<T, V>(hold[i], v);
            add_to<V>(v, first, s1, s2);
        }
    }
    if (one) {
#pragma unroll
        for (int j = 1; j < V; ++j) {
            s1[0] += s1[j];
            s2[0] += s2[j];
        }
        if (on) red[t] = make_double2(s1[0], s2[0]);
    } else if (on) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[t * V + j] = make_double2(s1[j], s2[j]);
    }
    __syncthreads();
    const int w = one ? a.Cg / V : a.Cg, pitch = one ? a.CV : a.C;
    group_sums<THREADS>(a.G, rows * w, [&](int g, int i) {
        const int r = i / w;
        return red[r * pitch + g * w + i - r * w];
    }, [&](int g, double2 u) {
        const float4 q = make_stats(u.x, u.y, st[g].x, (double)a.P * a.Cg, a.eps);
        st[g] = q;
        if (a.stats) a.stats[(long)n * a.G + g] = q;
    });
    __syncthreads();
    if (!on) return;
    Channel<V> k;
    load_params<V>(a, c0, k);
    load_stats<V>(a, st, c0, k);
    T* y = (T*)a.y + (long)n * a.P * a.C + c0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int p = row + i * rows;
        if (p < a.P) {
            float v[V];
            unpack<T, V>(hold[i], v);
            forward_of<V>(k, a.act, v);
            *reinterpret_cast<TV*>(y + (long)p * a.C) = pack<T, V>(v);
        }
    }
}

template <typename T, int V, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void bwd_resident_kernel(Args a) {
    extern __shared__ __align__(16) char smem[];
    float2* red = reinterpret_cast<float2*>(smem);
    float4* st = reinterpret_cast<float4*>(smem + (size_t)THREADS * V * sizeof(float2));
    float2* mm = reinterpret_cast<float2*>(st + a.G);
    typedef typename Vec<T, V>::type TV;
    const int n = blockIdx.x, t = threadIdx.x;
    const int rows = THREADS / a.CV, A = rows * a.CV;
    const int row = t / a.CV, c0 = (t - row * a.CV) * V;
    const bool on = t < A;
    const T* x = (const T*)a.x + n * a.x_sn + c0;
    const T* dy = (const T*)a.dy + n * a.g_sn + c0;
    TV hx[R], hg[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int p = row + i * rows;
        if (on && p < a.P) {
            hx[i] = *reinterpret_cast<const TV*>(x + p * a.x_sp);
            hg[i] = *reinterpret_cast<const TV*>(dy + p * a.g_sp);
        }
    }
    for (int g = t; g < a.G; g += THREADS) st[g] = a.stats[(long)n * a.G + g];
    Channel<V> k;
    if (on) load_params<V>(a, c0, k);
    __syncthreads();
    if (on) load_stats<V>(a, st, c0, k);
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (on && row + i * rows < a.P) {
            float v[V], d[V];
            unpack<T, V>(hx[i], v);
            unpack<T, V>(hg[i], d);
            backward_of<V>(k, a.act, v, d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1[j] += d[j];
                s2[j] = fmaf(d[j], v[j], s2[j]);
            }
        }
    }
    if (on)
#pragma unroll
        for (int j = 0; j < V; ++j) red[row * a.C + c0 + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    column_sums<THREADS>(red, rows, a.C, [&](int c, double2 u) {
        const float2 q = make_float2((float)u.x, (float)u.y);
        red[c] = q;
        a.bpart[(long)n * a.C + c] = q;
    });
    __syncthreads();
    group_sums<THREADS>(a.G, a.Cg, [&](int g, int i) {
        const int c = g * a.Cg + i;
        const double wt = (double)param(a.w, a.wtype, c, 1.f);
        return make_double2(wt * (double)red[c].x, wt * (double)red[c].y);
    }, [&](int g, double2 u) {
        const double m = (double)a.P * a.Cg;
        mm[g] = make_float2((float)(u.x / m), (float)(u.y / m));
    });
    __syncthreads();
    if (!on) return;
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 q = mm[(c0 + j) / a.Cg];
        m1[j] = q.x;
        m2[j] = q.y;
    }
    T* dx = (T*)a.dx + (long)n * a.P * a.C + c0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int p = row + i * rows;
        if (p < a.P) {
            float v[V], d[V];
            unpack<T, V>(hx[i], v);
            unpack<T, V>(hg[i], d);
            backward_of<V>(k, a.act, v, d);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = k.rs[j] * (fmaf(d[j], k.w[j], -m1[j]) - v[j] * m2[j]);
            *reinterpret_cast<TV*>(dx + (long)p * a.C) = pack<T, V>(v);
        }
    }
}

// ------------------------------------------------------------------------------------------------ in pieces
struct Piece {
    int n, pc, c0, row, rows, cw, p0, p1;
    bool on;
};
template <int V>
__device__ __forceinline__ Piece piece(const Args& a) {
    Piece q;
    int id = blockIdx.x;
    const int cc = id % a.cc;
    id /= a.cc;
    q.pc = id % a.pc;
    q.n = id / a.pc;
    q.cw = min(a.CV - cc * a.cw, a.cw);                           // vectors of channels in this piece
    q.rows = 256 / q.cw;
    q.row = (int)threadIdx.x / q.cw;
    q.on = q.row < q.rows;
    q.c0 = (cc * a.cw + (int)threadIdx.x - q.row * q.cw) * V;
    q.p0 = q.pc * a.rows_per;
    q.p1 = min(a.P, q.p0 + a.rows_per);
    return q;
}

template <typename T, int V>
__global__ __launch_bounds__(256) void fwd_sums_kernel(Args a) {
    __shared__ double2 red[256 * V];
    typedef typename Vec<T, V>::type TV;
    const Piece q = piece<V>(a);
    double s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0;
    const T* x = (const T*)a.x + q.n * a.x_sn + q.c0;
    if (q.on) {
        double first[V];
        load_first<T, V>(a, x - q.c0, q.c0, first);
#pragma unroll 4
        for (int p = q.p0 + q.row; p < q.p1; p += q.rows) {
            float v[V];
            unpack<T, V>(*reinterpret_cast<const TV*>(x + p * a.x_sp), v);
            add_to<V>(v, first, s1, s2);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) red[threadIdx.x * V + j] = make_double2(s1[j], s2[j]);
    __syncthreads();
    const int c0 = q.c0 - ((int)threadIdx.x - q.row * q.cw) * V;
    column_sums<256>(red, q.rows, q.cw * V, [&](int c, double2 u) { a.part[((long)q.n * a.pc + q.pc) * a.C + c0 + c] = u; });
}

// Sum over `rows` rows, `pitch` apart, of `width` neighbours of part (each times weight(i), i < width), in thread 0 of a
// workgroup of FIN threads: lanes beside each other take neighbours, four loads in flight each.
template <int FIN, typename S, typename W>
__device__ __forceinline__ double2 block_sum(const S* part, int rows, long pitch, int width, W&& weight) {
    __shared__ double2 red[FIN / 64];
    double2 s = make_double2(0.0, 0.0);
    const int across = min(width, FIN), step = FIN / across, r0 = (int)threadIdx.x / across;
    if (r0 < step)
        for (int c = (int)threadIdx.x - r0 * across; c < width; c += across) {
            double2 u = make_double2(0.0, 0.0);
#pragma unroll 4
            for (int r = r0; r < rows; r += step) u = add2(u, wide(part[r * pitch + c]));
            const double w = weight(c);
            s = add2(s, make_double2(w * u.x, w * u.y));
        }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = add2(s, make_double2(__shfl_xor(s.x, o), __shfl_xor(s.y, o)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < FIN / 64; ++i) s = add2(s, red[i]);
    return s;
}

// one workgroup per (sample, group)
template <int FIN>
__global__ __launch_bounds__(FIN) void fwd_finish_kernel(Args a) {
    const long ng = blockIdx.x;
    const int n = (int)(ng / a.G), g = (int)(ng - (long)n * a.G);
    const float first = value(a.x, a.xtype, n * a.x_sn + g * a.Cg);
    const double2 s = block_sum<FIN>(a.part + (long)n * a.pc * a.C + g * a.Cg, a.pc, a.C, a.Cg, [](int) { return 1.0; });
    if (threadIdx.x == 0) a.stats[ng] = make_stats(s.x, s.y, first, (double)a.P * a.Cg, a.eps);
}

template <typename T, int V>
__global__ __launch_bounds__(256) void fwd_apply_kernel(Args a) {
    typedef typename Vec<T, V>::type TV;
    const Piece q = piece<V>(a);
    if (!q.on) return;
    Channel<V> k;
    load_params<V>(a, q.c0, k);
    load_stats<V>(a, a.stats + (long)q.n * a.G, q.c0, k);
    const T* x = (const T*)a.x + q.n * a.x_sn + q.c0;
    T* y = (T*)a.y + (long)q.n * a.P * a.C + q.c0;
#pragma unroll 4
    for (int p = q.p0 + q.row; p < q.p1; p += q.rows) {
        float v[V];
        unpack<T, V>(*reinterpret_cast<const TV*>(x + p * a.x_sp), v);
        forward_of<V>(k, a.act, v);
        *reinterpret_cast<TV*>(y + (long)p * a.C) = pack<T, V>(v);
    }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void bwd_sums_kernel(Args a) {
    __shared__ float2 red[256 * V];
    typedef typename Vec<T, V>::type TV;
    const Piece q = piece<V>(a);
    float s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
    if (q.on) {
        Channel<V> k;
        load_params<V>(a, q.c0, k);
        load_stats<V>(a, a.stats + (long)q.n * a.G, q.c0, k);
        const T* x = (const T*)a.x + q.n * a.x_sn + q.c0;
        const T* dy = (const T*)a.dy + q.n * a.g_sn + q.c0;
#pragma unroll 2
        for (int p = q.p0 + q.row; p < q.p1; p += q.rows) {
            float v[V], d[V];
            unpack<T, V>(*reinterpret_cast<const TV*>(x + p * a.x_sp), v);
            unpack<T, V>(*reinterpret_cast<const TV*>(dy + p * a.g_sp), d);
            backward_of<V>(k, a.act, v, d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s1[j] += d[j];
                s2[j] = fmaf(d[j], v[j], s2[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) red[threadIdx.x * V + j] = make_float2(s1[j], s2[j]);
    __syncthreads();
    const int c0 = q.c0 - ((int)threadIdx.x - q.row * q.cw) * V;
    column_sums<256>(red, q.rows, q.cw * V, [&](int c, double2 u) {
        a.bpart[((long)q.n * a.pc + q.pc) * a.C + c0 + c] = make_float2((float)u.x, (float)u.y);
    });
}

template <int FIN>
__global__ __launch_bounds__(FIN) void bwd_finish_kernel(Args a) {
    const long ng = blockIdx.x;
    const int n = (int)(ng / a.G), g = (int)(ng - (long)n * a.G);
    const double2 s = block_sum<FIN>(a.bpart + (long)n * a.pc * a.C + g * a.Cg, a.pc, a.C, a.Cg,
                                [&](int c) { return (double)param(a.w, a.wtype, g * a.Cg + c, 1.f); });
    const double m = (double)a.P * a.Cg;
    if (threadIdx.x == 0) a.means[ng] = make_float2((float)(s.x / m), (float)(s.y / m));
}

template <typename T, int V>
__global__ __launch_bounds__(256) void bwd_apply_kernel(Args a) {
    typedef typename Vec<T, V>::type TV;
    const Piece q = piece<V>(a);
    if (!q.on) return;
    Channel<V> k;
    load_params<V>(a, q.c0, k);
    load_stats<V>(a, a.stats + (long)q.n * a.G, q.c0, k);
    float m1[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float2 s = a.means[(long)q.n * a.G + (q.c0 + j) / a.Cg];
        m1[j] = s.x;
        m2[j] = s.y;
    }
    const T* x = (const T*)a.x + q.n * a.x_sn + q.c0;
    const T* dy = (const T*)a.dy + q.n * a.g_sn + q.c0;
    T* dx = (T*)a.dx + (long)q.n * a.P * a.C + q.c0;
#pragma unroll 2
    for (int p = q.p0 + q.row; p < q.p1; p += q.rows) {
        float v[V], d[V];
        unpack<T, V>(*reinterpret_cast<const TV*>(x + p * a.x_sp), v);
        unpack<T, V>(*reinterpret_cast<const TV*>(dy + p * a.g_sp), d);
        backward_of<V>(k, a.act, v, d);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = k.rs[j] * (fmaf(d[j], k.w[j], -m1[j]) - v[j] * m2[j]);
        *reinterpret_cast<TV*>(dx + (long)p * a.C) = pack<T, V>(v);
    }
}

// dw, db: the sums of all samples' pieces.  A workgroup takes four channels and 256 lanes walk the pieces, 64 rows apart (16
// channels and 16 rows per workgroup took 42 us for 2048 pieces of 320 channels: too few loads in flight).
__global__ __launch_bounds__(256) void param_grad_kernel(Args a, long items) {
    __shared__ double2 red[256];
    const int cl = threadIdx.x & 3, c = blockIdx.x * 4 + cl;
    double u = 0.0, v = 0.0;
    if (c < a.C) {
#pragma unroll 4
        for (long i = threadIdx.x >> 2; i < items; i += 64) {
            const float2 s = a.bpart[i * a.C + c];
            u += (double)s.x;
            v += (double)s.y;
        }
    }
    red[threadIdx.x] = make_double2(u, v);
    for (int o = 128; o >= 4; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) {
            red[threadIdx.x].x += red[threadIdx.x + o].x;
            red[threadIdx.x].y += red[threadIdx.x + o].y;
        }
    }
    if (threadIdx.x >= 4 || c >= a.C) return;
    put_param(a.db, a.wtype, c, red[threadIdx.x].x);
    put_param(a.dw, a.wtype, c, red[threadIdx.x].y);
}

// ------------------------------------------------------------------------------------------------ launches
struct Plan {
    int threads, r;                             // resident: threads per sample and vectors per thread; 0: in pieces
    int pc, rows_per, cc, cw;
};

// Channels per thread: four where addresses allow it (16-bit types: eight, in 16-byte loads, cost twice the registers per thread
// and so half the workgroups: 66.9 us instead of 47.5 for 800 x 196 x 64 bf16 values forward and backward, 193 instead of 170
// of kernels for 16 x 9216 x 320), two where only pairs are aligned, else one.
static int vec_of(const cmvae_group_norm& d, bool backward) {
    const int es = d.dtype == CMVAE_F32 ? 4 : 2;
    auto fits = [&](int v) {
        auto ok = [&](const void* p, const int64_t* s) { return (uintptr_t)p % (v * es) == 0 && s[0] % v == 0 && s[1] % v == 0; };
        const int64_t dense[2] = {0, 0};
        return d.C % v == 0 && ok(d.x, d.x_stride) &&
               (backward ? ok(d.dy, d.dy_stride) && ok(d.dx, dense) : ok(d.y, dense));
    };
    if (fits(4)) return 4;
    if (fits(2)) return 2;
    return 1;
}

// Resident while a sample fits: 64 threads x 4 vectors, 256 x 4, 512 x 8, 1024 x 16 (forward; half in the backward, which holds
// two tensors).  Forward + backward in us, fp32, 64 channels, resident against in pieces: 4000 samples of 16 pixels 33 / 134, 800
// of 196 55 / 89, 256 of 512 43 / 70; the forward of 256 of 1024 (1024 x 16) 29 / 42.  64 x 2 and 256 x 2: 47 for the 4000 of 16,
// 35 instead of 27 for 800 of 64.
static Plan plan_of(const cmvae_group_norm& d, int V, bool backward) {
    Plan p = {0, 0, 1, d.P, 1, 0};
    const int CV = d.C / V;
    const struct { int threads, r; } sizes[4] = {{64, 4}, {256, 4}, {512, 8}, {1024, backward ? 8 : 16}};
    for (const auto& s : sizes) {
        if (CV > s.threads || d.G > 1024) continue;
        const int rows = s.threads / CV;
        if ((long)rows * s.r >= d.P) {
            p.threads = s.threads;
            p.r = s.r;
            return p;
        }
    }
    // In pieces: six workgroups per unit (3 x 16000 x 1280 bf16, forward + backward: 200 us; four 221, eight 229), of 64 vectors of
    // channels or 128 narrow ones, evenly shared out, and the rest in rows (256 and 6: 226).
    const int widest = V == 4 ? 64 : 128;
    p.cc = (CV + widest - 1) / widest;
    p.cw = (CV + p.cc - 1) / p.cc;
    const int rows = 256 / p.cw;
    const long target = 6L * compute_units(), have = (long)d.N * p.cc;
    long pc = (target + have - 1) / have;
    const long most = (d.P + 4L * rows - 1) / (4L * rows);          // at least four pixels per thread
    if (pc > most) pc = most;
    if (pc < 1) pc = 1;
    p.rows_per = (int)((d.P + pc - 1) / pc);
    p.pc = (d.P + p.rows_per - 1) / p.rows_per;
    return p;
}

static size_t ws_bytes(const cmvae_group_norm& d, const Plan& p, bool backward) {
    const size_t nc = (size_t)d.N * p.pc * d.C;
    if (!backward) return p.threads ? 0 : nc * sizeof(double2) + (size_t)d.N * d.G * sizeof(float4);
    return nc * sizeof(float2) + 256 + (size_t)d.N * d.G * sizeof(float2);
}

// One wave per (sample, group) while a lane has at most 16 values to add, else sixteen (the backward of 1000 samples of 30 x 1280
// bf16 values, 32 groups: 95 us by one, 241 by sixteen; forward + backward of one of 16384 x 1280: 88 by sixteen, 229 by four).
template <void (*WAVE)(Args), void (*WIDE)(Args)>
static int finish(const Args& a, void* stream, const char* what) {
    const long blocks = (long)a.N * a.G;
    return (long)a.pc * a.Cg <= 1024 ? launch_kernel<WAVE>(blocks, 64, 0, a, stream, what)
                                     : launch_kernel<WIDE>(blocks, 1024, 0, a, stream, what);
}

template <typename T, int V>
static int run_fwd(Args a, const Plan& p, void* stream) {
    if (p.threads) {
        const size_t lds = (size_t)p.threads * (a.Cg % V == 0 ? 1 : V) * sizeof(double2) + a.G * sizeof(float4);
        const char* what = "group_norm fwd_resident_kernel";
        switch (p.threads) {
            case 64: return launch_kernel<fwd_resident_kernel<T, V, 64, 4>>(a.N, 64, lds, a, stream, what);
            case 256: return launch_kernel<fwd_resident_kernel<T, V, 256, 4>>(a.N, 256, lds, a, stream, what);
            case 512: return launch_kernel<fwd_resident_kernel<T, V, 512, 8>>(a.N, 512, lds, a, stream, what);
            default: return launch_kernel<fwd_resident_kernel<T, V, 1024, 16>>(a.N, 1024, lds, a, stream, what);
        }
    }
    const long blocks = (long)a.N * a.pc * a.cc;
    if (int e = launch_kernel<fwd_sums_kernel<T, V>>(blocks, 256, 0, a, stream, "group_norm fwd_sums_kernel")) return e;
    if (int e = finish<fwd_finish_kernel<64>, fwd_finish_kernel<1024>>(a, stream, "group_norm fwd_finish_kernel")) return e;
    return launch_kernel<fwd_apply_kernel<T, V>>(blocks, 256, 0, a, stream, "group_norm fwd_apply_kernel");
}

template <typename T, int V>
static int run_bwd(Args a, const Plan& p, void* stream) {
    int e;
    if (p.threads) {
        const size_t lds = (size_t)p.threads * V * sizeof(float2) + a.G * (sizeof(float4) + sizeof(float2));
        const char* what = "group_norm bwd_resident_kernel";
        switch (p.threads) {
            case 64: e = launch_kernel<bwd_resident_kernel<T, V, 64, 4>>(a.N, 64, lds, a, stream, what); break;
            case 256: e = launch_kernel<bwd_resident_kernel<T, V, 256, 4>>(a.N, 256, lds, a, stream, what); break;
            case 512: e = launch_kernel<bwd_resident_kernel<T, V, 512, 8>>(a.N, 512, lds, a, stream, what); break;
            default: e = launch_kernel<bwd_resident_kernel<T, V, 1024, 8>>(a.N, 1024, lds, a, stream, what);
        }
    } else {
        const long blocks = (long)a.N * a.pc * a.cc;
        if ((e = launch_kernel<bwd_sums_kernel<T, V>>(blocks, 256, 0, a, stream, "group_norm bwd_sums_kernel"))) return e;
        if ((e = finish<bwd_finish_kernel<64>, bwd_finish_kernel<1024>>(a, stream, "group_norm bwd_finish_kernel"))) return e;
        e = launch_kernel<bwd_apply_kernel<T, V>>(blocks, 256, 0, a, stream, "group_norm bwd_apply_kernel");
    }
    if (e || (!a.dw && !a.db)) return e;
    hipLaunchKernelGGL(param_grad_kernel, dim3((a.C + 3) / 4), dim3(256), 0, (hipStream_t)stream, a, (long)a.N * a.pc);
    return check_launch("group_norm param_grad_kernel");
}

template <typename T>
static int run(const Args& a, const Plan& p, int V, bool backward, void* stream) {
    if (V == 4) return backward ? run_bwd<T, 4>(a, p, stream) : run_fwd<T, 4>(a, p, stream);
    if (V == 2) return backward ? run_bwd<T, 2>(a, p, stream) : run_fwd<T, 2>(a, p, stream);
    return backward ? run_bwd<T, 1>(a, p, stream) : run_fwd<T, 1>(a, p, stream);
}

static int check_desc(const char* who, const cmvae_group_norm* d) {
    CMVAE_REQUIRE(d != nullptr, "%s: NULL descriptor", who);
    CMVAE_REQUIRE(d->dtype >= CMVAE_F32 && d->dtype <= CMVAE_F16 && (d->wdtype == CMVAE_F32 || d->wdtype == d->dtype),
                  "%s: dtype %d, parameters %d (fp32 or the data's)", who, d->dtype, d->wdtype);
    CMVAE_REQUIRE(d->N >= 1 && d->P >= 1 && d->C >= 1 && d->G >= 1 && d->C % d->G == 0, "%s: N=%d P=%d C=%d groups=%d", who, d->N,
                  d->P, d->C, d->G);
    CMVAE_REQUIRE(d->act >= 0 && d->act <= 3, "%s: activation %d", who, d->act);
    CMVAE_REQUIRE(d->eps >= 0.f && std::isfinite(d->eps), "%s: eps %g", who, (double)d->eps);
    CMVAE_REQUIRE(d->x_stride[0] >= 0 && d->x_stride[1] >= 0, "%s: strides of x", who);
    CMVAE_REQUIRE((long)d->N * d->G < (1L << 31) && d->C <= (1 << 24) && d->P <= (1 << 30), "%s: too large", who);
    const uintptr_t es = d->dtype == CMVAE_F32 ? 4 : 2, ws = d->wdtype == CMVAE_F32 ? 4 : 2;
    CMVAE_REQUIRE((((uintptr_t)d->x | (uintptr_t)d->y | (uintptr_t)d->dy | (uintptr_t)d->dx) & (es - 1)) == 0 &&
                      (((uintptr_t)d->weight | (uintptr_t)d->bias | (uintptr_t)d->dweight | (uintptr_t)d->dbias) & (ws - 1)) == 0 &&
                      ((uintptr_t)d->stats & 15) == 0,
                  "%s: a tensor is not aligned", who);
    return 0;
}

static Args args_of(const cmvae_group_norm& d, const Plan& p, int V) {
    Args a = {};
    a.x = d.x; a.dy = d.dy; a.w = d.weight; a.b = d.bias;
    a.y = d.y; a.dx = d.dx; a.dw = d.dweight; a.db = d.dbias;
    a.stats = (float4*)d.stats;
    a.x_sn = d.x_stride[0]; a.x_sp = d.x_stride[1];
    a.g_sn = d.dy_stride[0]; a.g_sp = d.dy_stride[1];
    a.N = d.N; a.P = d.P; a.C = d.C; a.G = d.G; a.Cg = d.C / d.G; a.CV = d.C / V;
    a.act = d.act; a.wtype = d.wdtype; a.xtype = d.dtype; a.eps = d.eps;
    a.pc = p.pc; a.rows_per = p.rows_per; a.cc = p.cc; a.cw = p.cw;
    return a;
}

static int enter(const char* who, const cmvae_group_norm* d, bool backward, void* workspace, size_t workspace_bytes, void* stream) {
    if (int e = check_desc(who, d)) return e;
    if (backward)
        CMVAE_REQUIRE(d->x && d->dy && d->dx && d->stats && d->dy_stride[0] >= 0 && d->dy_stride[1] >= 0, "%s: NULL tensor", who);
    else
        CMVAE_REQUIRE(d->x && d->y, "%s: NULL tensor", who);
    const int V = vec_of(*d, backward);
    const Plan p = plan_of(*d, V, backward);
    const size_t need = ws_bytes(*d, p, backward);
    CMVAE_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= need),
                  "%s: workspace of %zu bytes, %zu needed", who, workspace_bytes, need);
    CMVAE_REQUIRE((long)d->N * p.pc * p.cc < (1L << 31), "%s: too large", who);
    Args a = args_of(*d, p, V);
    if (backward) {
        a.bpart = (float2*)workspace;
        a.means = (float2*)((char*)workspace + align_up((size_t)d->N * p.pc * d->C * sizeof(float2)));
    } else if (!p.threads) {
        a.part = (double2*)workspace;
        if (!a.stats) a.stats = (float4*)(a.part + (size_t)d->N * p.pc * d->C);
    }
    switch (d->dtype) {
        case CMVAE_F32: return run<float>(a, p, V, backward, stream);
        case CMVAE_BF16: return run<__bf16>(a, p, V, backward, stream);
        default: return run<_Float16>(a, p, V, backward, stream);
    }
}

}  // namespace gn
}  // namespace cmvae

using namespace cmvae;

extern "C" size_t cmvae_group_norm_workspace_bytes(const cmvae_group_norm* d, int backward) {
    cmvae::clear_stale_error();
    if (gn::check_desc("cmvae_group_norm_workspace_bytes", d)) return 0;
    const int V = gn::vec_of(*d, backward != 0);
    return gn::ws_bytes(*d, gn::plan_of(*d, V, backward != 0), backward != 0);
}

extern "C" int cmvae_group_norm_fwd(const cmvae_group_norm* d, void* workspace, size_t workspace_bytes, void* stream) {
    cmvae::clear_stale_error();
    return gn::enter("cmvae_group_norm_fwd", d, false, workspace, workspace_bytes, stream);
}

extern "C" int cmvae_group_norm_bwd(const cmvae_group_norm* d, void* workspace, size_t workspace_bytes, void* stream) {
    cmvae::clear_stale_error();
    return gn::enter("cmvae_group_norm_bwd", d, true, workspace, workspace_bytes, stream);
}
