// Losses and read-outs on rows of vocabulary logits (fp32, fp16 or bf16), gfx950 only: the k largest logits of a row,
// the log-probability of a row's token, and the distillation, policy and preference losses with their gradients.
//
// Every operator is a reduction over a row of V logits (a soft-max's maximum and sum and little else) followed, for a
// gradient, by a map over the same row.  Each does a handful of operations per logit, so what bounds them is the row's
// way through memory: V elements in, V elements out.  One block takes one row; sums are held in 32 bits, what is one
// number per row (logarithms, ratios, losses) in 64.
//
// A row whose target is the pad symbol, or whose mask byte is zero, is not read: its outputs are zero.
#include "gtg_internal.h"

#include <type_traits>

namespace gtg {
namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

constexpr double LOG2E = 1.4426950408889634, LN2 = 0.6931471805599453;
__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }
// The hardware's 2^x: 1 step off at most, 0 where the result would lie below 2^-126.  The library's exp2f spends five more
// instructions on those, as much again as everything else done per logit.
__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes of logits, element by element as fp32.
struct F32 {
    typedef float Store;
    // the larger elements of the vectors taken, of every vector's first and second half (16-bit types: even and odd places)
    struct Maxima {
        float a = -__builtin_inff(), b = -__builtin_inff();
        __device__ __forceinline__ void take(const u32x4& v)
        {
            a = fmaxf(fmaxf(a, get(v, 0)), get(v, 1));
            b = fmaxf(fmaxf(b, get(v, 2)), get(v, 3));
        }
        __device__ __forceinline__ float lo() const { return a; }
        __device__ __forceinline__ float hi() const { return b; }
    };
    static constexpr int VEC = 4;
    static constexpr unsigned NEG2 = 0xff800000u;  // -inf in every element of a dword
    __device__ static float get(const u32x4& v, int q) { return __uint_as_float(v[q]); }
    __device__ static void clear(u32x4& v, int q) { v[q] = 0xff800000u; }
    // element q, not known to the compiler, leaving -inf in its place
    __device__ static float take(u32x4& v, int q)
    {
        unsigned d = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            d = q == i ? v[i] : d;
            v[i] = q == i ? 0xff800000u : v[i];
        }
        return __uint_as_float(d);
    }
    __device__ static float load(const Store* p) { return *p; }
    __device__ static Store cvt(float f) { return f; }
    __device__ static u32x4 pack(const float* f)
    {
        u32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = __float_as_uint(f[q]);
        return v;
    }
};
// Without unpacking: 16-bit floats are in the order of their bits as integers where they are positive and in reverse where they are
// negative, so the largest is the largest signed integer, or, if that is negative, the smallest unsigned one.
template <unsigned NEG2, typename H>
struct Maxima16 {
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    unsigned p = NEG2, n = NEG2;
    __device__ __forceinline__ void take(const u32x4& v)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned w = v[i];  // (a bit cast of v[i] itself would read v[0])
            p = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(i16x2, p), __builtin_bit_cast(i16x2, w)));
            n = __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(u16x2, n), __builtin_bit_cast(u16x2, w)));
        }
    }
    __device__ __forceinline__ float lo() const { return H::widen((p & 0x8000u) ? n & 0xffffu : p & 0xffffu); }
    __device__ __forceinline__ float hi() const { return H::widen((p & 0x80000000u) ? n >> 16 : p >> 16); }
};
struct BF16 {
    typedef __bf16 Store;
    __device__ static float widen(unsigned bits) { return __uint_as_float(bits << 16); }
    typedef Maxima16<0xff80ff80u, BF16> Maxima;
    static constexpr int VEC = 8;
    static constexpr unsigned NEG2 = 0xff80ff80u;  // -inf in every element of a dword
    __device__ static float get(const u32x4& v, int q)
    {
        return __uint_as_float((q & 1) ? (v[q >> 1] & 0xffff0000u) : (v[q >> 1] << 16));
    }
    __device__ static void clear(u32x4& v, int q)
    {
        v[q >> 1] = (q & 1) ? ((v[q >> 1] & 0xffffu) | 0xff800000u) : ((v[q >> 1] & 0xffff0000u) | 0xff80u);
    }
    __device__ static float take(u32x4& v, int q)
    {
        const int at = (q & 1) * 16;
        unsigned d = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool here = q >> 1 == i;
            d = here ? v[i] : d;
            v[i] = here ? (v[i] & ~(0xffffu << at)) | (0xff80u << at) : v[i];
        }
        d = d >> at & 0xffffu;
        return __uint_as_float(d << 16);
    }
    __device__ static float load(const Store* p) { return (float)*p; }
    __device__ static Store cvt(float f) { return (__bf16)f; }
    __device__ static u32x4 pack(const float* f)
    {
        u32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x2 two = {f[2 * q], f[2 * q + 1]};
            v[q] = __builtin_bit_cast(unsigned, __builtin_convertvector(two, bf16x2));
        }
        return v;
    }
};
struct F16 {
    typedef _Float16 Store;
    __device__ static float widen(unsigned bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }
    typedef Maxima16<0xfc00fc00u, F16> Maxima;
    static constexpr int VEC = 8;
    static constexpr unsigned NEG2 = 0xfc00fc00u;  // -inf in every element of a dword
    __device__ static float get(const u32x4& v, int q)
    {
        return (float)__builtin_bit_cast(_Float16, (unsigned short)((q & 1) ? (v[q >> 1] >> 16) : (v[q >> 1] & 0xffffu)));
    }
    __device__ static void clear(u32x4& v, int q)
    {
        v[q >> 1] = (q & 1) ? ((v[q >> 1] & 0xffffu) | 0xfc000000u) : ((v[q >> 1] & 0xffff0000u) | 0xfc00u);
    }
    __device__ static float take(u32x4& v, int q)
    {
        const int at = (q & 1) * 16;
        unsigned d = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool here = q >> 1 == i;
            d = here ? v[i] : d;
            v[i] = here ? (v[i] & ~(0xffffu << at)) | (0xfc00u << at) : v[i];
        }
        d = d >> at & 0xffffu;
        return (float)__builtin_bit_cast(_Float16, (unsigned short)d);
    }
    __device__ static float load(const Store* p) { return (float)*p; }
    __device__ static Store cvt(float f) { return (_Float16)f; }
    __device__ static u32x4 pack(const float* f)
    {
        u32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x2 two = {f[2 * q], f[2 * q + 1]};
            v[q] = __builtin_bit_cast(unsigned, __builtin_convertvector(two, f16x2v));
        }
        return v;
    }
};

// ---- a row and how a block of NT threads walks over it --------------------------------------------------------
// The row is cut where 16-byte alignment begins and ends: up to VEC - 1 elements in front and behind, taken one each by
// the first 2 VEC threads (`xe`, `je`), and the body of whole vectors between them, vector i by thread i mod NT.  No
// access leaves the row, whatever its alignment and length.
// NV > 0: the body is loaded once into NV vectors of registers per thread (places past its end hold -inf) and every
// sweep works on those: one read of the row.  NV == 0: every sweep reads the row again.
// ONCE: nobody reads the row after this (loads that leave the caches to others).
// MARKED: classes marked in a bit map (LDS, Marks below) count as -inf: removed from the registers once, or as each vector is read.
// Waves per SIMD that the kernels on NV vectors a thread are held to: enough blocks per CU to load one row while another is
// summed or stored.
constexpr int min_waves(int nv) { return nv == 16 ? 4 : nv == 8 ? 6 : 8; }
template <typename E, int NT, int NV, bool MARKED = false, bool ONCE = false>
struct Row {
    typedef typename E::Store S;
    static constexpr int VEC = E::VEC;
    const S* p;
    int V, head, nb, je;  // elements in front, vectors in the body, this thread's single element or -1
    float xe;             // its value, -inf if there is none
    const unsigned char* marks;
    u32x4 v[NV > 0 ? NV : 1];

    __device__ Row(const S* row, int vocab) : p(row), V(vocab), marks(nullptr)
    {
        const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(S));
        head = off ? VEC - off : 0;
        if (head > V) head = V;
        nb = (V - head) / VEC;
        const int tail0 = head + nb * VEC, t = threadIdx.x;
        je = t < head ? t : (t >= VEC && t < 2 * VEC && tail0 + t - VEC < V ? tail0 + t - VEC : -1);
        xe = neg_inf();
    }
    __device__ const u32x4* body() const { return reinterpret_cast<const u32x4*>(p + head); }
    __device__ __forceinline__ void load()
    {
        if constexpr (NV > 0) {
            const u32x4* b = body();
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int i = threadIdx.x + k * NT;
                v[k] = u32x4{E::NEG2, E::NEG2, E::NEG2, E::NEG2};
                if (i < nb) v[k] = ONCE ? __builtin_nontemporal_load(b + i) : b[i];
            }
        }
        if (je >= 0) xe = E::load(p + je);
    }
    // the bit map's place of class j: one bit each, the body's vectors beginning at whole bytes (nibbles for VEC = 4)
    __device__ __forceinline__ int mark_place(int j) const { return j - head + VEC; }
    __device__ __forceinline__ void take_out(u32x4& x, int i) const
    {
        const unsigned m = VEC == 8 ? marks[i + 1] : (marks[(i + 1) >> 1] >> (4 * ((i + 1) & 1))) & 15u;
        if (m) {
#pragma unroll
            for (int q = 0; q < VEC; ++q)
                if (m >> q & 1) E::clear(x, q);
        }
    }
    __device__ __forceinline__ void mark(const unsigned* bits)
    {
        marks = reinterpret_cast<const unsigned char*>(bits);
        if constexpr (NV > 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int i = threadIdx.x + k * NT;
                if (i < nb) take_out(v[k], i);
            }
        }
        if (je >= 0) {
            const int at = mark_place(je);
            if (bits[at >> 5] >> (at & 31) & 1) xe = neg_inf();
        }
    }
    // f(value) in place of every value of the registers
    template <typename F>
    __device__ __forceinline__ void replace(F f)
    {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            asm volatile("" : "+v"(v[k]));
            float x[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) x[q] = f(E::get(v[k], q));
            v[k] = E::pack(x);
        }
        xe = f(xe);
    }
    // f(index of the vector's first element, vector); ALL: also the places past the body's end, which hold -inf
    template <bool ALL, typename F>
    __device__ __forceinline__ void each(F f)
    {
        if constexpr (NV > 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                // new to the compiler in every sweep, and one vector after the other: it would otherwise keep what it
                // unpacked for the last sweep, or unpack all vectors at once -- twice the registers, half the waves
                asm volatile("" : "+v"(v[k]));
                const int i = threadIdx.x + k * NT;
                if (ALL || i < nb) f(head + i * VEC, v[k]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            const u32x4* b = body();
            for (int i = threadIdx.x; i < nb; i += NT) {
                u32x4 x = b[i];
                if (MARKED) take_out(x, i);
                f(head + i * VEC, x);
            }
        }
    }
};

template <typename E>
__device__ __forceinline__ float vec_max(float m, const u32x4& v)
{
#pragma unroll
    for (int q = 0; q < E::VEC; ++q) m = fmaxf(m, E::get(v, q));
    return m;
}

// A gradient row: vectors where its alignment is the logits' own, single elements otherwise.  The vectors' stores are
// non-temporal: written back at leisure, a gradient of more than the last-level cache's 256 MB otherwise pushes out the logits that are still
// to be read (10 240 x 30 522: log-probability and its gradient, fp32, 558 us without and 445 us with; policy loss, bf16, 231 and 217).
template <typename E>
struct OutRow {
    typename E::Store* p;
    bool aligned;
    __device__ OutRow(void* base, int64_t ld, int64_t r, const typename E::Store* in)
        : p(reinterpret_cast<typename E::Store*>(base) + r * ld),
          aligned(((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(in)) & 15) == 0)
    {
    }
    __device__ __forceinline__ void vec(int j, const float* f) const
    {
        if (aligned) {
            __builtin_nontemporal_store(E::pack(f), reinterpret_cast<u32x4*>(p + j));
        } else {
#pragma unroll
            for (int q = 0; q < E::VEC; ++q) p[j + q] = E::cvt(f[q]);
        }
    }
    __device__ __forceinline__ void one(int j, float f) const { p[j] = E::cvt(f); }
};

// The i-th row of a launch of n, for kernels that write a gradient row by row: of every 256 rows each of the eight dies (blocks go to them
// in turn) takes 32 that follow each other.  Policy loss, 10 240 x 30 522 bf16: 226 us in plain order, 217 us so.
__device__ __forceinline__ unsigned dealt(unsigned i, unsigned n)
{
    constexpr unsigned G = 32, S = 8 * G;
    if (i >= n / S * S) return i;
    const unsigned w = i % S;
    return i - w + (w & 7) * G + (w >> 3);
}

template <int NT, typename R, typename E>
__device__ __forceinline__ void fill_row(const R& row, const OutRow<E>& out, float value)
{
    float f[E::VEC];
#pragma unroll
    for (int q = 0; q < E::VEC; ++q) f[q] = value;
    for (int i = threadIdx.x; i < row.nb; i += NT) out.vec(row.head + i * E::VEC, f);
    if (row.je >= 0) out.one(row.je, value);
}

// ---- reductions over a block ------------------------------------------------------------------------------------
// Within a row of 16 lanes by DPP (two quad permutations and two mirrors: 4 instructions, no LDS), across the four rows by
// reading one lane of each: the same bits in every lane.
template <int CTRL>
__device__ __forceinline__ int dpp(int v)
{
    return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v)
{
    return __int_as_float(dpp<CTRL>(__float_as_int(v)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v)
{
    return __hiloint2double(dpp<CTRL>(__double2hiint(v)), dpp<CTRL>(__double2loint(v)));
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float lane_value(float v, int lane) { return __int_as_float(lane_value(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_value(double v, int lane)
{
    return __hiloint2double(lane_value(__double2hiint(v), lane), lane_value(__double2loint(v), lane));
}
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T v, F f)
{
    v = f(v, dpp<0xb1>(v));   // lanes 1 0 3 2 of every four
    v = f(v, dpp<0x4e>(v));   // lanes 2 3 0 1
    v = f(v, dpp<0x141>(v));  // every eight mirrored
    v = f(v, dpp<0x140>(v));  // every sixteen mirrored
    return f(f(lane_value(v, 0), lane_value(v, 16)), f(lane_value(v, 32), lane_value(v, 48)));
}
__device__ __forceinline__ float wave_max(float v) { return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
template <typename T>
__device__ __forceinline__ T wave_sum(T v)
{
    return wave_reduce(v, [](T a, T b) { return a + b; });
}

// Over the block, through one place of LDS per wave.  AGAIN: the places may still be read from an earlier call.
template <int NT, bool AGAIN, typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* sh, F f)
{
    v = wave_reduce(v, f);
    if (NT == 64) return v;
    if (AGAIN) __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = f(v, sh[w]);
    return v;
}
template <int NT, bool AGAIN>
__device__ __forceinline__ float block_max(float v, float* sh)
{
    return block_reduce<NT, AGAIN>(v, sh, [](float a, float b) { return fmaxf(a, b); });
}
template <int NT, bool AGAIN, typename T>
__device__ __forceinline__ T block_sum(T v, T* sh)
{
    return block_reduce<NT, AGAIN>(v, sh, [](T a, T b) { return a + b; });
}

// ---- exponential and logarithm in 64 bits, for one number per row --------------------------------------------------
// Short forms, to 1e-14 relative: the row waits in registers while they run, and the library's need as many again.
// e^x = 2^n e^r with r = x - n ln 2, |r| <= 0.35, by its Taylor series; log x = e ln 2 + 2 atanh((m - 1) / (m + 1)) for x = 2^e m
// with m in [sqrt(1/2), sqrt(2)], by the series of atanh, |argument| <= 0.172.
__device__ __forceinline__ double exp_row(double x)
{
    const double in = fmin(fmax(x, -800.0), 800.0), n = rint(in * LOG2E);
    const double r = fma(-n, 1.9082149292705877e-10, fma(-n, 0.6931471803691238, in));
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return x != x ? x : ldexp(p, (int)n);
}
__device__ __forceinline__ double log_row(double x)
{
    int e;
    double m = frexp(x, &e);
    if (m < 0.70710678118654752) {
        m *= 2.0;
        e -= 1;
    }
    const double z = (m - 1.0) / (m + 1.0), q = z * z;
    double p = 1.0 / 19.0;
    p = fma(p, q, 1.0 / 17.0);
    p = fma(p, q, 1.0 / 15.0);
    p = fma(p, q, 1.0 / 13.0);
    p = fma(p, q, 1.0 / 11.0);
    p = fma(p, q, 1.0 / 9.0);
    p = fma(p, q, 1.0 / 7.0);
    p = fma(p, q, 1.0 / 5.0);
    p = fma(p, q, 1.0 / 3.0);
    p = fma(p, q, 1.0);
    const double l = fma((double)e, 0.69314718055994531, 2.0 * z * p);
    return x == 0.0 ? -__builtin_inf() : x == __builtin_inf() ? x : l;
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == neg_inf() ? 0.f : m; }
// An exponent from below at -1024, where its power is 0 already: what is multiplied with that 0 -- the exponent itself, or its
// product with a gradient's coefficient -- then stays finite and the product is 0, not NaN (masked logits).
__device__ __forceinline__ float clamped(float d) { return fmaxf(d, -1024.f); }

// ---- which rows count -------------------------------------------------------------------------------------------
struct Rows {
    const void* x;       // logits, row r at x + r ld
    int64_t ld;
    int vocab;
    const int64_t* targets;
    int64_t pad;
    const uint8_t* mask;  // nullable
    int64_t first;        // the launch's first row and their number (more rows than a launch takes go in several)
    unsigned n;
    __device__ __forceinline__ bool kept(int64_t r) const { return targets[r] != pad && (mask == nullptr || mask[r] != 0); }
};

// What a row's gradient is multiplied with: gloss[r], *gscale and *norm, each 1 where absent.
struct Weight {
    const float* gloss;
    const float* gscale;
    double* norm;
    int64_t count;  // 0, or: *norm is still to be found, by counting this many rows (block 0 stores it)
    __device__ __forceinline__ double of(int64_t r, double n) const
    {
        return (gloss ? (double)gloss[r] : 1.0) * (gscale ? (double)*gscale : 1.0) * n;
    }
};

// The factor of the mean, in every thread.  Up to COUNT_IN_ROWS rows every block counts them itself: at most 8 KB from
// L2 per block, against a launch and a block's latency in front of the rows (4.5 us).
constexpr int COUNT_IN_ROWS = 1024;
template <int NT>
__device__ __forceinline__ double mean_norm(const Rows& rows, const Weight& w)
{
    __shared__ int sh[16];
    if (w.count == 0) return w.norm ? *w.norm : 1.0;
    int n = 0;
    for (int r = threadIdx.x; r < (int)w.count; r += NT) n += rows.kept(r) ? 1 : 0;
    n = block_sum<NT, false>(n, sh);
    const double norm = n > 0 ? 1.0 / (double)n : 0.0;
    if (rows.first + blockIdx.x == 0 && threadIdx.x == 0) *w.norm = norm;
    return norm;
}

// 1 / (rows that count), 0 if none does.
__global__ __launch_bounds__(1024) void count_kernel(Rows rows, int64_t R, double* __restrict__ norm)
{
    __shared__ int sh[16];
    int n = 0;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < R; r += 1024) n += rows.kept(r) ? 1 : 0;
    n = block_sum<1024, false>(n, sh);
    if (threadIdx.x == 0) *norm = n > 0 ? 1.0 / (double)n : 0.0;
}

// loss = (*norm or 1) * sum of row_loss, in 64 bits and a fixed order
__global__ __launch_bounds__(1024) void total_kernel(const float* __restrict__ row_loss, int64_t R,
                                                     const double* __restrict__ norm, float* __restrict__ loss)
{
    __shared__ double sh[16];
    double s = 0.0;
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < R; r += 1024) s += (double)row_loss[r];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 16; ++w) s += sh[w];
        *loss = R > 0 ? (float)(s * (norm ? *norm : 1.0)) : 0.f;
    }
}

// ---- maximum, sum of exponentials and a second sum -----------------------------------------------------------------
// A logit's place below the row's maximum m is taken in powers of two with one rounding: y = x c - mu, c = log2(e) / tau
// and mu = m c, both rounded; 2^y is within 2^-24 |y| + 2^-23 of the exact power, and a sum of them is read relative to mu.
// mu's own rounding is a common factor of 2^(m c - mu).  Where mu is so large that this is no small one (logits of a million,
// masks of the type's lowest value in all places) the row is made flat first: x - m takes the place of x, mu is 0.
struct Scale {
    float c, mu, m;
    bool flat;
    __device__ __forceinline__ Scale(float m_, float c_) : c(c_), m(m_)
    {
        mu = m * c;
        flat = m != neg_inf() && m != __builtin_inff() && !(fabsf(mu) < 1048576.f);
        if (flat || m == neg_inf()) mu = 0.f;
    }
    __device__ __forceinline__ void make_flat()
    {
        flat = true;
        mu = 0.f;
    }
    __device__ __forceinline__ float y(float x) const { return fmaf(x, c, -mu); }
    // in 64 bits and units of e: the log of a logit's exponential relative to the sums' reference.  With the rounded c, like the
    // sums: a soft-max whose temperature is 2^-25 off is a soft-max still, and a divergence near zero stays near zero.
    __device__ __forceinline__ double log_of(float x) const
    {
        return flat ? ((double)x - (double)m) * (double)c * LN2 : fma((double)x, (double)c, -(double)mu) * LN2;
    }
    // the sums' own reference relative to another logit `to`, likewise
    __device__ __forceinline__ double log_ref(float to) const
    {
        if (m == neg_inf()) return -__builtin_inf();
        return flat ? ((double)m - (double)to) * (double)c * LN2 : fma(-(double)to, (double)c, (double)mu) * LN2;
    }
    // this reference minus another's, in powers of two
    __device__ __forceinline__ float above(const Scale& o) const
    {
        if (flat) return o.flat ? (m - o.m) * c : fmaf(m, c, -o.mu);
        return o.flat ? fmaf(-o.m, c, mu) : mu - o.mu;
    }
};

// s = sum 2^y and by KIND a second sum: MOMENT: t = sum 2^y y; TWO: t = sum 2^y1 by a second scale; NONE.
enum Second { NONE, MOMENT, TWO };
struct Stats {
    float s = 0.f, t = 0.f;
    template <Second KIND>
    __device__ __forceinline__ void add(float x, const Scale& a, const Scale& b)
    {
        const float y = a.y(x), e = exp2_raw(y);
        s += e;
        if (KIND == MOMENT) t = fmaf(e, clamped(y), t);
        if (KIND == TWO) t += exp2_raw(b.y(x));
    }
};

// Every thread gets the row's m (in a and b) and sums.  Rows in registers: the maximum of the whole row first, then the
// sums.  Rows read again in every sweep: one sweep for both, each thread relative to the largest logit it has met, joined at
// the end.  sh: 3 x 16 places.
template <Second KIND, typename E, int NT, int NV, bool MARKED, bool ONCE>
__device__ __forceinline__ Stats row_stats(Row<E, NT, NV, MARKED, ONCE>& row, float c, float c1, Scale& a, Scale& b, float* sh)
{
    Stats r;
    if constexpr (NV > 0) {
        float m = neg_inf();
        row.template each<true>([&](int, const u32x4& v) { m = vec_max<E>(m, v); });
        m = block_max<NT, false>(fmaxf(m, row.xe), sh);
        a = Scale(m, c);
        b = Scale(m, c1);
        if (a.flat || (KIND == TWO && b.flat)) {
            if (m != neg_inf()) row.replace([&](float x) { return x - m; });
            a.make_flat();
            b.make_flat();
        }
        row.template each<true>([&](int, const u32x4& v) {
#pragma unroll
            for (int q = 0; q < E::VEC; ++q) r.add<KIND>(E::get(v, q), a, b);
        });
        r.add<KIND>(row.xe, a, b);
    } else {
        float m = row.xe;
        auto start = [&](float M) {
            a = Scale(M, c);
            b = Scale(M, c1);
            if (KIND == TWO && (a.flat || b.flat)) {
                a.make_flat();
                b.make_flat();
            }
        };
        start(m);
        auto raise = [&](float M) {  // the sums so far to the maximum M > m
            const Scale o = a, o1 = b;
            start(M);
            const float d = o.m == neg_inf() ? neg_inf() : o.above(a), f = exp2_raw(d);
            if (KIND == MOMENT) r.t = f == 0.f ? 0.f : f * (r.t + d * r.s);
            if (KIND == TWO) r.t *= o.m == neg_inf() ? 0.f : exp2_raw(o1.above(b));
            r.s *= f;  // (0 of a sum without terms; a NaN stays)
            m = M;
        };
        if (m != neg_inf()) r.add<KIND>(a.flat ? 0.f : m, a, b);
        row.template each<true>([&](int, const u32x4& v) {
            const float vm = vec_max<E>(neg_inf(), v);
            if (vm > m) raise(vm);
#pragma unroll
            for (int q = 0; q < E::VEC; ++q) {
                const float x = E::get(v, q);
                r.add<KIND>(a.flat ? x - m : x, a, b);
            }
        });
        const float M = block_max<NT, false>(m, sh);
        if (M > m) raise(M);
    }
    // (kept from moving the sums, sweep and all, to where they are used)
    asm volatile("" : "+v"(r.s), "+v"(r.t));
    if (NT > 64) sh += 16;
    r.s = block_sum<NT, false>(r.s, sh);
    if (NT > 64) sh += 16;
    if (KIND != NONE) r.t = block_sum<NT, false>(r.t, sh);
    if (r.s == __builtin_inff()) r.s = __builtin_nanf("");
    return r;
}

// The gradient's sweep: grad(logit) for every one, gy more at class `target` (-1: none).  FLATTEN: the row's vectors hold
// logits as they stand in memory and the scale wants them flat.
template <bool FLATTEN, typename R, typename E, typename F>
__device__ __forceinline__ void store_sweep(R& row, const OutRow<E>& out, const Scale& a, int target, float gy, F grad)
{
    auto value = [&](float x) { return grad(FLATTEN ? x - a.m : x); };
    row.template each<false>([&](int j, const u32x4& v) {
        float f[E::VEC];
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) f[q] = value(E::get(v, q));
        if ((unsigned)(target - j) < (unsigned)E::VEC) {
#pragma unroll
            for (int q = 0; q < E::VEC; ++q)
                if (target == j + q) f[q] += gy;
        }
        out.vec(j, f);
    });
    if (row.je >= 0) out.one(row.je, value(row.xe) + (row.je == target ? gy : 0.f));
}
template <bool HELD, typename R, typename E, typename F>
__device__ __forceinline__ void store_row(R& row, const OutRow<E>& out, const Scale& a, int target, float gy, F grad)
{
    // (rows held in registers are flat already where the scale is)
    if (!HELD && a.flat) store_sweep<true>(row, out, a, target, gy, grad);
    else store_sweep<false>(row, out, a, target, gy, grad);
}

// ---- log-probability and entropy ---------------------------------------------------------------------------------
// logp = (x_y - m) / tau - log s, entropy H = log s + u, u = -ln 2 t / s.  stats (R, 4): m, 1 / s, u, unused: what the backward
// needs.  logp64 (R): the log-probability unrounded, for the sums of the preference loss.
struct LogprobOut {
    float* logp;
    float* entropy;
    float4* stats;
    double* logp64;
};

template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, min_waves(NV)) void logprob_kernel(Rows rows, double inv_tau, LogprobOut out)
{
    __shared__ float sh[48];
    const int64_t r = rows.first + blockIdx.x;
    if (!rows.kept(r)) {
        if (threadIdx.x == 0) {
            if (out.logp) out.logp[r] = 0.f;
            if (out.entropy) out.entropy[r] = 0.f;
            if (out.logp64) out.logp64[r] = 0.0;
        }
        return;
    }
    const typename E::Store* x = reinterpret_cast<const typename E::Store*>(rows.x) + r * rows.ld;
    Row<E, NT, NV> row(x, rows.vocab);
    row.load();
    Scale sc(neg_inf(), 0.f), unused(neg_inf(), 0.f);
    const Stats a = row_stats<MOMENT>(row, (float)(LOG2E * inv_tau), 0.f, sc, unused, sh);
    if (threadIdx.x == 0) {
        const int64_t y = rows.targets[r];
        const double log_s = log_row((double)a.s), u = -(double)a.t / (double)a.s * LN2;
        const double lp = (y >= 0 && y < rows.vocab) ? sc.log_of(E::load(x + y)) - log_s : __builtin_nan("");
        if (out.logp) out.logp[r] = (float)lp;
        if (out.entropy) out.entropy[r] = (float)(log_s + u);
        if (out.logp64) out.logp64[r] = lp;
        if (out.stats) out.stats[r] = make_float4(sc.m, 1.f / a.s, (float)u, 0.f);
    }
}

// d/dx_j = (1/tau) [ g_l (1[j = y] - p_j) - g_H p_j (log p_j + H) ],  log p_j + H = ln 2 y_j + u
// The coefficients g_l are one per row, or one per sequence: group 0: g_l[r], S > 0: g_l[r mod S] (time-major),
// S < 0: g_l[r / -S] (sequence by sequence).
struct RowGrad {
    const float4* stats;
    const float* g_logp;
    const float* g_entropy;  // nullable
    const float* gscale;     // nullable, one number
    const float* gloss;      // nullable, one number per pair of sequences: g_l times gloss[sequence mod (S / 2)]
    int64_t group;
    int64_t pairs;
    double inv_tau;
    void* dx;
    int64_t ldg;
};

// Nothing is reduced here, so a block takes not a row but a piece of one, BWD_VEC vectors a thread, and the pieces follow each
// other through memory, the last one first: the forward read the rows in order, and what it read last is still in the
// last-level cache.  10 240 x 30 522 fp32, 60 % of the rows counting, forward and backward: a block per row 576 us; pieces of one vector a thread
// 689 us, reversed 657 us, with non-temporal stores 560 us; of two vectors 534 us, reversed and non-temporal 445 us; of four 494 us.
constexpr int BWD_NT = 256, BWD_VEC = 2;

template <typename E>
__global__ __launch_bounds__(BWD_NT) void logprob_bwd_kernel(Rows rows, RowGrad g, unsigned pieces, unsigned per_row)
{
    constexpr int VEC = E::VEC;
    for (unsigned p0 = blockIdx.x; p0 < pieces; p0 += gridDim.x) {
        const unsigned p = pieces - 1 - p0, r = p / per_row, piece = p - r * per_row;
        const typename E::Store* x = reinterpret_cast<const typename E::Store*>(rows.x) + r * rows.ld;
        Row<E, BWD_NT, 0> row(x, rows.vocab);
        const OutRow<E> out(g.dx, g.ldg, r, x);
        const bool kept = rows.kept(r), single = piece == 0 && row.je >= 0;
        const int i0 = (int)piece * BWD_NT * BWD_VEC + threadIdx.x;
        u32x4 v[BWD_VEC];
        if (kept) {
#pragma unroll
            for (int k = 0; k < BWD_VEC; ++k) {
                v[k] = u32x4{0, 0, 0, 0};
                if (i0 + k * BWD_NT < row.nb) v[k] = row.body()[i0 + k * BWD_NT];
            }
            if (single) row.xe = E::load(x + row.je);
        }
        float gl = 0.f, gh = 0.f;
        float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
        int y = -1;
        if (kept) {
            const int64_t y64 = rows.targets[r];
            const unsigned S = (unsigned)(g.group < 0 ? -g.group : g.group), b = g.group == 0 ? r : g.group > 0 ? r % S : r / S;
            if (g.g_logp) gl = g.g_logp[b];
            if (g.gscale) gl *= *g.gscale;
            if (g.gloss) gl *= g.gloss[b % (unsigned)g.pairs];
            if (y64 < 0 || y64 >= rows.vocab) gl = __builtin_nanf("");
            else y = (int)y64;
            if (g.g_entropy) gh = g.g_entropy[r];
            st = g.stats[r];
        }
        const Scale a(st.x, (float)(LOG2E * g.inv_tau));
        // 2^y (k0 + k1 y) + [j = target] gy
        const float it = (float)g.inv_tau, gy = gl * it, k0 = -(gl + gh * st.z) * it * st.y, k1 = -gh * it * st.y * (float)LN2;
        auto value = [&](float xv) {
            const float e = a.y(a.flat ? xv - a.m : xv);
            return exp2_raw(e) * fmaf(k1, clamped(e), k0);
        };
#pragma unroll
        for (int k = 0; k < BWD_VEC; ++k) {
            const int i = i0 + k * BWD_NT, j = row.head + i * VEC;
            if (i >= row.nb) continue;
            float f[VEC];
#pragma unroll
            for (int q = 0; q < VEC; ++q) f[q] = kept ? value(E::get(v[k], q)) : 0.f;
            if ((unsigned)(y - j) < (unsigned)VEC) {
#pragma unroll
                for (int q = 0; q < VEC; ++q)
                    if (y == j + q) f[q] += gy;
            }
            out.vec(j, f);
        }
        if (single) out.one(row.je, kept ? value(row.xe) + (row.je == y ? gy : 0.f) : 0.f);
    }
}

// ---- clipped policy loss -------------------------------------------------------------------------------------------
// rho = exp(logp - old), l = -min(rho A, clip(rho, lo, hi) A) + kl (exp(ref - logp) - (ref - logp) - 1) - ent H
// dl/dlogp = -[rho A <= clip(rho) A] rho A + kl (1 - exp(ref - logp)),  dl/dH = -ent
struct Policy {
    const float* old_logp;
    const float* adv;
    int64_t adv_rows;         // adv[r mod adv_rows]
    const float* ref_logp;    // nullable
    double lo, hi, kl, ent, inv_tau;
    Weight w;
    int unless_unit;          // nothing is done where *w.gscale is 1
    float* row_loss;          // nullable, as the next two
    float* logp;
    float* entropy;
    void* dx;                 // nullable
    int64_t ldg;
};

template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, min_waves(NV)) void policy_kernel(Rows rows, Policy a)
{
    __shared__ float sh[48];
    __shared__ float coef[3];
    if (a.unless_unit && *a.w.gscale == 1.f) return;
    const double norm = mean_norm<NT>(rows, a.w);
    const int64_t r = rows.first + dealt(blockIdx.x, rows.n);
    const typename E::Store* x = reinterpret_cast<const typename E::Store*>(rows.x) + r * rows.ld;
    Row<E, NT, NV, false, true> row(x, rows.vocab);
    const OutRow<E> out(a.dx, a.ldg, r, x);
    if (!rows.kept(r)) {
        if (threadIdx.x == 0) {
            if (a.row_loss) a.row_loss[r] = 0.f;
            if (a.logp) a.logp[r] = 0.f;
            if (a.entropy) a.entropy[r] = 0.f;
        }
        if (a.dx) fill_row<NT>(row, out, 0.f);
        return;
    }
    row.load();
    Scale sc(neg_inf(), 0.f), unused(neg_inf(), 0.f);
    const Stats all = row_stats<MOMENT>(row, (float)(LOG2E * a.inv_tau), 0.f, sc, unused, sh);
    const float s = all.s, t = all.t;
    const int64_t y64 = rows.targets[r];
    const int y = (y64 >= 0 && y64 < rows.vocab) ? (int)y64 : -1;
    if (threadIdx.x < 64) {
        const double it = a.inv_tau, log_s = log_row((double)s), u = -(double)t / (double)s * LN2, H = log_s + u;
        const double lp = y >= 0 ? sc.log_of(E::load(x + y)) - log_s : __builtin_nan("");
        const double A = (double)a.adv[r % a.adv_rows], gap = a.ref_logp ? (double)a.ref_logp[r] - lp : 0.0;
        // two exponentials, side by side in two lanes
        const double both = exp_row(threadIdx.x == 0 ? lp - (double)a.old_logp[r] : gap);
        const double rho = lane_value(both, 0), away = lane_value(both, 1);
        const double free = rho * A, held = (rho < a.lo ? a.lo : rho > a.hi ? a.hi : rho) * A;
        double loss = free <= held ? -free : -held, g = free <= held ? -free : 0.0;
        if (free != free) loss = g = free;  // a NaN stays one
        if (a.ref_logp) {
            loss += a.kl * (away - gap - 1.0);
            g += a.kl * (1.0 - away);
        }
        if (a.ent != 0.0) loss -= a.ent * H;
        if (threadIdx.x == 0) {
            if (a.row_loss) a.row_loss[r] = (float)loss;
            if (a.logp) a.logp[r] = (float)lp;
            if (a.entropy) a.entropy[r] = (float)H;
            const double w = a.w.of(r, norm) * it;
            coef[0] = (float)(w * (-g + a.ent * u) / (double)s);
            coef[1] = (float)(w * a.ent * LN2 / (double)s);
            coef[2] = (float)(w * g);
        }
    }
    if (!a.dx) return;
    __syncthreads();
    const float k0 = coef[0], k1 = coef[1], gy = coef[2];
    if (k1 == 0.f) store_row<(NV > 0)>(row, out, sc, y, gy, [&](float v) { return exp2_raw(sc.y(v)) * k0; });
    else store_row<(NV > 0)>(row, out, sc, y, gy, [&](float v) {
        const float e = sc.y(v);
        return exp2_raw(e) * fmaf(k1, clamped(e), k0);
    });
}

// ---- distillation from a teacher's list of logits ----------------------------------------------------------------
// The teacher gives k classes with logits t_k, and the log mass `tail` of all others at the same temperature; q is the
// soft-max over the k + 1 of them.  The student's p is summed the same way: p_k, and p_t over the classes not listed.
//   l = (1 - a) tau^2 [ sum q_k log(q_k / p_k) + q_t log(q_t / p_t) ] + a CE(y)
//   dl/dx_j = (1 - a) tau (p_j - q_j)            for a listed class
//           = (1 - a) tau p_j (1 - q_t / p_t)    for the others          plus a (softmax(x)_j - 1[j = y])
// p_t is the sum of the others' own exponentials relative to their own maximum, not one minus the listed ones': it keeps
// its relative precision however little is left.  The listed classes are marked in a bit map over the row (LDS) and
// taken out of the sweeps; their gradients are stored after the row's.  A class listed twice is one class of the
// student's (counted once in p) with the sum of its q.
constexpr int DISTILL_MAX_K = 256;
constexpr int DISTILL_MAX_VOCAB = 400000;  // bit map of 50 KB

struct Distill {
    const void* values;
    int value_type;
    const int32_t* indices;
    int k;
    const float* tail;   // nullable
    double inv_tau, tau, ce;
    Weight w;
    int unless_unit;
    float* row_loss;     // nullable
    void* dx;            // nullable
    int64_t ldg;
};

__device__ __forceinline__ float load_as(const void* p, int type, int64_t i)
{
    if (type == GTG_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
    if (type == GTG_DTYPE_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return (float)reinterpret_cast<const __bf16*>(p)[i];
}

template <typename E, int NT, int NV, bool BOTH>
__global__ __launch_bounds__(NT, min_waves(NV)) void distill_kernel(Rows rows, Distill a)
{
    extern __shared__ unsigned bits[];  // a bit per class, see Row::mark_place: (vocab + 2 VEC + 31) / 32
    __shared__ float sh[48];
    __shared__ int sidx[DISTILL_MAX_K];    // class, -1 where the entry takes no part
    __shared__ float st[DISTILL_MAX_K], sx[DISTILL_MAX_K], sq[DISTILL_MAX_K];
    __shared__ unsigned char own[DISTILL_MAX_K];
    __shared__ int bad, twice;
    __shared__ float coef[3];  // of exp((x - m_t) / tau), of exp(x - m_t), of the target
    __shared__ double glob[6];

    if (a.unless_unit && *a.w.gscale == 1.f) return;
    const double norm = mean_norm<NT>(rows, a.w);
    const int64_t r = rows.first + dealt(blockIdx.x, rows.n);
    const typename E::Store* x = reinterpret_cast<const typename E::Store*>(rows.x) + r * rows.ld;
    Row<E, NT, NV, true, true> row(x, rows.vocab);
    const OutRow<E> out(a.dx, a.ldg, r, x);
    if (!rows.kept(r)) {
        if (threadIdx.x == 0 && a.row_loss) a.row_loss[r] = 0.f;
        if (a.dx) fill_row<NT>(row, out, 0.f);
        return;
    }
    const int tid = threadIdx.x;
    const int64_t y64 = rows.targets[r];
    const int y = (y64 >= 0 && y64 < rows.vocab) ? (int)y64 : -1;
    // the list first: its loads are the ones that others wait for
    constexpr int KP = (DISTILL_MAX_K + NT - 1) / NT;
    int jk[KP];
#pragma unroll
    for (int i = 0; i < KP; ++i) {
        const int k = tid + i * NT;
        jk[i] = k < a.k ? a.indices[r * a.k + k] : -1;
    }
    row.load();
    for (int i = tid; i < (rows.vocab + 2 * E::VEC + 31) / 32; i += NT) bits[i] = 0;
    if (tid == 0) {
        bad = y < 0;
        twice = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KP; ++i) {
        const int k = tid + i * NT, j = jk[i];
        if (k >= a.k) continue;
        const bool in = j >= 0 && j < rows.vocab;
        if (j >= rows.vocab) bad = 1;  // (every writer writes the same value)
        sidx[k] = in ? j : -1;
        st[k] = in ? load_as(a.values, a.value_type, r * a.k + k) : neg_inf();
        sx[k] = in ? E::load(x + j) : neg_inf();
        own[k] = in;
        if (in) {
            const int at = row.mark_place(j);
            if (atomicOr(&bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1) twice = 1;
        }
    }
    __syncthreads();
    if (twice) {  // of a class listed more than once the first entry stands for all: in a fixed order, so sums repeat
        for (int k = tid; k < a.k; k += NT)
            for (int i = 0; i < k; ++i)
                if (sidx[i] == sidx[k]) own[k] = 0;
        __syncthreads();
    }
    row.mark(bits);

    // the classes outside the list: maximum, sums at both temperatures
    const float c = (float)(LOG2E * a.inv_tau), c1 = (float)LOG2E;
    Scale sc(neg_inf(), c), sc1(neg_inf(), c1);
    const Stats rest = row_stats<BOTH ? TWO : NONE>(row, c, c1, sc, sc1, sh);
    const float m_rest = sc.m, s_tau = rest.s, s_one = BOTH ? rest.t : rest.s;

    // one wave: the teacher's distribution, the student's sums over everything, the loss
    if (tid < 64) {
        const double it = a.inv_tau, its = (double)c * LN2, its1 = (double)c1 * LN2;  // the teacher's; the student's, see Scale
        const double tail = a.tail ? (double)a.tail[r] : -(double)__builtin_inff();
        float tm = neg_inf(), xm = m_rest;
        for (int k = tid; k < a.k; k += 64) {
            tm = fmaxf(tm, st[k]);
            if (own[k]) xm = fmaxf(xm, sx[k]);
        }
        tm = wave_max(tm);
        xm = wave_max(xm);
        const double M0 = fmax((double)tm * it, tail), M = M0 > -1e300 ? M0 : 0.0;  // an infinite one would leave NaN in every difference
        const float m = finite_or_zero(xm);
        double z = 0.0, s = 0.0, s1 = 0.0, cross = 0.0;
        for (int k = tid; k < a.k; k += 64) {
            const double u = (double)st[k] * it;
            const float q = exp2_raw((float)((u - M) * LOG2E));
            sq[k] = q;
            z += (double)q;
            if (q != 0.f) cross += (double)q * ((u - M) - ((double)sx[k] - (double)m) * its);
            if (own[k]) {
                s += (double)exp2_raw((sx[k] - m) * c);
                if (BOTH) s1 += (double)exp2_raw((sx[k] - m) * c1);
            }
        }
        z = wave_sum(z);
        s = wave_sum(s);
        s1 = BOTH ? wave_sum(s1) : 0.0;
        cross = wave_sum(cross);
        // exponentials and logarithms side by side in the wave's lanes; those that scale every class outside the list,
        // of (the others' reference) - (the row's maximum), in 64 bits like the rest
        const double gap = sc.log_ref(m), gap1 = BOTH ? sc1.log_ref(m) : gap;
        const double e3 = exp_row(tid == 0 ? tail - M : tid == 1 ? gap : gap1);
        const double qt0 = lane_value(e3, 0), lift = lane_value(e3, 1), lift1 = BOTH ? lane_value(e3, 2) : lift;
        z += qt0;
        s += (double)s_tau * lift;
        s1 = BOTH ? s1 + (double)s_one * lift1 : s;
        const double l4 = log_row(tid == 0 ? z : tid == 1 ? s : tid == 2 ? (double)s_tau : s1);
        const double log_z = lane_value(l4, 0), log_s = lane_value(l4, 1), log_rest = lane_value(l4, 2), log_s1 = lane_value(l4, 3);
        const bool none = z == 0.0;  // the teacher says nothing about this row
        const double qt = none ? 0.0 : qt0 / z;
        double kd = 0.0;
        const double wkd = 1.0 - a.ce;
        if (!none && wkd != 0.0) {
            // everything relative to the two maxima M and m, which may be as large as the type's lowest value
            kd = cross / z - (log_z - log_s);
            if (qt != 0.0) kd += qt * ((tail - M) - (log_rest + gap));
            kd *= wkd * a.tau * a.tau;
        }
        double ce = 0.0;
        if (a.ce != 0.0 && y >= 0) ce = a.ce * (log_s1 - ((double)E::load(x + y) - (double)m) * its1);
        if (tid == 0) {
            double loss = kd + ce;
            if (bad) loss = __builtin_nan("");
            if (a.row_loss) a.row_loss[r] = (float)loss;
            const double w = bad ? __builtin_nan("") : a.w.of(r, norm);
            const double wk = none || wkd == 0.0 ? 0.0 : w * wkd * a.tau, wc = w * a.ce;
            const double ka = wk == 0.0 ? 0.0 : wk * (lift / s - (qt != 0.0 ? qt / (double)s_tau : 0.0)), kb = wc * lift1 / s1;
            coef[0] = (float)(BOTH ? ka : ka + kb);
            coef[1] = (float)kb;
            coef[2] = (float)wc;
            glob[0] = wk / s;                   // of exp((x_k - m) / tau)
            glob[1] = none ? 0.0 : wk / z;      // of q_k
            glob[2] = wc / s1;                  // of exp(x_k - m)
            glob[3] = (double)m;
        }
    }
    if (!a.dx) return;
    __syncthreads();
    const float ka = coef[0], kb = coef[1], gy = coef[2];
    store_row<(NV > 0)>(row, out, sc, y, -gy, [&](float v) {
        const float e = exp2_raw(sc.y(v)) * ka;
        return BOTH ? fmaf(exp2_raw(sc1.y(v)), kb, e) : e;
    });
    __syncthreads();  // the listed classes' gradients go over what the row's vectors left in their places
    for (int k = tid; k < a.k; k += NT) {
        if (!own[k]) continue;
        float q = sq[k];
        if (twice)
            for (int i = k + 1; i < a.k; ++i)
                if (sidx[i] == sidx[k]) q += sq[i];
        const float d = sx[k] - (float)glob[3];
        double v = (double)exp2_raw(d * c) * glob[0] - (double)q * glob[1];
        if (a.ce != 0.0) v += (double)exp2_raw(d * c1) * glob[2];
        if (sidx[k] == y) v -= (double)gy;
        out.one(sidx[k], (float)v);
    }
}

// ---- the k largest logits of a row --------------------------------------------------------------------------------
// Exact: larger first, equal ones by ascending index (-0 equals +0, a NaN is larger than every number).  The k-th
// largest is found bit by bit on integers in the order of the values, ties by bits of the index.
__device__ __forceinline__ unsigned order_key(float x)
{
    const unsigned b = __float_as_uint(x + 0.f);
    return x != x ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// The usual way takes two sweeps.  The first finds maxima of parts of the row, one per thread (two, of halves of its vectors,
// for a k that is not small beside the threads; up to eight where one wave has the row): the k-th largest of them is a bound
// that at least k elements reach and few more do.  The second puts what reaches the bound on a list and sums the exponentials
// of everything below, relative to the bound.  The list's elements then find their rank by comparing with each other.
// Where what lies below the bound vanishes beside it, the tail is summed in two more sweeps relative to its own maximum.
// Where the list would overflow (many equal values) or a NaN is about: a row that is its lowest value but for few elements (a
// mask's rows; all equal ones) has the k largest among those and its first k elements; in any other the k-th largest is found bit
// by bit with a sweep for each, 65 in all (10 240 rows of 30 522 bf16, 50 classes not masked: 64 largest 619 us so, 4121 bit by bit).

__device__ __forceinline__ float key_value(unsigned key)  // the float of a key that is no NaN's
{
    return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// One wave: the k-th largest of its 64 N keys, to 16 bits and rounded down.  The bits above the highest one in which any two
// keys differ are common to all.
template <int N>
__device__ __forceinline__ unsigned kth_key16(const unsigned (&mk)[N], int k)
{
    unsigned all_or = 0, all_and = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        all_or |= mk[i];
        all_and &= mk[i];
    }
    const unsigned differ = (unsigned)wave_reduce((int)all_or, [](int a, int b) { return a | b; }) ^
                            (unsigned)wave_reduce((int)all_and, [](int a, int b) { return a & b; });
    const int top = differ ? 31 - __builtin_clz(differ) : -1;
    unsigned kth = top >= 31 ? 0u : (unsigned)lane_value((int)all_and, 0) & (0xffffffffu << (top + 1));
#pragma unroll 1
    for (int bit = top; bit >= 16; --bit) {
        const unsigned cand = kth | (1u << bit);
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(mk[i] >= cand));
        if (c >= k) kth = cand;
    }
    return kth & 0xffff0000u;
}
template <int N>
__device__ __forceinline__ unsigned kth_key16_of(const unsigned* keys, int k)
{
    unsigned mk[N];
#pragma unroll
    for (int i = 0; i < N; ++i) mk[i] = keys[(threadIdx.x & 63) + 64 * i];
    return kth_key16<N>(mk, k);
}

// (waves per SIMD: what the LDS below leaves room for; 512 threads on 8 vectors with 6: 153 us, with 8: 136, 10 240 x 30 522 bf16)
constexpr int top_waves(int nt, int nv) { return nt == 64 ? 3 : nt == 256 ? 6 : nv == 8 ? 8 : min_waves(nv); }
template <typename E, int NT, int NV>
__global__ __launch_bounds__(NT, top_waves(NT, NV)) void top_kernel(const void* logits, int64_t ld, int64_t first, int V, int k,
                                                                    double inv_tau, void* __restrict__ values,
                                                                    int32_t* __restrict__ indices, float* __restrict__ tail)
{
    __shared__ float shf[16];
    __shared__ int sh[16];
    // places for listed elements, and per wave for vectors put aside
    // (k = 256 lists about 350 elements, which one wave finds in 250 vectors out of 512 and in 300 out of 1024)
    constexpr int NW = NT / 64, TOP_LIST = NT == 64 ? 512 : 1024;
    constexpr int ASIDE = NT == 1024 ? 64 : NT == 512 ? 96 : NT == 256 ? 160 : NV == 16 ? 384 : NV == 8 ? 320 : NV == 4 ? 256 : 64;
    static_assert(NT > 64 || NV > 0, "a streamed row has more than one wave");
    constexpr int SPARE = NT == 64 ? TOP_LIST : 2 * NT;
    __shared__ int fill;
    __shared__ u32x4 aside_vec[NW * ASIDE];
    __shared__ int aside_j[NW * ASIDE];
    __shared__ unsigned bound_key, kth_key;
    __shared__ int kth_idx;
    __shared__ unsigned long long list[TOP_LIST];  // key, then the complement of the index: larger is nearer the front
    __shared__ int ranks[TOP_LIST];
    __shared__ unsigned keys[SPARE];               // maxima; then the floats that are listed but not among the k, in order
    const int64_t r = first + blockIdx.x;
    const int tid = threadIdx.x;
    const typename E::Store* x = reinterpret_cast<const typename E::Store*>(logits) + r * ld;
    Row<E, NT, NV> row(x, V);
    row.load();
    const float c = (float)(LOG2E * inv_tau);

    if (tid == 0) fill = 0;
    for (int i = tid; i < TOP_LIST; i += NT) ranks[i] = 0;
    if constexpr (NT == 64) {
        // one wave: up to eight maxima a lane, of the halves of every vector or every few, and no LDS
        constexpr int PARTS = NV < 4 ? NV : 4, EACH = NV / PARTS;
        unsigned mk[2 * PARTS];
        float single = row.xe;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            typename E::Maxima part;
#pragma unroll
            for (int e = 0; e < EACH; ++e) part.take(row.v[i * EACH + e]);
            mk[2 * i] = order_key(fmaxf(part.lo(), single));
            mk[2 * i + 1] = order_key(part.hi());
            single = neg_inf();
        }
        // (a row of so few vectors that it has fewer maxima than k is listed whole)
        const unsigned key = k > 128 * PARTS ? 0u : kth_key16<2 * PARTS>(mk, k);
        if (tid == 0) bound_key = key;
    } else {
        const bool halves = 4 * k > NT;
        typename E::Maxima parts;
        row.template each<true>([&](int, const u32x4& v) { parts.take(v); });
        const float lo = fmaxf(parts.lo(), row.xe), hi = parts.hi();
        keys[tid] = order_key(halves ? lo : fmaxf(lo, hi));
        if (halves) keys[NT + tid] = order_key(hi);
        __syncthreads();
        if (tid < 64) {
            const unsigned key = halves ? kth_key16_of<2 * NT / 64>(keys, k) : kth_key16_of<NT / 64>(keys, k);
            if (tid == 0) bound_key = key;
        }
    }
    __syncthreads();
    const float bound = bound_key > order_key(neg_inf()) ? key_value(bound_key) : neg_inf();
    auto put = [&](int at, int j, float f) {
        if (at < TOP_LIST) list[at] = (unsigned long long)order_key(f) << 32 | (unsigned)~j;
    };
    const Scale sc(bound, c);
    float s = 0.f;
    const int wave = tid >> 6, lane = tid & 63;
    u32x4* vec_aside = &aside_vec[wave * ASIDE];
    int* j_aside = &aside_j[wave * ASIDE];
    int na = 0;  // the same in every lane
    row.template each<false>([&](int j, u32x4& v) {
        const bool hit = !(vec_max<E>(neg_inf(), v) < bound);
        const unsigned long long hits = __ballot(hit);
        if (hits) {
            // (two of three wave-wide vectors hold one of 64 elements out of 30 522: here they are only put aside)
            const int at = na + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0));
            if (hit) {
                if (at < ASIDE) {
                    vec_aside[at] = v;
                    j_aside[at] = j;
                }
                v = u32x4{E::NEG2, E::NEG2, E::NEG2, E::NEG2};
            }
            na += __popcll(hits);
        }
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) s += exp2_raw(sc.y(E::get(v, q)));  // (a NaN that the maximum passed over shows in the sum)
    });
    if (row.je >= 0) {
        if (row.xe < bound) s += exp2_raw(sc.y(row.xe));
        else put(atomicAdd(&fill, 1), row.je, row.xe);
    }
    // (lanes past the row's end have missed the last vectors' count; the largest is the wave's)
    na = wave_reduce(na, [](int a, int b) { return max(a, b); });
    if (na > ASIDE && lane == 0) atomicAdd(&fill, TOP_LIST + 1);
    for (int i = lane; i < min(na, ASIDE); i += 64) {
        u32x4 v = vec_aside[i];
        const int j = j_aside[i];
        unsigned found = 0;
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) found |= !(E::get(v, q) < bound) ? 1u << q : 0u;
        int at = atomicAdd(&fill, __popc(found));
        while (found) {
            const int q = __ffs(found) - 1;
            found &= found - 1;
            put(at++, j + q, E::take(v, q));
        }
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) s += exp2_raw(sc.y(E::get(v, q)));
    }
    s = block_sum<NT, false>(s, shf);
    __syncthreads();
    int n = fill;
    const bool exact = n > TOP_LIST || s != s;
    Row<E, NT, 0> again(x, V);  // the rare ways read the row anew: their loops need no registers of the usual one's
    if (exact) {
        again.load();
        auto count = [&](auto pred) {
            int cnt = again.je >= 0 && pred(again.je, again.xe) ? 1 : 0;
            again.template each<false>([&](int j, const u32x4& v) {
#pragma unroll
                for (int q = 0; q < E::VEC; ++q) cnt += pred(j + q, E::get(v, q)) ? 1 : 0;
            });
            return block_sum<NT, true>(cnt, sh);
        };
        __syncthreads();
        if (tid == 0) fill = 0;
        __syncthreads();
        // Rows of which most is one lowest value (a mask's): what is above it and the first k elements hold the k largest.
        float low = again.je >= 0 ? again.xe : __builtin_inff();
        again.template each<false>([&](int, const u32x4& v) {
#pragma unroll
            for (int q = 0; q < E::VEC; ++q) low = fminf(low, E::get(v, q));
        });
        low = block_reduce<NT, true>(low, shf, [](float a, float b) { return fminf(a, b); });
        auto above = [&](int j, float v) { return j < k || !(v <= low); };
        const int few = count(above);
        unsigned kth = 0;  // the largest key that at least k elements reach
        int last = 0;      // the last one of that key, by index, that is taken
        auto take = [&](int j, float f) {
            const unsigned key = order_key(f);
            if (few <= TOP_LIST ? above(j, f) : key > kth || (key == kth && j <= last)) put(atomicAdd(&fill, 1), j, f);
        };
        if (few > TOP_LIST) {
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned cand = kth | (1u << bit);
                if (count([&](int, float v) { return order_key(v) >= cand; }) >= k) kth = cand;
            }
            const int need = k - count([&](int, float v) { return order_key(v) > kth; });
            for (int bit = 30; bit >= 0; --bit) {
                const int cand = last + (1 << bit);
                if (cand < V && count([&](int j, float v) { return j < cand && order_key(v) == kth; }) < need) last = cand;
            }
        }
        if (again.je >= 0) take(again.je, again.xe);
        again.template each<false>([&](int j, const u32x4& v) {
#pragma unroll
            for (int q = 0; q < E::VEC; ++q) take(j + q, E::get(v, q));
        });
        __syncthreads();
        n = fill;
    }
    // ranks: a wave compares 64 of the list's elements with its share of the whole list
    {
        const int w = wave;
        const int share = (n + NW - 1) / NW, o0 = w * share, o1 = min(n, o0 + share);
        for (int i0 = 0; i0 < n; i0 += 64) {
            const unsigned long long mine = list[min(i0 + lane, n - 1)];
            int rank = 0;
#pragma unroll 4
            for (int o = o0; o < o1; ++o) rank += list[o] > mine ? 1 : 0;
            if (i0 + lane < n && rank) atomicAdd(&ranks[i0 + lane], rank);
        }
    }
    __syncthreads();
    float* rest = reinterpret_cast<float*>(keys);
    const bool spare = n - k <= SPARE;  // (the maxima's places hold what is listed beyond k; more than they are goes the long way)
    for (int i = tid; i < n; i += NT) {
        const unsigned key = (unsigned)(list[i] >> 32);
        const int j = (int)~(unsigned)list[i], rank = ranks[i];
        if (rank < k) {
            indices[r * k + rank] = j;
            reinterpret_cast<typename E::Store*>(values)[r * k + rank] = x[j];
            if (rank == k - 1) {
                kth_key = key;
                kth_idx = j;
            }
        } else if (spare) {
            rest[rank - k] = key_value(key);
        }
    }
    __syncthreads();
    if (!exact && spare && !sc.flat && (s > 1e-30f || n == V)) {
        // what lies below the bound, and the list's own remainder relative to its first
        if (tid < 64) {
            const float first = n > k ? rest[0] : neg_inf();
            float t = 0.f;
            for (int i = tid; i < n - k; i += 64) t += first == neg_inf() ? 0.f : exp2_raw((rest[i] - first) * c);
            t = wave_sum(t);
            const double low = s > 0.f ? (double)sc.mu * LN2 : (double)neg_inf(), high = (double)first * inv_tau;
            const double top = fmax(low, high);
            const double e = exp_row(tid == 0 ? low - top : high - top);
            const double sum = (s > 0.f ? (double)s * lane_value(e, 0) : 0.0) + (t > 0.f ? (double)t * lane_value(e, 1) : 0.0);
            // (an infinite first, and a NaN, which is before every number, are the sum themselves)
            if (tid == 0) tail[r] = first == __builtin_inff() || first != first ? first : sum > 0.0 ? (float)(top + log_row(sum)) : neg_inf();
        }
        return;
    }
    const unsigned kth = kth_key;
    const int last = kth_idx;
    auto chosen = [&](int j, float f) {
        const unsigned key = order_key(f);
        return key > kth || (key == kth && j <= last);
    };
    again.load();
    float mx = again.je >= 0 && !chosen(again.je, again.xe) ? again.xe : neg_inf();
    again.template each<false>([&](int j, const u32x4& v) {
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) {
            const float f = E::get(v, q);
            if (!chosen(j + q, f)) mx = fmaxf(mx, f);
        }
    });
    const float m_rest = block_max<NT, true>(mx, shf), m = finite_or_zero(m_rest);
    s = again.je >= 0 && !chosen(again.je, again.xe) ? exp2_raw((again.xe - m) * c) : 0.f;
    again.template each<false>([&](int j, const u32x4& v) {
#pragma unroll
        for (int q = 0; q < E::VEC; ++q) {
            const float f = E::get(v, q);
            if (!chosen(j + q, f)) s += exp2_raw((f - m) * c);
        }
    });
    s = block_sum<NT, true>(s, shf);
    if (tid == 0) tail[r] = m_rest == __builtin_inff() && s != s ? m_rest : (float)(log_row((double)s) + (double)m * inv_tau);
}

// ---- preference loss over pairs of sequences -------------------------------------------------------------------------
// seq_b = sum over time of logp, margin = beta ((seq_c - ref_c) - (seq_r - ref_r)),
// l = -(1 - e) log sigma(margin) - e log sigma(-margin);  the first `pairs` sequences are the chosen ones, sequence
// b + pairs is the one rejected for b.  One block: sums in 64 bits and in a fixed order.
struct Prefer {
    const double* logp;   // (rows)
    double* seq;          // (2 pairs) scratch
    int64_t T, pairs;
    int batch_first;
    const float* ref;     // (2 pairs)
    double beta, eps;
    int mean;
    float* seq_logp;      // (2 pairs)
    float* coef;          // (2 pairs): dl / dseq
    float* pair_loss;     // (pairs)
    float* loss;          // nullable
};

__global__ __launch_bounds__(1024) void prefer_kernel(Prefer a)
{
    __shared__ double part[1024];
    const int64_t S = 2 * a.pairs;
    // G threads per sequence, neighbours on neighbouring sequences
    const int width = (int)(S < 1024 ? S : 1024), G = 1024 / width;
    const int lane = threadIdx.x % width, g = threadIdx.x / width;
    for (int64_t b0 = 0; b0 < S; b0 += width) {
        const int64_t b = b0 + lane;
        double s = 0.0;
        if (b < S && g < G)
#pragma unroll 8
            for (int64_t t = g; t < a.T; t += G) s += a.logp[a.batch_first ? b * a.T + t : t * S + b];
        part[threadIdx.x] = s;
        __syncthreads();
        if (g == 0 && b < S) {
            for (int i = 1; i < G; ++i) s += part[i * width + lane];
            a.seq[b] = s;
            a.seq_logp[b] = (float)s;
        }
        __syncthreads();
    }
    double total = 0.0;
    for (int64_t p = threadIdx.x; p < a.pairs; p += 1024) {
        const double mg = a.beta * ((a.seq[p] - (double)a.ref[p]) - (a.seq[p + a.pairs] - (double)a.ref[p + a.pairs]));
        const double both = log1p(exp(-fabs(mg)));
        double l = (1.0 - a.eps) * (both + (mg < 0.0 ? -mg : 0.0));
        if (a.eps != 0.0) l += a.eps * (both + (mg > 0.0 ? mg : 0.0));
        const double dm = (a.eps - 1.0 / (1.0 + exp(mg))) * a.beta / (a.mean ? (double)a.pairs : 1.0);
        a.pair_loss[p] = (float)l;
        a.coef[p] = (float)dm;
        a.coef[p + a.pairs] = (float)-dm;
        total += l;
    }
    if (!a.loss) return;
    part[threadIdx.x] = total;
    __syncthreads();
    if (threadIdx.x < 64) {
        total = 0.0;
        for (int i = 0; i < 16; ++i) total += part[threadIdx.x + 64 * i];
        total = wave_sum(total);
        if (threadIdx.x == 0) *a.loss = (float)(a.mean ? total / (double)a.pairs : total);
    }
}

// A block per row, by the row's 16-byte vectors: as many threads as they keep busy, and the row in registers up to 16 vectors
// (64 registers) a thread and 1024 threads -- 128 K elements of 16 bits, 64 K of 32.  One wave for up to 512 vectors: a block
// of four has a quarter of the lanes idle there and passes sums through LDS (40 000 rows of 2500 bf16: log-probability 82 us with
// 256 threads, 45 with 64; policy loss 154 and 92; the k largest 200 and 140).  From 513 to 1024 two waves, but one for the
// k largest, which has no LDS to wait for then: 40 000 rows of 2500 fp32 169 and 142 us; the distillation 187 with two, 198 with one.
// One wave is slow to rank a long list, though: above k = 64 the rows of 257 to 1024 vectors take four (k = 256, 20 000 rows of
// 4000 fp32: 635 us with one, 406 with four; k = 64 141 and 130, and of 2000 fp32 207 and 238).  Longer rows than registers hold
// are read again in every sweep, by 1024 threads (1500 rows of 150 000 bf16, policy loss: 256 threads 284 us, 512 247, 1024 215;
// 16 rows: 63, 37, 32).  Registers where they hold the row all the same: distillation of 1533 rows of 131 072 bf16 170 us, streamed 185.
template <typename E_, int NT_, int NV_>
struct Shape {
    typedef E_ E;
    static constexpr int NT = NT_, NV = NV_;
};
template <typename E, int MID, typename F>
void by_vectors(int64_t n, F launch)
{
    if (n <= 64) launch(Shape<E, 64, 1>());
    else if (n <= 256) launch(Shape<E, 64, 4>());
    else if (MID < 256 && n <= 512) launch(Shape<E, 64, MID < 256 ? 8 : 4>());
    else if (n <= 1024) launch(Shape<E, MID, 1024 / MID>());
    else if (n <= 2048) launch(Shape<E, 256, 8>());
    else if (n <= 4096) launch(Shape<E, 512, 8>());
    else if (n <= 8192) launch(Shape<E, 512, 16>());
    else if (n <= 16384) launch(Shape<E, 1024, 16>());
    else launch(Shape<E, 1024, 0>());
}
template <int MID = 128, typename F>
void by_size(int dtype, int vocab, F launch)
{
    if (dtype == GTG_DTYPE_F32) by_vectors<F32, MID>(((int64_t)vocab + 3) / 4, launch);
    else if (dtype == GTG_DTYPE_F16) by_vectors<F16, MID>(((int64_t)vocab + 7) / 8, launch);
    else by_vectors<BF16, MID>(((int64_t)vocab + 7) / 8, launch);
}

Rows as_rows(const TokenRows& t, int64_t first = 0, unsigned n = 0)
{
    return Rows{t.logits, t.ld, t.vocab, t.targets, t.padidx, t.mask, first, n};
}

// A launch holds fewer than 2^32 threads: f(first row, rows) for every slice of 2 M rows.
template <typename F>
void by_slices(int64_t R, F f)
{
    constexpr int64_t SLICE = 1 << 21;
    for (int64_t r = 0; r < R; r += SLICE) f(r, (unsigned)(R - r < SLICE ? R - r : SLICE));
}

}  // namespace

int top_logits(const void* logits, int dtype, int64_t R, int V, int64_t ld, int k, double temperature, void* values,
               int32_t* indices, float* tail, hipStream_t s)
{
    ProfScope prof(s, "top_logits", R, V, k);
    const double it = 1.0 / temperature;
    auto launch = [&](auto shape) {
        typedef decltype(shape) P;
        by_slices(R, [&](int64_t r0, unsigned n) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(top_kernel<typename P::E, P::NT, P::NV>), dim3(n), dim3(P::NT), 0, s, logits, ld, r0,
                               V, k, it, values, indices, tail);
        });
    };
    if (k > 64) by_size<256>(dtype, V, launch);
    else by_size<64>(dtype, V, launch);
    return check_launch("top_kernel");
}

int token_logprob_fwd(const TokenRows& t, double temperature, float* logp, float* entropy, float* stats, double* logp64,
                      hipStream_t s)
{
    ProfScope prof(s, "token_logprob_fwd", t.rows, t.vocab, 0);
    const LogprobOut out{logp, entropy, reinterpret_cast<float4*>(stats), logp64};
    const double it = 1.0 / temperature;
    by_size(t.dtype, t.vocab, [&](auto shape) {
        typedef decltype(shape) P;
        by_slices(t.rows, [&](int64_t r0, unsigned n) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(logprob_kernel<typename P::E, P::NT, P::NV>), dim3(n), dim3(P::NT), 0, s,
                               as_rows(t, r0, n), it, out);
        });
    });
    return check_launch("logprob_kernel");
}

int token_logprob_bwd(const TokenRows& t, double temperature, const float* stats, const float* g_logp, const float* g_entropy,
                      const float* gscale, const float* gloss, int64_t group, int64_t pairs, void* dx, int64_t ldg,
                      hipStream_t s)
{
    ProfScope prof(s, "token_logprob_bwd", t.rows, t.vocab, 0);
    const RowGrad g{reinterpret_cast<const float4*>(stats), g_logp, g_entropy, gscale, gloss, group, pairs, 1.0 / temperature, dx, ldg};
    const int64_t vectors = (int64_t)t.vocab / (t.dtype == GTG_DTYPE_F32 ? 4 : 8);
    const int64_t per_row = vectors / (BWD_NT * BWD_VEC) + 1, pieces = t.rows * per_row;
    if (pieces > 0x7fffffffll) return set_error(GTG_ERR_UNSUPPORTED, "token_logprob_bwd: too many logits for one call");
    const unsigned blocks = (unsigned)(pieces < (1 << 22) ? pieces : 1 << 22);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(BWD_NT), 0, s, as_rows(t), g, (unsigned)pieces, (unsigned)per_row);
    };
    if (t.dtype == GTG_DTYPE_F32) launch(logprob_bwd_kernel<F32>);
    else if (t.dtype == GTG_DTYPE_F16) launch(logprob_bwd_kernel<F16>);
    else launch(logprob_bwd_kernel<BF16>);
    return check_launch("logprob_bwd_kernel");
}

bool counts_in_rows(int64_t R) { return R <= COUNT_IN_ROWS; }

int count_rows(const TokenRows& t, double* norm, hipStream_t s)
{
    hipLaunchKernelGGL(count_kernel, dim3(1), dim3(1024), 0, s, as_rows(t), t.rows, norm);
    return check_launch("count_kernel");
}

int total_loss(const float* row_loss, int64_t R, const double* norm, float* loss, hipStream_t s)
{
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, s, row_loss, R, norm, loss);
    return check_launch("total_kernel");
}

int policy_rows(const TokenRows& t, const PolicyRows& p, const float* gloss, const float* gscale, double* norm, bool count,
                bool unless_unit, float* row_loss, float* logp, float* entropy, void* dx, int64_t ldg, hipStream_t s)
{
    ProfScope prof(s, "policy_rows", t.rows, t.vocab, dx != nullptr);
    const Policy a{p.old_logp, p.advantages, p.adv_rows, p.ref_logp, 1.0 - p.clip_low, 1.0 + p.clip_high, p.kl_coef, p.entropy_coef,
                   1.0 / p.temperature, Weight{gloss, gscale, norm, count ? t.rows : 0}, unless_unit ? 1 : 0, row_loss, logp, entropy, dx, ldg};
    by_size(t.dtype, t.vocab, [&](auto shape) {
        typedef decltype(shape) P;
        by_slices(t.rows, [&](int64_t r0, unsigned n) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(policy_kernel<typename P::E, P::NT, P::NV>), dim3(n), dim3(P::NT), 0, s,
                               as_rows(t, r0, n), a);
        });
    });
    return check_launch("policy_kernel");
}

int distill_max_vocab() { return DISTILL_MAX_VOCAB; }

int distill_rows(const TokenRows& t, const DistillRows& d, const float* gloss, const float* gscale, double* norm, bool count,
                 bool unless_unit, float* row_loss, void* dx, int64_t ldg, hipStream_t s)
{
    ProfScope prof(s, "distill_rows", t.rows, t.vocab, dx != nullptr);
    const Distill a{d.values, d.value_dtype, d.indices, d.k, d.tail, 1.0 / d.temperature, d.temperature, d.ce_weight,
                    Weight{gloss, gscale, norm, count ? t.rows : 0}, unless_unit ? 1 : 0, row_loss, dx, ldg};
    const size_t lds = (size_t)((t.vocab + 16 + 31) / 32) * 4;
    auto launch = [&](auto both) {
        by_size(t.dtype, t.vocab, [&](auto shape) {
            typedef decltype(shape) P;
            by_slices(t.rows, [&](int64_t r0, unsigned n) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(distill_kernel<typename P::E, P::NT, P::NV, decltype(both)::value>), dim3(n),
                                   dim3(P::NT), lds, s, as_rows(t, r0, n), a);
            });
        });
    };
    if (d.ce_weight != 0.0 && d.temperature != 1.0) launch(std::true_type());
    else launch(std::false_type());
    return check_launch("distill_kernel");
}

int prefer_pairs(const double* logp, double* seq, int64_t T, int64_t pairs, bool batch_first, const float* ref, double beta,
                 double label_smoothing, bool mean, float* seq_logp, float* coef, float* pair_loss, float* loss, hipStream_t s)
{
    const Prefer a{logp, seq, T, pairs, batch_first ? 1 : 0, ref, beta, label_smoothing, mean ? 1 : 0, seq_logp, coef, pair_loss, loss};
    hipLaunchKernelGGL(prefer_kernel, dim3(1), dim3(1024), 0, s, a);
    return check_launch("prefer_kernel");
}

}  // namespace gtg
