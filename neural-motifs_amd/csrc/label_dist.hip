// label_dist.hip -- operators on rows of class logits: a teacher's top logits, distillation from them (forward and gradient) and
// drawing labels with temperature, top-k, top-p and min-p.  Definitions: include/motifs_hip.h, "label distributions".
//
// The order of a row's classes is ONE order everywhere: descending logit, ties to the lowest class, NaN before everything.  It is
// carried as the integer distance D = key(row maximum) - key(x), key = the order-preserving 32-bit image of a float, so that
// infinities, NaN and the type's lowest value need no cases of their own; (D << 32 | class), ascending, is the order.
//
// Times below: one MI355X, kernel alone.  A copy of 262 MB runs at 5.4 TB/s there (read and write), one of 2 GiB at 4.9: a stream of rows is
// measured against 5 TB/s.
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "label_cut.h"

namespace mh {
namespace ld {

typedef unsigned long long u64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct bf16 {
    uint16_t v;
};
struct f16 {
    uint16_t v;
};

// ---- rows -------------------------------------------------------------------------------------------------------------------
// 16 bytes of a row at an address that is aligned to its elements only: odd class counts and column offsets are ordinary
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    static constexpr int N = 4;
    typedef u32x4 raw __attribute__((aligned(4)));
    static __device__ __forceinline__ void expand(const u32x4 &r, float *x)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(r[j]);
    }
    static __device__ __forceinline__ u32x4 pack(const float *x)
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __float_as_uint(x[j]);
        return r;
    }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ float to(float x) { return x; }
};
__device__ __forceinline__ uint16_t f16_bits(float x) { return __half_as_ushort(__float2half_rn(x)); }
__device__ __forceinline__ float f16_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t bf16_pair(float x, float y)        // round to nearest even, NaN kept: one instruction here
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), bf16x2));
}
template <>
struct Pack<bf16> {
    static constexpr int N = 8;
    typedef u32x4 raw __attribute__((aligned(2)));
    static __device__ __forceinline__ void expand(const u32x4 &r, float *x)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(r[j] << 16);
            x[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float *x)
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = bf16_pair(x[2 * j], x[2 * j + 1]);
        return r;
    }
    static __device__ __forceinline__ float one(const bf16 *p) { return __uint_as_float((uint32_t)p->v << 16); }
    static __device__ __forceinline__ bf16 to(float x) { return bf16{(uint16_t)bf16_pair(x, x)}; }
};
template <>
struct Pack<f16> {
    static constexpr int N = 8;
    typedef u32x4 raw __attribute__((aligned(2)));
    static __device__ __forceinline__ void expand(const u32x4 &r, float *x)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = f16_float((uint16_t)(r[j] & 0xffffu));
            x[2 * j + 1] = f16_float((uint16_t)(r[j] >> 16));
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float *x)
    {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = (uint32_t)f16_bits(x[2 * j]) | ((uint32_t)f16_bits(x[2 * j + 1]) << 16);
        return r;
    }
    static __device__ __forceinline__ float one(const f16 *p) { return f16_float(p->v); }
    static __device__ __forceinline__ f16 to(float x) { return f16{f16_bits(x)}; }
};

// class j of a vector, j known at run time only
template <typename T>
__device__ __forceinline__ float pick(const u32x4 &v, int j)
{
    constexpr int PER = Pack<T>::N / 4;
    const int w = j / PER;
    const uint32_t lo = w & 1 ? v[1] : v[0], hi = w & 1 ? v[3] : v[2], word = w & 2 ? hi : lo;
    float x[Pack<T>::N];
    Pack<T>::expand(u32x4{word, 0, 0, 0}, x);
    return PER == 2 && (j & 1) ? x[PER - 1] : x[0];
}
template <typename T>
__device__ __forceinline__ u32x4 load_vector(const T *__restrict__ row, int base)
{
    return *reinterpret_cast<const typename Pack<T>::raw *>(row + base);
}
// the row's last classes, fewer than a vector, with -inf behind them
template <typename T>
__device__ __forceinline__ u32x4 load_tail(const T *__restrict__ row, int n, int base)
{
    constexpr int N = Pack<T>::N;
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = n - base > j ? Pack<T>::one(row + base + j) : -__builtin_inff();
    return Pack<T>::pack(x);
}
template <typename T>
__device__ __forceinline__ u32x4 load_any(const T *__restrict__ row, int n, int base)
{
    return n - base >= Pack<T>::N ? load_vector(row, base) : load_tail(row, n, base);
}
// batch(raw[AHEAD], vector of raw[0], how many of them count) for the vectors of a row, NT threads: vector i + j NT stands at raw[j].  All loads of a
// batch are made before the first is used, in the last batch too: what lies behind the last whole vector reads that one again (a load that asks
// for the row's end first waits for the one before it).  The classes behind the last whole vector come as a batch of one.
template <typename T, int NT, int AHEAD, typename F>
__device__ __forceinline__ void stream_batches(const T *__restrict__ row, int n, F batch)
{
    constexpr int N = Pack<T>::N;
    const int whole = n / N;
    u32x4 v[AHEAD];
    for (int i = threadIdx.x; i < whole; i += AHEAD * NT) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) v[j] = load_vector(row, min(i + j * NT, whole - 1) * N);
        batch(v, i, min(AHEAD, (whole - i + NT - 1) / NT));
    }
    if (n % N != 0 && (int)threadIdx.x == whole % NT) {
        v[0] = load_tail(row, n, whole * N);
        batch(v, whole, 1);
    }
}
// f(raw, vector) for every vector
template <typename T, int NT, int AHEAD, typename F>
__device__ __forceinline__ void stream_row(const T *__restrict__ row, int n, F f)
{
    stream_batches<T, NT, AHEAD>(row, n, [&](const u32x4 (&v)[AHEAD], int i, int count) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (j < count) f(v[j], i + j * NT);
    });
}

// the largest of N values, NaN if there is one
template <int N>
__device__ __forceinline__ float largest(const float *x)
{
    float m = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = __builtin_elementwise_maximum(m, x[j]);
    return m;
}

// One workgroup's row.  each(f): f(x[N], base) for every vector of N = 16 bytes of classes, in any order; what lies behind the end is -inf.
// HELD: the row is read from memory once, into `lds`, and every pass over it reads it there.  Else every pass reads it from memory again (from
// the caches, where it is recent).
template <typename T, int NT, bool HELD>
struct Row {
    typedef Pack<T> pack;
    static constexpr int N = Pack<T>::N;
    const T *row;
    int n;
    u32x4 *lds;
    __device__ __forceinline__ Row(const T *__restrict__ row_, int n_, u32x4 *lds_) : row(row_), n(n_), lds(lds_) {}
    // the threads' own maxima (NaN where there is one), and, HELD, the copy (whole after the next barrier)
    __device__ __forceinline__ float first_pass() const
    {
        float m = -__builtin_inff();
        stream_row<T, NT, 8>(row, n, [&](const u32x4 &v, int i) {
            float x[N];
            Pack<T>::expand(v, x);
            m = __builtin_elementwise_maximum(m, largest<N>(x));
            if (HELD) lds[i] = v;
        });
        return m;
    }
    template <int AHEAD, typename F>
    __device__ __forceinline__ void raw(F f) const          // f(raw, vector)
    {
        if (HELD) {
            const int nv = (n + N - 1) / N;
            for (int i = threadIdx.x; i < nv; i += NT) f(lds[i], i);
        } else
            stream_row<T, NT, AHEAD>(row, n, f);
    }
    template <int AHEAD = 8, typename F>
    __device__ __forceinline__ void each(F f) const
    {
        raw<AHEAD>([&](const u32x4 &v, int i) {
            float x[N];
            Pack<T>::expand(v, x);
            f(x, i * N);          // (x: float[N])
        });
    }
};
// f(x, class) for every class; a word at a time, so that f, large in the passes that are seldom made, stands in the code once or twice
template <typename R, typename F>
__device__ __forceinline__ void each_class(const R &r, F f)
{
    constexpr int PER = R::N / 4;
    r.template raw<1>([&](u32x4 v, int i) {
#pragma unroll 1
        for (int w = 0; w < 4; ++w) {
            float x[R::N];
            R::pack::expand(v, x);
            const int at = i * R::N + w * PER;
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (j < r.n - at) f(x[j], at + j);
            v = u32x4{v[1], v[2], v[3], v[0]};
        }
    });
}

// ---- order ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order_key(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.0f);            // -0 becomes +0: the two are one value
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k)
{
    if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu, kKeyNan = 0xffffffffu;

// distances in bins of 1/64 octave: fine next to the maximum, where the first k of a row end; exactly invertible
constexpr int kBins = 2048;
__device__ __forceinline__ int octave_bin(uint32_t D)
{
    if (D < 128) return (int)D;
    const int s = 25 - __clz((int)D);
    return (s << 6) + (int)(D >> s);
}
__device__ __forceinline__ void octave_range(int b, uint32_t &lo, uint32_t &hi)
{
    if (b < 128) {
        lo = hi = (uint32_t)b;
        return;
    }
    const int s = (b >> 6) - 1;
    lo = (uint32_t)((b & 63) + 64) << s;
    hi = lo + ((1u << s) - 1);
}

// ---- block helpers ----------------------------------------------------------------------------------------------------------
template <typename V, typename F>
__device__ __forceinline__ V wave_all(V v, F f)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o));
    return v;
}
template <int NT, typename V, typename F>
__device__ V block_all(V v, F f, V *red)           // red [NT / 64] in LDS; every thread gets the result
{
    v = wave_all(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    V r = red[0];
    for (int w = 1; w < NT / 64; ++w) r = f(r, red[w]);
    return r;
}
// exclusive sum over the block in thread order; total = the whole
template <int NT, typename V>
__device__ V block_scan(V v, V &total, V *red)
{
    const int lane = threadIdx.x & 63;
    V inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V up = __shfl_up(inc, o);
        if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 63) red[threadIdx.x >> 6] = inc;
    __syncthreads();
    V before = 0, all = 0;
    for (int w = 0; w < NT / 64; ++w) {
        if (w == (int)(threadIdx.x >> 6)) before = all;
        all += red[w];
    }
    total = all;
    return before + inc - v;
}
// the bin at which a running sum over h[0 .. kBins) reaches `need`; before = the sum in front of it.  False: it never does.
template <int NT, typename V>
__device__ bool find_bin(const V *h, V need, int &bin, V &before, V *red, u64 *answer)
{
    constexpr int PER = kBins / NT;
    V mine[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += mine[i] = h[threadIdx.x * PER + i];
    V total;
    V at = block_scan<NT, V>(sum, total, red);
    if (total < need) return false;
    if (at < need && at + sum >= need) {
        int i = 0;
        while (at + mine[i] < need) at += mine[i++];
        answer[0] = (u64)(threadIdx.x * PER + i);
        answer[1] = (u64)at;
    }
    __syncthreads();
    bin = (int)answer[0];
    before = (V)answer[1];
    return true;
}
// list [0 .. n) in LDS, ascending, all different.  Short lists by counting for each entry those before it (one barrier), longer ones by
// a bitonic network.
template <int NT>
__device__ void sort_list(u64 *list, int n)
{
    if (n <= NT && n <= 256) {
        // (eight entries a step: one at a time would wait for LDS each time)
        const u64 mine = (int)threadIdx.x < n ? list[threadIdx.x] : 0;
        __syncthreads();
        if (threadIdx.x < 8) list[n + (int)threadIdx.x] = ~0ull;
        __syncthreads();
        int rank = 0;
        if ((int)threadIdx.x < n)
            for (int i = 0; i < n; i += 8) {
                u64 x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = list[i + j];
#pragma unroll
                for (int j = 0; j < 8; ++j) rank += x[j] < mine;
            }
        __syncthreads();
        if ((int)threadIdx.x < n) list[rank] = mine;
        __syncthreads();
        return;
    }
    int cap = 2;
    while (cap < n) cap <<= 1;
    for (int i = n + (int)threadIdx.x; i < cap; i += NT) list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= cap; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int t = threadIdx.x; t < cap / 2; t += NT) {
                const int a = ((t & ~(j - 1)) << 1) | (t & (j - 1)), b = a | j;
                const u64 x = list[a], y = list[b];
                if ((x > y) == ((a & k) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
            __syncthreads();
        }
}

// ---- selection --------------------------------------------------------------------------------------------------------------
constexpr int kList = 2048;          // candidates that are sorted
constexpr int kMaxTop = 1024;        // longest head of a row that is kept as a sorted list (k of the top logits, short top-k)

struct Shared {                      // one workgroup's LDS
    union {                          // (never in use at once)
        u64 list[kList];
        uint32_t count[kBins];
    };
    u64 red64[16];
    uint32_t red32[16];
    u64 answer[2];
    int n;
};
struct SharedMass : Shared {
    u64 mass[kBins];
    uint32_t classes[kBins];
    int n2;
};

// The `want`-th class (from 0) among those with distance D, in class order; runs to the first hit only.
template <typename T, int NT>
__device__ int nth_tie(const T *row, int n, uint32_t kmax, uint32_t D, uint32_t want, Shared &s)
{
    uint32_t seen = 0;
    for (int base = 0; base < n; base += NT) {
        const int i = base + (int)threadIdx.x;
        const uint32_t hit = i < n && kmax - order_key(Pack<T>::one(row + i)) == D;
        uint32_t total;
        const uint32_t at = block_scan<NT, uint32_t>(hit, total, s.red32);
        if (seen + total > want) {
            if (hit && seen + at == want) s.answer[0] = (u64)i;
            __syncthreads();
            return (int)s.answer[0];
        }
        seen += total;
        if (base > n - NT) break;
    }
    return -1;
}

__device__ __forceinline__ void push(Shared &s, uint32_t D, int i)
{
    const int at = atomicAdd(&s.n, 1);
    if (at < kList) s.list[at] = (u64)D << 32 | (uint32_t)i;
}

// The first k classes of the order (k <= min(n, kMaxTop)) as a sorted list in s.list, for any row: by histograms of the distances, narrowed
// until what reaches the k-th class fits the list.  Returns the list's length.
template <typename T, int NT, typename R>
__device__ __noinline__ int top_list(R r, const T *row, int n, uint32_t kmax, int k, Shared *shared)
{
    Shared &s = *shared;
    uint32_t lo = 0, hi = 0xffffffffu, above = 0, inside = (uint32_t)n;
    bool octaves = true;
    int shift = 0;
    while (above + inside > (uint32_t)kList && lo != hi) {       // [lo, hi]: the distances among which the k-th class is
        for (int i = threadIdx.x; i < kBins; i += NT) s.count[i] = 0;
        __syncthreads();
        each_class(r, [&](float x, int) {
            const uint32_t D = kmax - order_key(x);
            if (octaves)
                atomicAdd(&s.count[octave_bin(D)], 1u);
            else if (D >= lo && D <= hi)
                atomicAdd(&s.count[(D - lo) >> shift], 1u);
        });
        __syncthreads();
        int bin = kBins - 1;
        uint32_t before = 0;
        find_bin<NT, uint32_t>(s.count, (uint32_t)k - above, bin, before, s.red32, s.answer);
        inside = s.count[bin];
        above += before;
        if (octaves)
            octave_range(bin, lo, hi);
        else {
            lo += (uint32_t)bin << shift;
            hi = lo + ((1u << shift) - 1);
        }
        octaves = false;
        shift = 0;
        while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
        __syncthreads();
    }
    const bool whole = above + inside <= (uint32_t)kList;       // else: more equal values at lo than fit, the first of them by class
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each_class(r, [&](float x, int i) {
        const uint32_t D = kmax - order_key(x);
        if (whole ? D <= hi : D < lo) push(s, D, i);
    });
    __syncthreads();
    int m = min(s.n, kList);
    if (!whole) {
        const uint32_t need = (uint32_t)k - above;
        uint32_t seen = 0;
        for (int base = 0; base < n && seen < need; base += NT) {
            const int i = base + (int)threadIdx.x;
            const uint32_t hit = i < n && kmax - order_key(Pack<T>::one(row + i)) == lo;
            uint32_t total;
            const uint32_t at = seen + block_scan<NT, uint32_t>(hit, total, s.red32);
            if (hit && at < need && m + (int)at < kList) s.list[m + (int)at] = (u64)lo << 32 | (uint32_t)i;
            seen += total;
            if (base > n - NT) break;
        }
        m = k;
        __syncthreads();
    }
    sort_list<NT>(s.list, m);
    return m;
}

// A value that at least k classes reach, and few more: the k-th largest of the threads' own maxima, rounded down to its distance's bin.
// Each maximum is a class of its own, so k of them are k classes; with k well below the number of threads, on classes in no
// particular order, hardly more than k lie above it.  One histogram of NT values instead of one of the row.
template <int NT>
__device__ float head_bound(float mine, uint32_t kmax, int k, Shared &s)
{
    for (int i = threadIdx.x; i < kBins; i += NT) s.count[i] = 0;
    __syncthreads();
    atomicAdd(&s.count[octave_bin(kmax - order_key(mine))], 1u);
    __syncthreads();
    int bin = kBins - 1;
    uint32_t before = 0, lo, hi;
    find_bin<NT, uint32_t>(s.count, (uint32_t)k, bin, before, s.red32, s.answer);
    octave_range(bin, lo, hi);
    const uint32_t key = hi < kmax ? kmax - hi : 0;
    return key_value(max(key, kKeyMinusInf));
}
template <int NT>
__device__ uint32_t block_max_key(float mine, Shared &s)
{
    return block_all<NT>(order_key(mine), [](uint32_t a, uint32_t b) { return max(a, b); }, s.red32);
}
// k that head_bound serves; beyond, the list is likely to overflow and the histograms of top_list are the shorter way
template <int NT>
__device__ __forceinline__ bool bound_serves(uint32_t kmax, int k, int n)
{
    return n > kList && k <= NT / 2 && kmax != kKeyNan;
}

// running maximum (NaN from the first NaN on) and sum of exp2((x - m) c): the softmax statistics in one pass
struct MaxSum {
    float m, sum;
};
__device__ __forceinline__ float base_of(float m) { return m == -__builtin_inff() ? 0.f : m; }
__device__ __forceinline__ void add_exp(MaxSum &a, float x, float c)
{
    if (x > a.m || x != x) {
        a.sum *= __builtin_amdgcn_exp2f((a.m - x) * c);
        a.m = x;
    }
    a.sum += __builtin_amdgcn_exp2f((x - base_of(a.m)) * c);
}
__device__ __forceinline__ float lowered(float sum, float from, float to, float c)        // a sum taken at maximum `from`, at `to` >= from
{
    return from == to ? sum : sum * __builtin_amdgcn_exp2f((from - to) * c);
}
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c)
{
    const float m = __builtin_elementwise_maximum(a.m, b.m);
    return MaxSum{m, lowered(a.sum, a.m, m, c) + lowered(b.sum, b.m, m, c)};
}
template <int NT>
__device__ MaxSum block_join(MaxSum a, float c, u64 *red64)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, MaxSum{__shfl_xor(a.m, o), __shfl_xor(a.sum, o)}, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red64[threadIdx.x >> 6] = (u64)__float_as_uint(a.m) << 32 | __float_as_uint(a.sum);
    __syncthreads();
    MaxSum r{__uint_as_float((uint32_t)(red64[0] >> 32)), __uint_as_float((uint32_t)red64[0])};
    for (int w = 1; w < NT / 64; ++w)
        r = join(r, MaxSum{__uint_as_float((uint32_t)(red64[w] >> 32)), __uint_as_float((uint32_t)red64[w])}, c);
    return r;
}

// ---- temperature -----------------------------------------------------------------------------------------------------------
struct Scale {                  // of a temperature T, divided on the host: a division in 64 bits costs a wave more than its share of a short row
    double inv;                 // 1 / T
    float c;                    // log2(e) / T
    double loss, grad;          // what a divergence and its gradient are multiplied by: T^2 and T times the caller's factor
    explicit Scale(double t, double factor = 1.0)
        : inv(1.0 / t), c((float)(1.4426950408889634074 / t)), loss(t * t * factor), grad(t * factor)
    {
    }
};

// ---- top logits -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float record_rest(float m, float sum, const Scale &scale)
{
    // the maximum may be far larger than the logarithm: one rounding for the two; at m = +inf the sum is a NaN that says nothing
    return (m == -__builtin_inff() && sum == 0.f) || m == __builtin_inff() ? m : (float)((double)m * scale.inv + (double)logf(sum));
}

// One workgroup a row, two passes: the threads' maxima, then the head (what reaches head_bound) to a list that is sorted and all others into
// the log-sum-exp.  Rows of up to 64 KiB stay in LDS between the two.  2048 x 32000 bf16, k = 32: 45 us = 2.9 TB/s (a histogram of every row
// instead of the bound: 212 us; the row read twice instead of held: 50 us).  No unit bounds it alone: with the row in LDS two workgroups fit a CU, 3.7
// waves a SIMD are in flight, the vector units are busy for 64 % of the time, and each workgroup loads or works.  One row of 100003 fp32, k = 64: 16 us, the latency of two passes of one workgroup; the call's host side is 13 us.
template <typename T, int NT, bool HELD>
__global__ __launch_bounds__(NT) void top_logits_kernel(const T *__restrict__ logits, long long stride, int n, int k, Scale scale,
                                                        T *__restrict__ values, int *__restrict__ indices, float *__restrict__ rest)
{
    __shared__ Shared s;
    const T *row = logits + (size_t)blockIdx.x * stride;
    const size_t out = (size_t)blockIdx.x * k;
    const float c = scale.c;
    extern __shared__ u32x4 held[];
    const Row<T, NT, HELD> r(row, n, held);
    const float mine = r.first_pass();
    const uint32_t kmax = block_max_key<NT>(mine, s);
    if (kmax <= kKeyMinusInf) {             // nothing but -inf: the first classes
        for (int i = threadIdx.x; i < k; i += NT) {
            values[out + i] = row[i];
            indices[out + i] = i;
        }
        if (threadIdx.x == 0) rest[blockIdx.x] = -__builtin_inff();
        return;
    }
    int m = kList + 1;
    float bound = 0.f, sum = 0.f;
    if (bound_serves<NT>(kmax, k, n)) {
        bound = head_bound<NT>(mine, kmax, k, s);
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        // the head goes to the list, all others are summed up at the bound
        r.each([&](const float *x, int base) {
            float e[r.N];
#pragma unroll
            for (int j = 0; j < r.N; ++j) e[j] = __builtin_amdgcn_exp2f((x[j] - bound) * c);
            if (largest<r.N>(x) >= bound) {
#pragma unroll
                for (int j = 0; j < r.N; ++j)
                    if (x[j] >= bound) {
                        e[j] = 0.f;
                        if (j < n - base) push(s, kmax - order_key(x[j]), base + j);
                    }
            }
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < r.N; ++j) part += e[j];
            sum += part;
        });
        __syncthreads();
        m = s.n;
        if (m <= kList) sort_list<NT>(s.list, m);
    }
    MaxSum a{-__builtin_inff(), 0.f};
    bool again = m > kList;                 // (uniform) the others have to be gone through by their own maximum
    if (again)
        top_list<T, NT>(r, row, n, kmax, k, &s);
    else {
        // the list's own tail is the first of the others; where it is empty and the bound is so far above the others that their sum has
        // no digits left, they are taken again
        const float top = m > k ? key_value(kmax - (uint32_t)(s.list[k] >> 32)) : bound;
        sum = sum == 0.f ? 0.f : sum * __builtin_amdgcn_exp2f((bound - top) * c);
        for (int i = k + (int)threadIdx.x; i < m; i += NT) sum += __builtin_amdgcn_exp2f((key_value(kmax - (uint32_t)(s.list[i] >> 32)) - top) * c);
        a = MaxSum{top, block_all<NT>(sum, [](float x, float y) { return x + y; }, reinterpret_cast<float *>(s.red32))};
        again = !(a.sum >= 0x1p-60f);
    }
    for (int i = threadIdx.x; i < k; i += NT) {
        values[out + i] = Pack<T>::to(key_value(kmax - (uint32_t)(s.list[i] >> 32)));
        indices[out + i] = (int)(uint32_t)s.list[i];
    }
    if (again) {
        const u64 last = s.list[k - 1];
        a = MaxSum{-__builtin_inff(), 0.f};
        each_class(r, [&](float x, int i) {
            if (((u64)(kmax - order_key(x)) << 32 | (uint32_t)i) > last) add_exp(a, x, c);
        });
        a = block_join<NT>(a, c, s.red64);
    }
    if (threadIdx.x == 0) rest[blockIdx.x] = record_rest(a.m, a.sum, scale);
}

// ---- rows of up to 256 classes: one wave each, sorted in registers --------------------------------------------------------------
// (1536 x 51 fp32, k = 8: 4.2 us against 16.8 with a workgroup a row; beyond 256 classes the network's steps outgrow a workgroup's two passes)
// slot j of lane l is place l * NE + j of the order; 64 * NE places, filled up with ~0
template <int NE>
__device__ __forceinline__ void sort_wave(u64 (&v)[NE])
{
    const int lane = threadIdx.x & 63;
    constexpr int CAP = 64 * NE;
#pragma unroll
    for (int k = 2; k <= CAP; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (j >= NE) {
#pragma unroll
                for (int i = 0; i < NE; ++i) {
                    const u64 other = __shfl_xor(v[i], j / NE);
                    const int at = lane * NE + i;
                    const bool low = (at & j) == 0, up = (at & k) == 0;
                    v[i] = (low == up) == (other < v[i]) ? other : v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < NE; ++i)
                    if ((i & j) == 0) {
                        const bool up = ((lane * NE + i) & k) == 0;
                        const u64 x = v[i], y = v[i | j];
                        const bool swap = (y < x) == up;
                        v[i] = swap ? y : x;
                        v[i | j] = swap ? x : y;
                    }
            }
        }
}
template <typename T, int NE>
__device__ __forceinline__ uint32_t load_wave(const T *__restrict__ row, int n, u64 (&v)[NE])
{
    const int lane = threadIdx.x & 63;
    uint32_t key[NE], kmax = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
        key[j] = j * 64 + lane < n ? order_key(Pack<T>::one(row + j * 64 + lane)) : 0;
        kmax = max(kmax, key[j]);
    }
    kmax = wave_all(kmax, [](uint32_t a, uint32_t b) { return max(a, b); });
#pragma unroll
    for (int j = 0; j < NE; ++j) v[j] = j * 64 + lane < n ? (u64)(kmax - key[j]) << 32 | (uint32_t)(j * 64 + lane) : ~0ull;
    sort_wave<NE>(v);
    return kmax;
}
constexpr int kSmall = 256;

template <typename T, int NE>
__global__ __launch_bounds__(256) void top_logits_small_kernel(const T *__restrict__ logits, long long stride, int rows, int n, int k,
                                                               Scale scale, T *__restrict__ values, int *__restrict__ indices,
                                                               float *__restrict__ rest)
{
    const int row = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    u64 v[NE];
    const uint32_t kmax = load_wave<T, NE>(logits + (size_t)row * stride, n, v);
    const float c = scale.c;
    float x[NE], m = -__builtin_inff(), sum = 0.f;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
        const int at = lane * NE + j;
        x[j] = key_value(kmax - (uint32_t)(v[j] >> 32));
        if (at < k) {
            values[(size_t)row * k + at] = Pack<T>::to(x[j]);
            indices[(size_t)row * k + at] = (int)(uint32_t)v[j];
        } else if (at < n)
            m = __builtin_elementwise_maximum(m, x[j]);
    }
    m = wave_all(m, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
#pragma unroll
    for (int j = 0; j < NE; ++j)
        if (lane * NE + j >= k && lane * NE + j < n) sum += __builtin_amdgcn_exp2f((x[j] - base_of(m)) * c);
    sum = wave_all(sum, [](float a, float b) { return a + b; });
    if (lane == 0) rest[row] = record_rest(m, sum, scale);
}

// ---- distillation -----------------------------------------------------------------------------------------------------------
constexpr int kStats = 10;      // floats a row: struct RowStats
constexpr int kPart = 4;        // floats a segment: struct Part
constexpr int kSegment = 65536; // classes of one workgroup: its share of the record's membership is a bitmap in LDS

struct Teacher {
    const void *values;
    int dtype;
    const void *indices;
    int wide;                   // indices are int64
    const float *rest;          // or NULL
    int k;
};
__device__ __forceinline__ float teacher_value(const Teacher &t, size_t i)
{
    if (t.dtype == MH_F32) return static_cast<const float *>(t.values)[i];
    if (t.dtype == MH_F16) return Pack<f16>::one(static_cast<const f16 *>(t.values) + i);
    return Pack<bf16>::one(static_cast<const bf16 *>(t.values) + i);
}
__device__ __forceinline__ int teacher_class(const Teacher &t, size_t i, int classes)       // -1: the entry is left out
{
    const long long c = t.wide ? static_cast<const long long *>(t.indices)[i] : static_cast<const int *>(t.indices)[i];
    return c >= 0 && c < classes ? (int)c : -1;
}

// What a workgroup found in its classes outside and inside the record: the sums of exp2((x - m) c), each at a maximum of its own.  A student that is
// sure leaves so little outside that it would be 0 at the row's maximum, in 32 bits as in 64; its logarithm is what the rest's bin asks for.
struct Part {
    MaxSum out, in;
};
__device__ __forceinline__ Part join(Part a, Part b, float c) { return Part{join(a.out, b.out, c), join(a.in, b.in, c)}; }

// A row's record in LDS: sized by k, asked for at the start of the row, so that its end waits for nothing but arithmetic.
struct Record {
    int *cls;                   // -1: none
    float *value, *student;     // student: the logits of these classes
    __device__ __forceinline__ Record(uint32_t *lds, int k) : cls((int *)lds), value((float *)lds + k), student((float *)lds + 2 * k) {}
};

struct RowStats {               // what a row's gradient needs: of the classes outside the record the maximum, log2 of the sum at it and the gradient
    float mo, l2o, factor, tm;  // of their whole share (q_rest - p_rest); the teacher's maximum; the logarithms of the student's sum at m
    double ls, lz;              // and of the teacher's
    float m;
    bool live;
};
// one wave: the row's loss and what its gradient needs, from the sums over the classes outside and inside the record, each at its own maximum
// (whole in lane 0).  In 64 bits: a divergence is a small difference of logarithms where the student is near the teacher.
__device__ __forceinline__ RowStats finish_row(const Record &e, int k, bool with_rest, float rest, float weight, int r, const Scale &scale, float mo,
                                               double out, float mi, double in, float *stats, float *row_loss)
{
    const int lane = threadIdx.x & 63;
    auto plus = [](double x, double y) { return x + y; };
    float tm = -__builtin_inff();
    bool some = false;               // an entry that is not -inf (a NaN is one)
    for (int i = lane; i < k; i += 64)
        if (e.cls[i] >= 0) {
            tm = fmaxf(tm, e.value[i]);
            some |= !(e.value[i] == -__builtin_inff());
        }
    tm = wave_all(tm, [](float x, float y) { return fmaxf(x, y); });
    // the sum of all at the larger maximum, and the logarithm of the share outside (-inf where every class there is)
    const float m = fmaxf(mo, mi);
    auto at_m = [&](double sum, float from) { return sum == 0.0 ? 0.0 : from == m ? sum : sum * exp(((double)from - (double)m) * scale.inv); };
    const double S = at_m(out, mo) + at_m(in, mi);
    const bool live = __any(some) && !(S == 0.0);
    // the teacher's bins, in units of T: (t - tm) / T, and the others' log-sum-exp minus tm / T
    const double yr = with_rest ? (double)rest - (double)tm * scale.inv : -__builtin_inf();
    const double shift = __builtin_fmax(0.0, yr), p_rest = with_rest ? exp(yr - shift) : 0.0;
    double z = 0.0;
    for (int i = lane; i < k; i += 64)
        if (e.cls[i] >= 0) z += exp(((double)e.value[i] - (double)tm) * scale.inv - shift);
    z = wave_all(z, plus) + p_rest;
    const double lz = shift + log(z), ls = log(S);
    double sum = 0.0;
    for (int i = lane; i < k; i += 64)
        if (e.cls[i] >= 0) {
            const double logp = ((double)e.value[i] - (double)tm) * scale.inv - lz, p = exp(logp);
            if (!(p == 0.0)) sum += p * (logp - (((double)e.student[i] - (double)m) * scale.inv - ls));
        }
    sum = wave_all(sum, plus);
    const double lo = log(out), logq = out == 0.0 ? -__builtin_inf() : mo == m ? lo - ls : ((double)mo - (double)m) * scale.inv + lo - ls;
    double factor = exp(logq);
    if (with_rest) {
        const double p = exp(yr - lz);
        if (!(p == 0.0)) {
            sum += p * ((yr - lz) - logq);
            factor -= p;
        }
    }
    // (nothing but -inf outside: no gradient there)
    const RowStats q{out == 0.0 ? 0.f : mo, out == 0.0 ? 0.f : (float)(lo * 1.4426950408889634074), out == 0.0 ? 0.f : (float)factor, tm, ls, lz, m, live};
    if (lane == 0) {
        row_loss[r] = live && weight != 0.f ? (float)(scale.loss * sum * weight) : 0.f;
        float *st = stats + (size_t)r * kStats;
        st[0] = q.mo;
        st[1] = q.l2o;
        st[2] = q.factor;
        st[3] = q.tm;
        reinterpret_cast<double *>(st)[2] = ls;
        reinterpret_cast<double *>(st)[3] = lz;
        st[8] = live ? 1.f : 0.f;
        st[9] = q.m;
    }
    return q;
}
__device__ __forceinline__ MaxSum wave_join(MaxSum a, float c)          // the reference first, so that each lane is lowered once
{
    const float m = wave_all(a.m, [](float x, float y) { return fmaxf(x, y); });
    return MaxSum{m, wave_all(lowered(a.sum, a.m, m, c), [](float x, float y) { return x + y; })};
}
__device__ __forceinline__ Part wave_join(Part a, float c) { return Part{wave_join(a.out, c), wave_join(a.in, c)}; }

// The gradient of n classes of a row, all of it written; NT threads.  Outside the record it is the class's share of the mass there, at most 1, times
// q_rest - p_rest: q (1 - p_rest / q_rest) would be a product of a number that overflows and one that is flushed to 0 where the student is sure.
// entry(i, cls, prob, student): entry i of the record, class -1 where it is none of these; prob in 64 bits.  scratch: 3 k words of LDS.
template <typename T, int NT, typename ENTRY>
__device__ __forceinline__ void write_gradient(const T *__restrict__ row, ENTRY entry, int n, T *__restrict__ out, int k, const RowStats &q, double up,
                                               bool zero, const Scale &scale, uint32_t *scratch)
{
    constexpr int N = Pack<T>::N, PER = kMaxTop / NT, AHEAD = 4;
    int *cls = (int *)scratch;
    float *high = (float *)scratch + k, *low = (float *)scratch + 2 * k, student[PER];          // (a probability as the sum of two floats)
    const int whole = n / N;
    if (zero) {
        for (int i = threadIdx.x; i < whole; i += NT) *reinterpret_cast<typename Pack<T>::raw *>(out + i * N) = u32x4{0, 0, 0, 0};
        for (int i = whole * N + (int)threadIdx.x; i < n; i += NT) out[i] = Pack<T>::to(0.f);
        return;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * NT >= k) break;
        const int i = (int)threadIdx.x + j * NT;
        if (i < k) {
            double p = 0.0;
            entry(i, cls[i], p, student[j]);
            high[i] = (float)p;
            low[i] = (float)(p - (double)(float)p);
        }
    }
    const float f = (float)(up * q.factor);
    for (int i = threadIdx.x; i < whole; i += AHEAD * NT) {
        u32x4 v[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) v[j] = load_vector(row, min(i + j * NT, whole - 1) * N);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i + j * NT < whole) {
                float x[N];
                Pack<T>::expand(v[j], x);
#pragma unroll
                for (int l = 0; l < N; ++l) x[l] = f * __builtin_amdgcn_exp2f(__builtin_fmaf(x[l] - q.mo, scale.c, -q.l2o));
                *reinterpret_cast<typename Pack<T>::raw *>(out + (i + j * NT) * N) = Pack<T>::pack(x);
            }
    }
    for (int i = whole * N + (int)threadIdx.x; i < n; i += NT)
        out[i] = Pack<T>::to(f * __builtin_amdgcn_exp2f(__builtin_fmaf(Pack<T>::one(row + i) - q.mo, scale.c, -q.l2o)));
    // the record's classes, written over the row's; the first entry of a class carries the sum over its entries
    __syncthreads();
#pragma unroll
    for (int l = 0; l < PER; ++l) {
        if (l * NT >= k) break;
        const int i = (int)threadIdx.x + l * NT, mine = i < k ? cls[i] : -1;
        if (mine < 0) continue;
        double p = 0.0;
        bool first = true;
        for (int j = 0; j < k; ++j)
            if (cls[j] == mine) {
                p += (double)high[j] + (double)low[j];
                first = first && j >= i;
            }
        if (first) out[mine] = Pack<T>::to((float)(up * (exp(((double)student[l] - (double)q.m) * scale.inv - q.ls) - p)));
    }
}

// One workgroup of 256 a row (of a segment of one beyond kSegment classes): the sums over the classes outside and inside the record in one pass.
// 2048 x 32000 fp32 without gradient: 59 us = 4.5 TB/s of 5.
// GRAD: the row's gradient at an upstream of 1 too (nseg = 1), by reading the row again.  4096 x 32000 bf16: 165 us for both, 3.2 TB/s of what has to
// move; a pass of its own for the gradient makes it 192.  The second reading does not hit the L2s (5.3 waves a SIMD keep more rows in flight
// than they hold): 566 MB fetched and 272 written, 5.1 TB/s, a copy's rate.  Measured and left: the row held in LDS 184 us (two workgroups
// of 512 a CU), 512 threads a row 182, 1024 227: fewer rows in flight.  References apart for the classes outside and inside the record cost 1 us.
template <typename T, int NT, bool REST, bool GRAD>
__global__ __launch_bounds__(NT) void distill_fwd_kernel(const T *__restrict__ logits, long long stride, int classes, Teacher t, Scale scale,
                                                         const float *__restrict__ row_weight, float *__restrict__ stats,
                                                         float *__restrict__ row_loss, float *__restrict__ parts, int nseg,
                                                         float divisor, const float *__restrict__ divided_by, T *__restrict__ grad)
{
    extern __shared__ uint32_t lds[];
    __shared__ Part red[NT / 64];
    __shared__ RowStats shared_stats;
    __shared__ int twice;
    constexpr int N = Pack<T>::N, AHEAD = 4, PER = kMaxTop / NT;
    const int r = nseg == 1 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)nseg), seg = nseg == 1 ? 0 : (int)(blockIdx.x % (unsigned)nseg);
    const int first = seg * kSegment, n = min(kSegment, classes - first), nv = (n + N - 1) / N;
    const T *row = logits + (size_t)r * stride, *at = row + first;
    const float c = scale.c;
    const float rest = REST ? t.rest[r] : 0.f, weight = row_weight ? row_weight[r] : 1.f;
    const Record record(lds, t.k);
    uint32_t *member = lds + 3 * t.k;
    auto bits = [&](int i) { return member[i * N >> 5] >> (i * N & 31) & ((1u << N) - 1); };
    // The record's classes, one bit each.  The vectors that hold any are few: the loop over the row leaves them out whole, and each is taken
    // by the entry that names its lowest class of the record (the first such entry), so that sums run in a fixed order.
    if (REST) {
        for (int i = threadIdx.x; i < (n + 31) / 32; i += NT) member[i] = 0;
        if (threadIdx.x == 0) twice = 0;
        __syncthreads();
    }
    float student[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (j * NT >= t.k) break;
        const int i = (int)threadIdx.x + j * NT;
        if (i < t.k) {
            const int cls = teacher_class(t, (size_t)r * t.k + i, classes), k = cls - first;
            const bool here = cls >= 0 && k >= 0 && k < n;
            record.cls[i] = cls;
            if (cls >= 0 && nseg == 1) {
                record.value[i] = teacher_value(t, (size_t)r * t.k + i);
                student[j] = Pack<T>::one(row + cls);
            }
            if (REST && here && (atomicOr(&member[k >> 5], 1u << (k & 31)) >> (k & 31) & 1)) twice = 1;
        }
    }
    if (REST) __syncthreads();
    auto special = [&](auto f) {          // f(vector, its classes of the record)
        if (!REST) return;
        for (int i = threadIdx.x; i < t.k; i += NT) {
            const int cls = record.cls[i], k = cls - first;
            if (cls < 0 || k < 0 || k >= n) continue;
            const uint32_t inside = bits(k / N);
            if ((inside & -inside) != 1u << (k % N)) continue;
            bool again = false;
            if (twice)
                for (int j = 0; j < i; ++j) again |= record.cls[j] == cls;
            if (!again) f(k / N, inside);
        }
    };
    // Sums at references of this thread, one for the classes outside the record and one for those inside, no more than 8 octaves below the largest
    // class of the side.  The exponent is fma(x, c, -base), base = m c rounded: one operation a class, and one rounding of a number that is
    // small where the weight is not; the base's own rounding, at most 2^4 within +-kBase, is taken out at the end.  The reference is looked at
    // once in AHEAD vectors and seldom raised.  A base beyond kBase, whose rounding would be an exponent of any size, stays at kBase: a class
    // far below weighs 0 until a larger one raises the reference, and a thread that meets none ends with its differences (below).
    constexpr float kBase = 0x1p29f;
    struct Side {
        float m, base, most, sum;
    };
    Side out{-__builtin_inff(), -kBase, -__builtin_inff(), 0.f}, in = out;
    auto raise = [&](Side &a, float m) {
        a.most = fmaxf(a.most, m);
        if (__any(__builtin_fmaf(m, c, -a.base) > 8.f)) {
            if (__builtin_fmaf(m, c, -a.base) > 8.f) {
                const float from = a.base;
                a.base = __builtin_isinf(m) ? m : fminf(fmaxf(m * c, -kBase), kBase);
                a.m = m;
                a.sum *= __builtin_amdgcn_exp2f(from - a.base);
            }
        }
    };
    auto weight_of = [&](const Side &a, float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -a.base)); };
    stream_batches<T, NT, AHEAD>(at, n, [&](const u32x4 (&raw)[AHEAD], int i, int count) {
        float x[AHEAD][N], m = -__builtin_inff();
        bool mixed[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (j < count) {
                mixed[j] = REST && bits(i + j * NT);
                Pack<T>::expand(raw[j], x[j]);
                float top = x[j][0];
#pragma unroll
                for (int l = 1; l < N; ++l) top = fmaxf(top, x[j][l]);
                m = mixed[j] ? m : fmaxf(m, top);
            }
        raise(out, m);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (j < count) {
                float sum = weight_of(out, x[j][0]);
#pragma unroll
                for (int l = 1; l < N; ++l) sum += weight_of(out, x[j][l]);
                out.sum += mixed[j] ? 0.f : sum;
            }
    });
    special([&](int v, uint32_t inside) {
        float x[N], mo = -__builtin_inff(), mi = mo;
        Pack<T>::expand(load_any(at, n, v * N), x);
#pragma unroll
        for (int l = 0; l < N; ++l)
            if (inside >> l & 1)
                mi = fmaxf(mi, x[l]);
            else
                mo = fmaxf(mo, x[l]);
        raise(out, mo);
        raise(in, mi);
#pragma unroll
        for (int l = 0; l < N; ++l)
            if (inside >> l & 1)
                in.sum += weight_of(in, x[l]);
            else
                out.sum += weight_of(out, x[l]);
    });
    Part a;
    auto beyond = [&](const Side &a) { return !__builtin_isinf(a.most) && __builtin_fabsf(a.most * c) > kBase / 2; };
    if (beyond(out) || beyond(in)) {
        // this thread's largest class times c is beyond half of kBase (all of them at the type's lowest value): differences first
        a = Part{{out.most, 0.f}, {in.most, 0.f}};
        const float mo = base_of(out.most), mi = base_of(in.most);
        auto one = [&](int v, uint32_t inside) {
            for (int l = 0; l < N && v * N + l < n; ++l) {
                const float x = Pack<T>::one(at + v * N + l);
                if (inside >> l & 1)
                    a.in.sum += __builtin_amdgcn_exp2f((x - mi) * c);
                else
                    a.out.sum += __builtin_amdgcn_exp2f((x - mo) * c);
            }
        };
        for (int i = threadIdx.x; i < nv; i += NT)
            if (!REST || !bits(i)) one(i, 0);
        special(one);
    } else {
        auto settled = [&](const Side &a) {
            return MaxSum{a.m, a.m == -__builtin_inff() ? a.sum : a.sum * __builtin_amdgcn_exp2f(-__builtin_fmaf(a.m, c, -a.base))};
        };
        a = Part{settled(out), settled(in)};
    }
    a = wave_join(a, c);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    if (nseg == 1) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (j * NT >= t.k) break;
            const int i = (int)threadIdx.x + j * NT;
            if (i < t.k) record.student[i] = student[j];
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        a = red[0];
        for (int w = 1; w < NT / 64; ++w) a = join(a, red[w], c);
        if (nseg == 1) {
            const RowStats q = finish_row(record, t.k, REST, rest, weight, r, scale, a.out.m, a.out.sum, a.in.m, a.in.sum, stats, row_loss);
            if (GRAD && threadIdx.x == 0) shared_stats = q;
        } else if (threadIdx.x == 0) {
            float *p = parts + (size_t)blockIdx.x * kPart;
            p[0] = a.out.m;
            p[1] = a.out.sum;
            p[2] = a.in.m;
            p[3] = a.in.sum;
        }
    }
    if (!GRAD) return;
    __syncthreads();
    const RowStats q = shared_stats;
    write_gradient<T, NT>(
        row,
        [&](int i, int &cls, double &prob, float &s) {          // (over the record itself: each entry reads its own words first)
            s = record.student[i];
            prob = exp(((double)record.value[i] - (double)q.tm) * scale.inv - q.lz);
            cls = record.cls[i];
        },
        n, grad + (size_t)r * classes, t.k, q, scale.grad * weight / (divisor > 0.f ? divisor : *divided_by), !q.live || weight == 0.f, scale, lds);
}
// Rows of up to kShort classes: the maxima outside and inside the record and the sums at them in 64 bits.  Their divergences may be far smaller than
// the logarithms they are differences of (a head of few classes, sure of one), and 64 bits cost such a row next to nothing (1536 x 51: 13 us;
// the calls around the kernel take five to ten times that).
constexpr int kShort = 2048;
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_short_kernel(const T *__restrict__ logits, long long stride, int n, Teacher t, Scale scale,
                                                           const float *__restrict__ row_weight, float *__restrict__ stats,
                                                           float *__restrict__ row_loss, float divisor, const float *__restrict__ divided_by,
                                                           T *__restrict__ grad)
{
    extern __shared__ uint32_t lds[];
    __shared__ uint32_t member[kShort / 32];
    __shared__ double red[NT / 64];
    __shared__ RowStats shared_stats;
    const int r = blockIdx.x;
    const T *row = logits + (size_t)r * stride;
    const float rest = t.rest ? t.rest[r] : 0.f, weight = row_weight ? row_weight[r] : 1.f;
    const Record record(lds, t.k);
    for (int i = threadIdx.x; i < kShort / 32; i += NT) member[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < t.k; i += NT) {
        const int cls = teacher_class(t, (size_t)r * t.k + i, n);
        record.cls[i] = cls;
        if (cls >= 0) {
            record.value[i] = teacher_value(t, (size_t)r * t.k + i);
            record.student[i] = Pack<T>::one(row + cls);
            if (t.rest) atomicOr(&member[cls >> 5], 1u << (cls & 31));
        }
    }
    float x[kShort / NT], mo = -__builtin_inff(), mi = mo;
#pragma unroll
    for (int j = 0; j < kShort / NT; ++j) {
        const int i = (int)threadIdx.x + j * NT;
        x[j] = i < n ? Pack<T>::one(row + i) : -__builtin_inff();
    }
    __syncthreads();          // (member is whole)
    auto inside = [&](int i) { return member[i >> 5] >> (i & 31) & 1; };
#pragma unroll
    for (int j = 0; j < kShort / NT; ++j) {
        const int i = (int)threadIdx.x + j * NT;
        if (inside(i))
            mi = fmaxf(mi, x[j]);
        else
            mo = fmaxf(mo, x[j]);
    }
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    mo = block_all<NT>(mo, larger, reinterpret_cast<float *>(red));
    mi = block_all<NT>(mi, larger, reinterpret_cast<float *>(red));
    double out = 0.0, in = 0.0;
#pragma unroll
    for (int j = 0; j < kShort / NT; ++j) {
        const int i = (int)threadIdx.x + j * NT;
        if (i < n) {
            // (nothing but -inf: every difference would be a NaN)
            const bool is_in = inside(i);
            const double e = x[j] == -__builtin_inff() ? 0.0 : exp(((double)x[j] - (double)(is_in ? mi : mo)) * scale.inv);
            (is_in ? in : out) += e;
        }
    }
    auto plus = [](double a, double b) { return a + b; };
    out = block_all<NT>(out, plus, red);
    in = block_all<NT>(in, plus, red);
    if (threadIdx.x < 64) {
        const RowStats q = finish_row(record, t.k, t.rest != nullptr, rest, weight, r, scale, mo, out, mi, in, stats, row_loss);
        if (threadIdx.x == 0) shared_stats = q;
    }
    if (!grad) return;
    __syncthreads();
    const RowStats q = shared_stats;
    write_gradient<T, NT>(
        row,
        [&](int i, int &cls, double &prob, float &s) {
            s = record.student[i];
            prob = exp(((double)record.value[i] - (double)q.tm) * scale.inv - q.lz);
            cls = record.cls[i];
        },
        n, grad + (size_t)r * n, t.k, q, scale.grad * weight / (divisor > 0.f ? divisor : *divided_by), !q.live || weight == 0.f, scale, lds);
}
template <typename T>
__global__ __launch_bounds__(64) void distill_join_kernel(const T *__restrict__ logits, long long stride, int classes, Teacher t, Scale scale,
                                                          const float *__restrict__ row_weight, float *__restrict__ stats,
                                                          float *__restrict__ row_loss, const float *__restrict__ parts, int nseg)
{
    extern __shared__ uint32_t lds[];
    const int r = blockIdx.x;
    const Record record(lds, t.k);
    for (int i = threadIdx.x; i < t.k; i += 64) {
        const int cls = teacher_class(t, (size_t)r * t.k + i, classes);
        record.cls[i] = cls;
        if (cls >= 0) {
            record.value[i] = teacher_value(t, (size_t)r * t.k + i);
            record.student[i] = Pack<T>::one(logits + (size_t)r * stride + cls);
        }
    }
    __syncthreads();
    const MaxSum none{-__builtin_inff(), 0.f};
    Part a{none, none};
    for (int i = threadIdx.x; i < nseg; i += 64) {
        const float *p = parts + ((size_t)r * nseg + i) * kPart;
        a = join(a, Part{{p[0], p[1]}, {p[2], p[3]}}, scale.c);
    }
    a = wave_join(a, scale.c);
    finish_row(record, t.k, t.rest != nullptr, t.rest ? t.rest[r] : 0.f, row_weight ? row_weight[r] : 1.f, r, scale, a.out.m, a.out.sum, a.in.m, a.in.sum,
               stats, row_loss);
}
// the sum of the weights, which the rows' sum is divided by (1 where it is 0)
__global__ __launch_bounds__(1024) void distill_weight_kernel(const float *__restrict__ row_weight, int rows, float *__restrict__ divided_by)
{
    __shared__ float red[16];
    float w = 0.f;
    for (int i = threadIdx.x; i < rows; i += 1024) w += row_weight[i];
    w = block_all<1024>(w, [](float x, float y) { return x + y; }, red);
    if (threadIdx.x == 0) *divided_by = w == 0.f ? 1.f : w;
}
// total = sum of the rows' losses over divided_by, which is `divisor` where that is above 0
__global__ __launch_bounds__(1024) void distill_total_kernel(const float *__restrict__ row_loss, int rows, float divisor, float *__restrict__ total,
                                                             float *__restrict__ divided_by)
{
    __shared__ float red[16];
    float a = 0.f;
    for (int i = threadIdx.x; i < rows; i += 1024) a += row_loss[i];
    a = block_all<1024>(a, [](float x, float y) { return x + y; }, red);
    if (threadIdx.x != 0) return;
    if (divisor > 0.f) *divided_by = divisor;
    *total = a / (divisor > 0.f ? divisor : *divided_by);
}

// 4096 x 32000 bf16: 122 us = 4.3 TB/s behind the forward pass; 4 us where the gradient is there already (an upstream of 1).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void distill_bwd_kernel(const T *__restrict__ logits, long long stride, int classes, Teacher t, Scale scale,
                                                         const float *__restrict__ row_weight, const float *__restrict__ stats,
                                                         const float *__restrict__ divided_by, const float *__restrict__ upstream,
                                                         int upstream_rows, int written, T *__restrict__ grad, int nseg)
{
    extern __shared__ uint32_t lds[];
    const int r = nseg == 1 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)nseg), seg = nseg == 1 ? 0 : (int)(blockIdx.x % (unsigned)nseg);
    const int first = seg * kSegment, n = min(kSegment, classes - first);
    const float upstream_r = upstream[upstream_rows ? r : 0];
    if (written && upstream_r == 1.f) return;
    const T *row = logits + (size_t)r * stride + first;
    const float *st = stats + (size_t)r * kStats;
    const RowStats q{st[0], st[1], st[2], st[3], reinterpret_cast<const double *>(st)[2], reinterpret_cast<const double *>(st)[3], st[9], st[8] != 0.f};
    const float w = row_weight ? row_weight[r] : 1.f;
    const double up = (double)upstream_r * scale.grad * w / (divided_by ? *divided_by : 1.f);
    write_gradient<T, NT>(row,
                          [&](int i, int &cls, double &prob, float &s) {
                              const int k = teacher_class(t, (size_t)r * t.k + i, classes) - first;          // (left out: -1 - first, or less)
                              cls = k >= 0 && k < n ? k : -1;
                              if (cls < 0) return;
                              prob = exp(((double)teacher_value(t, (size_t)r * t.k + i) - (double)q.tm) * scale.inv - q.lz);
                              s = Pack<T>::one(row + k);
                          },
                          n, grad + (size_t)r * classes + first, t.k, q, up, !q.live || w == 0.f, scale, lds);
}

// ---- sampling ---------------------------------------------------------------------------------------------------------------
// A class's weight is 2^S exp((x - max) / T) rounded to a whole number, S = min(51, 62 - ceil(log2(classes))): sums of weights are exact
// and the same in every order and split, so a border between two classes, which decides a whole number, does not depend on how the row
// was cut.  Their step, 2^-S of the largest class, is the one rounding; classes further than S octaves below the maximum weigh nothing.
struct Weigher {
    double c, top, floor;  // log2(e) / T, row maximum (finite), -(S + 2)
    float per_octave;      // bins of the histogram
    int S;
    __device__ __forceinline__ Weigher(float top_, float temperature, int S_) : top(top_), S(S_)
    {
        c = 1.4426950408889634074 / (double)temperature;
        floor = -(double)(S + 2);
        per_octave = (float)(kBins - 1) / 32.f;
    }
    // log2 of the weight, the maximum's being 0; at least `floor`, which weighs nothing
    __device__ __forceinline__ double octaves(float x) const { return __builtin_fmax(((double)x - top) * c, floor); }
    __device__ __forceinline__ u64 weight(double y) const
    {
        // y = n + r, |r| <= 1/2: the sum with 1.5 * 2^52 holds n in its low word
        const double t = y + 6755399441055744.0;
        const double r = y - (t - 6755399441055744.0);
        // 2^r, interpolated at Chebyshev points, degree 8, exact at 0: off by at most 2.2e-12 of itself
        double p = 1.3250805530063054e-06;
        p = __builtin_fma(p, r, 1.530370071158824e-05);
        p = __builtin_fma(p, r, 1.5403475186470873e-04);
        p = __builtin_fma(p, r, 1.3333478473684418e-03);
        p = __builtin_fma(p, r, 9.618129135236225e-03);
        p = __builtin_fma(p, r, 5.550410906325868e-02);
        p = __builtin_fma(p, r, 2.40226506958885e-01);
        p = __builtin_fma(p, r, 6.931471805568324e-01);
        p = __builtin_fma(p, r, 1.0);
        // times 2^(n + S), on the exponent; the sum with 2^52 is rounded to a whole number in its low 52 bits
        const int n = (int)(uint32_t)(u64)__double_as_longlong(t);
        const u64 scaled = (u64)__double_as_longlong(p) + ((u64)(uint32_t)(n + S) << 52);
        return (u64)__double_as_longlong(__longlong_as_double((long long)scaled) + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 operator()(float x) const { return weight(octaves(x)); }
    // 0 .. kBins - 1, falls with x: 64 an octave; the last holds all that is more than 32 octaves below the maximum
    __device__ __forceinline__ int bin(double y) const { return min((int)(-(float)y * per_octave), kBins - 1); }
    // every value of the bins first .. last lies in [lo, hi] (a few others may)
    __device__ __forceinline__ void bin_range(int first, int last, float &lo, float &hi) const
    {
        const double step = 1.0 / (double)per_octave;
        const double x0 = top - ((double)(last + 1) * step * 1.000001 + 1e-6) / c, x1 = top - ((double)first * step * 0.999999 - 1e-6) / c;
        lo = last >= kBins - 2 ? -__builtin_inff() : (float)(x0 - __builtin_fabs(x0) * 1e-6);
        hi = (float)(x1 + __builtin_fabs(x1) * 1e-6);
    }
};
// x * m rounded down, x in [0, 1) with a step of 2^-64
__device__ __forceinline__ u64 share_down(float x, u64 m) { return __umul64hi((u64)((double)x * 18446744073709551616.0), m); }
__device__ __forceinline__ u64 share_up(float x, u64 m)
{
    const u64 f = (u64)((double)x * 18446744073709551616.0);
    return __umul64hi(f, m) + (f * m ? 1 : 0);
}
__device__ __forceinline__ u64 plus64(u64 x, u64 y) { return x + y; }

// Candidates list [0 .. m): behind `mass` in `count` classes, the running weight with the one at which it reaches `need` (by mass) or that is
// the need-th class (by count), and that class.  A need that is never reached ends at the last candidate.
template <int NT>
__device__ u64 reach(u64 *list, int m, uint32_t kmax, const Weigher &W, bool by_count, u64 need, u64 mass, uint32_t count, int &cls, SharedMass &s)
{
    sort_list<NT>(list, m);
    const int per = (m + NT - 1) / NT, first = (int)threadIdx.x * per;
    u64 sum = 0, total;
    for (int i = first; i < min(first + per, m); ++i) sum += W(key_value(kmax - (uint32_t)(list[i] >> 32)));
    u64 at = mass + block_scan<NT, u64>(sum, total, s.red64);
    if (threadIdx.x == 0) {
        s.answer[0] = mass + total;
        s.answer[1] = m > 0 ? (uint32_t)list[m - 1] : 0;
    }
    __syncthreads();
    for (int i = first; i < min(first + per, m); ++i) {
        const u64 w = W(key_value(kmax - (uint32_t)(list[i] >> 32)));
        if (by_count ? (u64)count + i + 1 == need : at < need && at + w >= need) {
            s.answer[0] = at + w;
            s.answer[1] = (uint32_t)list[i];
        }
        at += w;
    }
    __syncthreads();
    cls = (int)s.answer[1];
    return s.answer[0];
}

// The same among all classes of the histogram's bin `b`, however many they are.  Out of line: seldom called, and its registers would be
// every row's.
struct Reached {
    u64 mass;
    int cls;
};
template <typename T, int NT, typename R>
__device__ __noinline__ Reached resolve(R r, const T *row, int n, uint32_t kmax, Weigher W, bool by_count, u64 need, int b, u64 mass, uint32_t count,
                                        SharedMass *shared)
{
    SharedMass &s = *shared;
    int cls = -1;
    uint32_t lo = 0, hi = 0xffffffffu;
    bool ranged = false;
    float x0, x1;
    W.bin_range(b, b, x0, x1);
    auto members = [&](auto f) {
        each_class(r, [&](float x, int i) {
            if (x >= x0 && x <= x1 && W.bin(W.octaves(x)) == b) f(x, i);
        });
    };
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        members([&](float x, int i) {
            const uint32_t D = kmax - order_key(x);
            if (D >= lo && D <= hi) push(s, D, i);
        });
        __syncthreads();
        const int m = s.n;
        if (m <= kList) {
            const u64 at = reach<NT>(s.list, m, kmax, W, by_count, need, mass, count, cls, s);
            return Reached{at, cls};
        }
        if (!ranged) {
            uint32_t first = 0xffffffffu, last = 0;
            members([&](float x, int) {
                const uint32_t D = kmax - order_key(x);
                first = min(first, D);
                last = max(last, D);
            });
            lo = block_all<NT>(first, [](uint32_t x, uint32_t y) { return min(x, y); }, s.red32);
            hi = block_all<NT>(last, [](uint32_t x, uint32_t y) { return max(x, y); }, s.red32);
            ranged = true;
        }
        if (lo == hi) {       // more equal values than the list holds
            const u64 w = W(key_value(kmax - lo));
            u64 j = by_count ? need - count : (w ? (need - mass + w - 1) / w : (u64)m);
            j = j < 1 ? 1 : j > (u64)m ? (u64)m : j;
            cls = nth_tie<T, NT>(row, n, kmax, lo, (uint32_t)(j - 1), s);
            return Reached{mass + j * w, cls};
        }
        int shift = 0;
        while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
        // (the first histogram stays where later searches need it: these bins are the list's memory and the classes')
        static_assert(kList >= kBins, "the list holds a histogram");
        u64 *part = s.list;
        uint32_t *cnt = s.classes;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += NT) {
            part[i] = 0;
            cnt[i] = 0;
        }
        __syncthreads();
        members([&](float x, int) {
            const uint32_t D = kmax - order_key(x);
            if (D >= lo && D <= hi) {
                atomicAdd(&part[(D - lo) >> shift], W(x));
                atomicAdd(&cnt[(D - lo) >> shift], 1u);
            }
        });
        __syncthreads();
        int at = 0;
        u64 massb = 0;
        uint32_t countb = 0;
        bool found;
        if (by_count)
            found = find_bin<NT, uint32_t>(cnt, (uint32_t)need - count, at, countb, s.red32, s.answer);
        else
            found = find_bin<NT, u64>(part, need - mass, at, massb, s.red64, s.answer);
        if (!found) at = (int)((hi - lo) >> shift);
        u64 pm = 0;
        uint32_t pc = 0;
        for (int i = threadIdx.x; i < at; i += NT) {
            pm += part[i];
            pc += cnt[i];
        }
        mass += block_all<NT>(pm, plus64, s.red64);
        count += block_all<NT>(pc, [](uint32_t x, uint32_t y) { return x + y; }, s.red32);
        lo += (uint32_t)at << shift;
        hi = min(hi, lo + ((1u << shift) - 1));
    }
}

struct SampleArgs {
    const float *u, *temperature, *top_p, *min_p;       // temperature .. min_p: one value a row, or NULL and the value for all
    const int *top_k;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
    long long *labels;
};
struct Draw {               // one row's parameters
    float temperature, top_p, min_p, u;
    int k;
    double least;           // log2(min_p)
    bool with_p, with_m, greedy;
    __device__ __forceinline__ Draw(const SampleArgs &a, int r, int n)
    {
        temperature = a.temperature ? a.temperature[r] : a.temperature_all;
        top_p = a.top_p ? a.top_p[r] : a.top_p_all;
        min_p = a.min_p ? a.min_p[r] : a.min_p_all;
        k = a.top_k ? a.top_k[r] : a.top_k_all;
        if (k <= 0 || k > n) k = n;
        u = a.u[r];
        u = u > 0.f ? fminf(u, 0.99999994f) : 0.f;
        with_p = top_p < 1.f;
        with_m = min_p > 0.f;
        greedy = !(temperature > 0.f) || k == 1;
        least = with_m ? log2((double)min_p) : 0.0;
    }
    __device__ __forceinline__ bool long_head() const { return !greedy && k > kMaxTop; }
};

// The weights of some classes of a row into the histogram, and the weight of those that min-p keeps
template <typename SOURCE>
__device__ __forceinline__ u64 add_masses(SOURCE each, const Weigher &W, const Draw &d, int n, bool counted, SharedMass &s)
{
    u64 above = 0;
    each([&](const auto &x, int base) {
        constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double y = W.octaves(x[j]);
            const u64 w = W.weight(y);
            const int b = W.bin(y);
            if (w) atomicAdd(&s.mass[b], w);
            if (counted && j < n - base) atomicAdd(&s.classes[b], 1u);
            if (d.with_m && y >= d.least) above += w;
            if (j % 4 == 3) __builtin_amdgcn_sched_barrier(0);          // (all N at once do not fit the registers)
        }
    });
    return above;
}

// Few long rows: one workgroup a row leaves most of the chip idle, and the weights are what takes it long.  Their histogram is then
// made by nseg workgroups a row, which find the row's maximum first (a launch of its own), and joined in memory by whole-number additions:
// the same sums in any order.  64 x 100003 bf16, p = 0.9: 6 + 14 + 33 us against 72 in one kernel; with 1024 rows the two launches more cost what
// they gain (27 + 77 + 80 us against 162), so rows that fill half of the chip keep to themselves.
struct Cut {
    int nseg, length;           // workgroups a row (0: the row's own workgroup does it all), classes of each
    uint32_t *top;              // [rows][nseg] largest key of a segment
    u64 *mass, *above;          // [rows][kBins], [rows]
    uint32_t *classes;          // [rows][kBins]
};
template <typename T>
__global__ __launch_bounds__(256) void sample_top_kernel(const T *__restrict__ logits, long long stride, int n, Cut cut)
{
    __shared__ uint32_t red[4];
    constexpr int N = Pack<T>::N;
    const int r = (int)(blockIdx.x / (unsigned)cut.nseg), seg = (int)(blockIdx.x % (unsigned)cut.nseg), first = seg * cut.length;
    float m = -__builtin_inff();
    stream_row<T, 256, 4>(logits + (size_t)r * stride + first, min(cut.length, n - first), [&](const u32x4 &v, int) {
        float x[N];
        Pack<T>::expand(v, x);
        m = __builtin_elementwise_maximum(m, largest<N>(x));
    });
    const uint32_t key = block_all<256>(order_key(m), [](uint32_t a, uint32_t b) { return max(a, b); }, red);
    if (threadIdx.x == 0) cut.top[blockIdx.x] = key;
    for (int i = seg + (int)threadIdx.x * cut.nseg; i < kBins; i += 256 * cut.nseg) {
        cut.mass[(size_t)r * kBins + i] = 0;
        cut.classes[(size_t)r * kBins + i] = 0;
    }
    if (seg == 0 && threadIdx.x == 0) cut.above[r] = 0;
}
__device__ __forceinline__ uint32_t row_top(const Cut &cut, int r)
{
    uint32_t m = 0;
    for (int i = 0; i < cut.nseg; ++i) m = max(m, cut.top[(size_t)r * cut.nseg + i]);
    return m;
}
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_mass_kernel(const T *__restrict__ logits, long long stride, int n, int S, SampleArgs a, Cut cut)
{
    __shared__ SharedMass s;
    constexpr int N = Pack<T>::N;
    const int r = (int)(blockIdx.x / (unsigned)cut.nseg), seg = (int)(blockIdx.x % (unsigned)cut.nseg), first = seg * cut.length;
    const Draw d(a, r, n);
    const uint32_t kmax = row_top(cut, r);
    const float top = key_value(kmax);
    if (!d.long_head() || kmax == kKeyNan || __builtin_isinf(top)) return;
    const Weigher W(top, d.temperature, S);
    const bool counted = d.k < n;
    for (int i = threadIdx.x; i < kBins; i += NT) {
        s.mass[i] = 0;
        s.classes[i] = 0;
    }
    __syncthreads();
    const int length = min(cut.length, n - first);
    u64 above = add_masses(
        [&](auto f) {
            stream_row<T, NT, 1>(logits + (size_t)r * stride + first, length, [&](const u32x4 &v, int i) {
                float x[N];
                Pack<T>::expand(v, x);
                f(x, i * N);
            });
        },
        W, d, length, counted, s);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += NT) {
        if (s.mass[i]) atomicAdd(&cut.mass[(size_t)r * kBins + i], s.mass[i]);
        if (counted && s.classes[i]) atomicAdd(&cut.classes[(size_t)r * kBins + i], s.classes[i]);
    }
    if (!d.with_m) return;
    above = block_all<NT>(above, plus64, s.red64);
    if (threadIdx.x == 0 && above) atomicAdd(&cut.above[r], above);
}

// the rest of the way from a head that is sorted: weights w of PER places from `first` on, all in all `head`; scan and sum of the group
// (wave or workgroup) as functions.  Returns the place of the label or -1 in all threads but its own.
template <int PER, typename SCAN, typename SUM>
__device__ __forceinline__ int draw_from_head(const u64 (&w)[PER], const bool (&in_m)[PER], int first, const Draw &d, SCAN scan, SUM sum_all)
{
    u64 sum = 0, head;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += w[j];
    const u64 start = scan(sum, head);
    const u64 need = d.with_p ? share_up(fmaxf(d.top_p, 0.f), head) : ~0ull;
    u64 kept = 0, run = start;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (in_m[j] && (run < need || first + j == 0)) kept += w[j];
        run += w[j];
    }
    const u64 target = share_down(d.u, sum_all(kept));
    int place = -1;
    run = start;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (run <= target && run + w[j] > target) place = first + j;
        run += w[j];
    }
    return place;
}

// One workgroup a row.  A short head (top-k up to kMaxTop) is sorted whole: one row of 32000 fp32, k = 50, 11 us.  A long one has no sort: 64-bit
// weights go into a histogram by distance (64 bins an octave), top-p's border and the draw are bins of it, and only the classes of those bins
// are gathered and sorted.  1024 x 65536 fp16, p = 0.95: 162 us, of which about 80 are the weights -- some 38 instructions a class, 16 of them
// in 64 bits -- against 27 us of reading; 4 waves a SIMD (at 2, what 196 registers leave: 331 us).
template <typename T, int NT, bool HELD>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(NT >= 512 ? 4 : 3))) void sample_kernel(const T *__restrict__ logits, long long stride, int n, int S,
                                                                                                            SampleArgs a, Cut cut)
{
    __shared__ SharedMass s;
    const T *row = logits + (size_t)blockIdx.x * stride;
    extern __shared__ u32x4 held[];
    const Row<T, NT, HELD> r(row, n, held);
    const Draw d(a, blockIdx.x, n);
    const bool ready = !HELD && cut.nseg > 0 && d.long_head();          // (the histogram is there)
    const float mine = ready ? 0.f : r.first_pass();
    const uint32_t kmax = ready ? row_top(cut, blockIdx.x) : block_max_key<NT>(mine, s);
    if (kmax == kKeyNan || kmax <= kKeyMinusInf) {
        if (threadIdx.x == 0) a.labels[blockIdx.x] = -1;
        return;
    }
    if (d.greedy) {
        const float top = key_value(kmax);
        uint32_t best = 0xffffffffu;
        r.each([&](const float *x, int base) {
#pragma unroll
            for (int j = r.N - 1; j >= 0; --j)
                if (x[j] == top) best = min(best, (uint32_t)(base + j));
        });
        best = block_all<NT>(best, [](uint32_t x, uint32_t y) { return min(x, y); }, s.red32);
        if (threadIdx.x == 0) a.labels[blockIdx.x] = (long long)best;
        return;
    }
    if (key_value(kmax) == __builtin_inff()) {          // +inf takes all the weight: so many equal classes, no others
        uint32_t equal = 0;
        each_class(r, [&](float x, int) { equal += x == __builtin_inff(); });
        equal = min(block_all<NT>(equal, [](uint32_t x, uint32_t y) { return x + y; }, s.red32), (uint32_t)d.k);
        const u64 w = 1ull << S, need = d.with_p ? max(share_up(fmaxf(d.top_p, 0.f), equal * w), (u64)1) : equal * w;
        const int cls = nth_tie<T, NT>(row, n, kmax, 0, (uint32_t)(share_down(d.u, (need + w - 1) / w * w) / w), s);
        if (threadIdx.x == 0) a.labels[blockIdx.x] = cls;
        return;
    }
    const Weigher W(key_value(kmax), d.temperature, S);

    if (d.k <= kMaxTop) {          // the head of the row is short: all of it is sorted
        int m = kList + 1;
        if (bound_serves<NT>(kmax, d.k, n)) {
            const float bound = head_bound<NT>(mine, kmax, d.k, s);
            if (threadIdx.x == 0) s.n = 0;
            __syncthreads();
            r.each([&](const float *x, int base) {
                if (largest<r.N>(x) >= bound) {
#pragma unroll
                    for (int j = 0; j < r.N; ++j)
                        if (x[j] >= bound && j < n - base) push(s, kmax - order_key(x[j]), base + j);
                }
            });
            __syncthreads();
            m = s.n;
            if (m <= kList) sort_list<NT>(s.list, m);
        }
        if (m > kList) top_list<T, NT>(r, row, n, kmax, d.k, &s);
        constexpr int PER = kMaxTop / NT;
        const int first = (int)threadIdx.x * PER;
        u64 w[PER];
        bool in_m[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool is = first + j < d.k;
            const double y = is ? W.octaves(key_value(kmax - (uint32_t)(s.list[first + j] >> 32))) : 0.0;
            w[j] = is ? W.weight(y) : 0;
            in_m[j] = !d.with_m || first + j == 0 || y >= d.least;
        }
        const int place = draw_from_head<PER>(
            w, in_m, first, d, [&](u64 v, u64 &total) { return block_scan<NT, u64>(v, total, s.red64); },
            [&](u64 v) { return block_all<NT>(v, plus64, s.red64); });
        if (place >= 0) a.labels[blockIdx.x] = (long long)(uint32_t)s.list[place];
        return;
    }

    // a long head: weights by distance in a histogram, borders and the draw are found in it
    const bool counted = d.k < n;
    for (int i = threadIdx.x; i < kBins; i += NT) {
        s.mass[i] = ready ? cut.mass[(size_t)blockIdx.x * kBins + i] : 0;
        s.classes[i] = ready ? cut.classes[(size_t)blockIdx.x * kBins + i] : 0;
    }
    __syncthreads();
    u64 above_m = ready && threadIdx.x == 0 ? cut.above[blockIdx.x] : 0;
    if (!ready) above_m = add_masses([&](auto f) { r.template each<1>(f); }, W, d, n, counted, s);
    __syncthreads();
    u64 kept = 0;
    for (int i = threadIdx.x; i < kBins; i += NT) kept += s.mass[i];
    kept = block_all<NT>(kept, plus64, s.red64);
    int cls = -1;
    if (counted) {
        int b = kBins - 1;
        uint32_t classes = 0;
        find_bin<NT, uint32_t>(s.classes, (uint32_t)d.k, b, classes, s.red32, s.answer);
        u64 before = 0;
        for (int i = threadIdx.x; i < b; i += NT) before += s.mass[i];
        before = block_all<NT>(before, plus64, s.red64);
        kept = min(kept, resolve<T, NT>(r, row, n, kmax, W, true, (u64)d.k, b, before, classes, &s).mass);
    }
    // what top-p and min-p leave: between `low` and `kept`, the border's bin apart
    u64 need_p = 0, before_p = 0, low = kept;
    int bin_p = -1;
    if (d.with_p) {
        need_p = max(share_up(fmaxf(d.top_p, 0.f), kept), (u64)1);
        find_bin<NT, u64>(s.mass, need_p, bin_p, before_p, s.red64, s.answer);
        low = before_p + 1;
        bin_p = max(bin_p, 0);
        kept = min(kept, before_p + s.mass[bin_p]);
    }
    if (d.with_m) {
        const u64 best = max(block_all<NT>(above_m, plus64, s.red64), W.weight(0.0));        // the best class stays
        low = min(low, best);
        kept = min(kept, best);
    }
    // so the draw ends in one of few bins, mostly one: its classes and the border's are gathered in one pass over the row
    const u64 need_low = share_down(d.u, low) + 1, need_high = share_down(d.u, kept) + 1;
    int bin_d = 0, bin_e = 0;
    u64 before_d = 0, skip;
    find_bin<NT, u64>(s.mass, need_low, bin_d, before_d, s.red64, s.answer);
    find_bin<NT, u64>(s.mass, need_high, bin_e, skip, s.red64, s.answer);
    if (threadIdx.x == 0) s.n = s.n2 = 0;
    __syncthreads();
    float p0 = 1.f, p1 = 0.f, d0, d1;                // (nothing lies between 1 and 0)
    if (d.with_p) W.bin_range(bin_p, bin_p, p0, p1);
    W.bin_range(bin_d, bin_e, d0, d1);
    r.template raw<8>([&](const u32x4 &v, int i) {
        float x[r.N];
        Pack<T>::expand(v, x);
        uint32_t hits = 0;
#pragma unroll
        for (int j = 0; j < r.N; ++j) hits |= ((x[j] >= p0) & (x[j] <= p1)) | ((x[j] >= d0) & (x[j] <= d1)) ? 1u << j : 0;
        if (!hits) return;                           // one place in the list is asked for a vector, not for each class
        int at = atomicAdd(&s.n, __popc(hits));
        for (; hits; hits &= hits - 1, ++at) {
            const int j = __ffs(hits) - 1;
            if (at < kList) s.list[at] = (u64)(kmax - order_key(pick<T>(v, j))) << 32 | (uint32_t)(i * r.N + j);
        }
    });
    __syncthreads();
    // what was gathered, by its bin proper: the border's to the front of the list, the draw's behind it
    constexpr int HALF = kList / 2, PER = kList / NT;
    const int gathered = s.n;
    bool fits = gathered <= kList;
    u64 entry[PER];
    int at_p[PER], at_d[PER];
    if (fits) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = (int)threadIdx.x + j * NT;
            entry[j] = i < gathered ? s.list[i] : 0;
        }
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool is = (int)threadIdx.x + j * NT < gathered && (uint32_t)entry[j] < (uint32_t)n;          // (behind the row's end: -inf)
            const int b = is ? W.bin(W.octaves(key_value(kmax - (uint32_t)(entry[j] >> 32)))) : -2;
            at_p[j] = b == bin_p ? atomicAdd(&s.n, 1) : HALF;
            at_d[j] = b >= bin_d && b <= bin_e ? atomicAdd(&s.n2, 1) : HALF;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (at_p[j] < HALF) s.list[at_p[j]] = entry[j];
            if (at_d[j] < HALF) s.list[HALF + at_d[j]] = entry[j];
        }
        __syncthreads();
        fits = s.n <= HALF && s.n2 <= HALF;
    }
    const int in_p = s.n, in_d = s.n2;
    if (d.with_p)
        kept = min(kept, fits ? reach<NT>(s.list, in_p, kmax, W, false, need_p, before_p, 0, cls, s)
                              : resolve<T, NT>(r, row, n, kmax, W, false, need_p, bin_p, before_p, 0, &s).mass);
    const u64 need = share_down(d.u, kept) + 1;
    if (fits)
        reach<NT>(s.list + HALF, in_d, kmax, W, false, need, before_d, 0, cls, s);
    else {
        find_bin<NT, u64>(s.mass, need, bin_d, before_d, s.red64, s.answer);
        cls = resolve<T, NT>(r, row, n, kmax, W, false, need, bin_d, before_d, 0, &s).cls;
    }
    if (threadIdx.x == 0) a.labels[blockIdx.x] = cls;
}

template <typename T, int NE>
__global__ __launch_bounds__(256) void sample_small_kernel(const T *__restrict__ logits, long long stride, int rows, int n, int S, SampleArgs a)
{
    const int row = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    u64 v[NE];
    const uint32_t kmax = load_wave<T, NE>(logits + (size_t)row * stride, n, v);
    const Draw d(a, row, n);
    if (kmax == kKeyNan || kmax <= kKeyMinusInf || d.greedy) {
        if (lane == 0) a.labels[row] = kmax == kKeyNan || kmax <= kKeyMinusInf ? -1 : (long long)(uint32_t)v[0];
        return;
    }
    const bool infinite = key_value(kmax) == __builtin_inff();          // +inf takes all the weight
    const Weigher W(infinite ? 0.f : key_value(kmax), d.temperature, S);
    u64 w[NE];
    bool in_m[NE];
#pragma unroll
    for (int j = 0; j < NE; ++j) {
        const bool is = lane * NE + j < d.k;
        float x = key_value(kmax - (uint32_t)(v[j] >> 32));
        if (infinite) x = x == __builtin_inff() ? 0.f : -__builtin_inff();
        const double y = is ? W.octaves(x) : 0.0;
        w[j] = is ? W.weight(y) : 0;
        in_m[j] = !d.with_m || lane * NE + j == 0 || y >= d.least;
    }
    const int place = draw_from_head<NE>(
        w, in_m, lane * NE, d,
        [&](u64 x, u64 &total) {
            u64 inc = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 up = __shfl_up(inc, o);
                if (lane >= o) inc += up;
            }
            total = __shfl(inc, 63);
            return inc - x;
        },
        [&](u64 x) { return wave_all(x, plus64); });
    if (place >= 0) {
#pragma unroll
        for (int j = 0; j < NE; ++j)
            if (place == lane * NE + j) a.labels[row] = (long long)(uint32_t)v[j];
    }
}

inline int weight_bits(int classes)
{
    int bits = 0;
    while ((1ll << bits) < classes) ++bits;
    return bits > 11 ? 62 - bits : 51;
}

template <typename F>
int by_type(int dtype, F f)
{
    switch (dtype) {
    case MH_F32: return f((float *)nullptr);
    case MH_F16: return f((f16 *)nullptr);
    default: return f((bf16 *)nullptr);
    }
}
// The kernel for rows of n classes: one wave a row up to kSmall, then a workgroup; the row stays in LDS up to kHeld bytes.
constexpr int kHeld = 64 * 1024;
template <typename T, typename SMALL, typename LARGE>
int by_classes(int n, SMALL small, LARGE large)
{
    if (n <= 64) return small(std::integral_constant<int, 1>());
    if (n <= 128) return small(std::integral_constant<int, 2>());
    if (n <= kSmall) return small(std::integral_constant<int, 4>());
    const size_t bytes = align_up((size_t)n * sizeof(T), 16);
    if (bytes <= 16 * 1024) return large(std::integral_constant<int, 256>(), std::true_type(), bytes);
    if (bytes <= kHeld) return large(std::integral_constant<int, 512>(), std::true_type(), bytes);
    return large(std::integral_constant<int, 512>(), std::false_type(), 0);
}
template <auto Kern, typename... Args>
int launch_row_kernel(unsigned rows, int threads, size_t lds, hipStream_t st, const char *name, Args... args)
{
    if (lds > 0) {               // more than 64 KiB of LDS a workgroup has to be asked for, once a device
        static bool asked[64] = {};
        int dev = 0;
        const hipError_t e = hipGetDevice(&dev);
        if (e != hipSuccess) {
            set_last_error("hipGetDevice", e);
            return (int)e;
        }
        if (dev >= 64 || !asked[dev]) {
            const hipError_t f = hipFuncSetAttribute(reinterpret_cast<const void *>(Kern), hipFuncAttributeMaxDynamicSharedMemorySize, kHeld);
            if (f != hipSuccess) {
                set_last_error("hipFuncSetAttribute", f);
                return (int)f;
            }
            if (dev < 64) asked[dev] = true;
        }
    }
    hipLaunchKernelGGL(Kern, dim3(rows), dim3(threads), lds, st, args...);
    return check_launch(name);
}
constexpr double kColdest = 1e-30, kHottest = 1e30;       // log2(e) / T is a normal 32-bit number between
inline bool type_ok(int dtype) { return dtype == MH_F32 || dtype == MH_F16 || dtype == MH_BF16; }
// (a launch has fewer than 2^32 work-items: 512 for every row and segment, at the most)
inline bool rows_ok(int rows, int classes) { return rows >= 0 && classes > 0 && (long long)rows * (((long long)classes + kSegment - 1) / kSegment) < (1 << 23); }
inline int segments(int classes) { return (int)(((long long)classes + kSegment - 1) / kSegment); }

}  // namespace ld
}  // namespace mh

using namespace mh;
using namespace mh::ld;

extern "C" {

int mh_top_logits_max_k(void) { return kMaxTop; }

int mh_top_logits(const void *logits, int dtype, long long row_stride, int rows, int classes, int k, double temperature, void *values, int *indices,
                  float *rest, void *stream)
{
    MH_REQUIRE(type_ok(dtype) && rows_ok(rows, classes) && k > 0 && k <= classes && k <= kMaxTop && temperature >= kColdest && temperature <= kHottest);
    if (rows == 0) return MH_OK;
    MH_REQUIRE(logits && values && indices && rest);
    return by_type(dtype, [&](auto *tag) {
        typedef std::remove_pointer_t<decltype(tag)> T;
        const T *x = static_cast<const T *>(logits);
        T *v = static_cast<T *>(values);
        hipStream_t st = as_stream(stream);
        return by_classes<T>(
            classes,
            [&](auto ne) {
                hipLaunchKernelGGL((top_logits_small_kernel<T, ne.value>), dim3(((unsigned)rows + 3) / 4), dim3(256), 0, st, x, row_stride, rows,
                                   classes, k, Scale(temperature), v, indices, rest);
                return check_launch("top_logits_small_kernel");
            },
            [&](auto nt, auto held, size_t lds) {
                return launch_row_kernel<top_logits_kernel<T, nt.value, held.value>>((unsigned)rows, nt.value, lds, st, "top_logits_kernel", x,
                                                                                     row_stride, classes, k, Scale(temperature), v, indices, rest);
            });
    });
}

size_t mh_distill_ws_bytes(int rows, int classes)
{
    if (rows <= 0 || classes <= 0 || segments(classes) == 1) return 0;
    return (size_t)rows * segments(classes) * kPart * sizeof(float);
}

int mh_distill_stats(void) { return kStats; }

int mh_distill_fwd(const void *logits, int dtype, long long row_stride, int rows, int classes, const void *t_values, int t_dtype,
                   const void *t_indices, int t_wide, const float *t_rest, int k, double temperature, double factor, const float *row_weight, int mean,
                   float *stats, float *row_loss, float *total, float *divided_by, void *grad, void *workspace, size_t ws_bytes,
                   void *stream)
{
    MH_REQUIRE(type_ok(dtype) && type_ok(t_dtype) && rows_ok(rows, classes) && k > 0 && k <= kMaxTop && temperature >= kColdest && temperature <= kHottest);
    MH_REQUIRE(ws_bytes >= mh_distill_ws_bytes(rows, classes) && (total || !grad) && (!total || divided_by));
    hipStream_t st = as_stream(stream);
    const float divisor = !mean ? 1.f : row_weight ? 0.f : (float)std::max(rows, 1);          // 0: *divided_by has it
    if (total && divisor == 0.f) {
        hipLaunchKernelGGL(distill_weight_kernel, dim3(1), dim3(1024), 0, st, row_weight, rows, divided_by);
        const int e = check_launch("distill_weight_kernel");
        if (e) return e;
    }
    if (rows > 0) {
        MH_REQUIRE(logits && t_values && t_indices && stats && row_loss && (reinterpret_cast<uintptr_t>(stats) & 7) == 0);
        const int nseg = segments(classes);
        MH_REQUIRE((nseg == 1 || workspace) && (nseg == 1 || !grad));
        const Teacher t{t_values, t_dtype, t_indices, t_wide, t_rest, k};
        const Scale scale(temperature, factor);
        int rc = by_type(dtype, [&](auto *tag) {
            typedef std::remove_pointer_t<decltype(tag)> T;
            const T *x = static_cast<const T *>(logits);
            T *g = static_cast<T *>(grad);
            float *parts = static_cast<float *>(workspace);
            const size_t record = 3 * (size_t)k * 4, member = t_rest ? (size_t)(std::min(classes, kSegment) + 31) / 32 * 4 : 0;
            const unsigned blocks = (unsigned)nseg * (unsigned)rows;
            auto go = [&](auto rest, auto with_grad) {
                hipLaunchKernelGGL((distill_fwd_kernel<T, 256, decltype(rest)::value, decltype(with_grad)::value>), dim3(blocks), dim3(256),
                                   record + member, st, x, row_stride, classes, t, scale, row_weight, stats, row_loss, parts, nseg, divisor,
                                   (const float *)divided_by, g);
                return check_launch("distill_fwd_kernel");
            };
            auto with_rest = [&](auto rest) { return g ? go(rest, std::true_type()) : go(rest, std::false_type()); };
            if (classes <= kShort) {
                hipLaunchKernelGGL((distill_short_kernel<T, 256>), dim3((unsigned)rows), dim3(256), record, st, x, row_stride, classes, t, scale, row_weight,
                                   stats, row_loss, divisor, (const float *)divided_by, g);
                return check_launch("distill_short_kernel");
            }
            int e = t_rest ? with_rest(std::true_type()) : with_rest(std::false_type());
            if (e || nseg == 1) return e;
            hipLaunchKernelGGL((distill_join_kernel<T>), dim3((unsigned)rows), dim3(64), record, st, x, row_stride, classes, t, scale, row_weight, stats,
                               row_loss, parts, nseg);
            return check_launch("distill_join_kernel");
        });
        if (rc) return rc;
    }
    if (!total) return MH_OK;
    hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(1024), 0, st, row_loss, rows, divisor, total, divided_by);
    return check_launch("distill_total_kernel");
}

int mh_capture_id(void *stream, unsigned long long *id)
{
    MH_REQUIRE(id);
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long capture = 0;
    const hipError_t e = hipStreamGetCaptureInfo(as_stream(stream), &status, &capture);
    if (e != hipSuccess) {
        set_last_error("hipStreamGetCaptureInfo", e);
        return (int)e;
    }
    *id = status == hipStreamCaptureStatusNone ? 0 : capture;
    return MH_OK;
}

int mh_distill_grad_in_fwd(int classes) { return classes > 0 && segments(classes) == 1; }

int mh_distill_bwd(const void *logits, int dtype, long long row_stride, int rows, int classes, const void *t_values, int t_dtype,
                   const void *t_indices, int t_wide, const float *t_rest, int k, double temperature, double factor, const float *row_weight,
                   const float *stats, const float *divided_by, const float *upstream, int upstream_rows, int written, void *grad, void *stream)
{
    MH_REQUIRE(type_ok(dtype) && type_ok(t_dtype) && rows_ok(rows, classes) && k > 0 && k <= kMaxTop && temperature >= kColdest && temperature <= kHottest);
    if (rows == 0) return MH_OK;
    const int nseg = segments(classes);
    MH_REQUIRE(logits && t_values && t_indices && stats && (reinterpret_cast<uintptr_t>(stats) & 7) == 0 && upstream && grad && !(written && upstream_rows));
    const Teacher t{t_values, t_dtype, t_indices, t_wide, t_rest, k};
    return by_type(dtype, [&](auto *tag) {
        typedef std::remove_pointer_t<decltype(tag)> T;
        hipLaunchKernelGGL((distill_bwd_kernel<T, 256>), dim3((unsigned)nseg * (unsigned)rows), dim3(256), 3 * (size_t)k * 4, as_stream(stream),
                           static_cast<const T *>(logits), row_stride, classes, t, Scale(temperature, factor), row_weight, stats, divided_by, upstream, upstream_rows,
                           written, static_cast<T *>(grad), nseg);
        return check_launch("distill_bwd_kernel");
    });
}

size_t mh_sample_ws_bytes(int rows, int classes)
{
    const int nseg = row_cut(rows, classes).nseg;
    return nseg ? (size_t)rows * (kBins * 12 + 8 + (size_t)nseg * 4) : 0;
}

int mh_sample_labels(const void *logits, int dtype, long long row_stride, int rows, int classes, const float *u, const float *temperature,
                     const int *top_k, const float *top_p, const float *min_p, float temperature_all, int top_k_all, float top_p_all,
                     float min_p_all, long long *labels, void *workspace, size_t ws_bytes, void *stream)
{
    MH_REQUIRE(type_ok(dtype) && rows_ok(rows, classes));
    if (rows == 0) return MH_OK;
    MH_REQUIRE(logits && u && labels);
    const SampleArgs a{u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, labels};
    Cut cut{0, 0, nullptr, nullptr, nullptr, nullptr};
    // (no workspace: the rows' own workgroups; rows that are known to be drawn from a short head have no histogram)
    const bool may_be_long = (temperature || temperature_all > 0.f) && (top_k || top_k_all <= 0 || top_k_all > kMaxTop);
    const RowCut parts = row_cut(rows, classes);
    if (may_be_long && workspace && parts.nseg > 0) {
        MH_REQUIRE(ws_bytes >= mh_sample_ws_bytes(rows, classes) && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0);
        cut.nseg = parts.nseg;
        cut.length = parts.length;
        cut.mass = static_cast<u64 *>(workspace);
        cut.above = cut.mass + (size_t)rows * kBins;
        cut.classes = reinterpret_cast<uint32_t *>(cut.above + rows);
        cut.top = cut.classes + (size_t)rows * kBins;
    }
    return by_type(dtype, [&](auto *tag) {
        typedef std::remove_pointer_t<decltype(tag)> T;
        const T *x = static_cast<const T *>(logits);
        const int S = weight_bits(classes);
        hipStream_t st = as_stream(stream);
        if (cut.nseg > 0) {
            const dim3 grid((unsigned)rows * (unsigned)cut.nseg);
            hipLaunchKernelGGL((sample_top_kernel<T>), grid, dim3(256), 0, st, x, row_stride, classes, cut);
            int e = check_launch("sample_top_kernel");
            if (e) return e;
            hipLaunchKernelGGL((sample_mass_kernel<T, 512>), grid, dim3(512), 0, st, x, row_stride, classes, S, a, cut);
            e = check_launch("sample_mass_kernel");
            if (e) return e;
            return launch_row_kernel<sample_kernel<T, 512, false>>((unsigned)rows, 512, 0, st, "sample_kernel", x, row_stride, classes, S, a, cut);
        }
        return by_classes<T>(
            classes,
            [&](auto ne) {
                hipLaunchKernelGGL((sample_small_kernel<T, ne.value>), dim3(((unsigned)rows + 3) / 4), dim3(256), 0, st, x, row_stride, rows, classes,
                                   S, a);
                return check_launch("sample_small_kernel");
            },
            [&](auto nt, auto held, size_t lds) {
                return launch_row_kernel<sample_kernel<T, nt.value, held.value>>((unsigned)rows, nt.value, lds, st, "sample_kernel", x, row_stride,
                                                                                 classes, S, a, cut);
            });
    });
}

}  // extern "C"
