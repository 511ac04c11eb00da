// sm_100a kernels of the operators on rows of raw logits (see logits.h):
// sampling, the best log-probs of a row, and the distillation loss.
#include "logits.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <mutex>
#include <tuple>
#include <vector>

#include "dbs_engine.h"

namespace cg = cooperative_groups;

namespace dbs_logits {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Threads of the kernels that give a row to a cluster, their `kTeam`: lists are
// bound by their barriers, searches and sums over a slice by arithmetic. One
// row of 32000 bf16, top_k 50: 9.8 us with 256, 11.2 us with 512; one of
// 128256, top_p alone: 38.3 us with 256, 37.7 us with 512.
constexpr int kListTeam = 256;
constexpr int kMassTeam = 512;
constexpr int kMostWarps = kMassTeam / 32;
constexpr int kMaxCluster = 16;
constexpr int kBins = 2048;
constexpr int kSampleList = 512;   // longest top-k that goes through a candidate list
constexpr uint32_t kAll = 0xFFFFFFFFu;

// ---------------------------------------------------------------------------
// Element types. A vector is 16 bytes; `Elem<E>::max` is the elementwise
// maximum of two vectors, which drops NaN for the other operand.
// ---------------------------------------------------------------------------
template <class E>
struct Elem;

template <>
struct Elem<float> {
    static constexpr int kVec = 4;
    static constexpr int kKeyShift = 0;
    static constexpr uint32_t kNegInf = 0xFF800000u;   // two packed values for the 16-bit types
    __device__ static float widen(float v) { return v; }
    __device__ static float narrow(float v) { return v; }
    __device__ static void unpack(const uint4& v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
    __device__ static uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
    __device__ static uint32_t max1(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
};

template <>
struct Elem<__half> {
    static constexpr int kVec = 8;
    static constexpr int kKeyShift = 13;   // a widened half has 13 zero low bits
    static constexpr uint32_t kNegInf = 0xFC00FC00u;
    __device__ static float widen(__half v) { return __half2float(v); }
    __device__ static __half narrow(float v) { return __float2half_rn(v); }
    __device__ static void unpack(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
    __device__ static uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static uint32_t max1(uint32_t a, uint32_t b) {
        const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

template <>
struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static constexpr int kKeyShift = 16;
    static constexpr uint32_t kNegInf = 0xFF80FF80u;
    __device__ static float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
    __device__ static __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
    __device__ static void unpack(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    __device__ static uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ static uint32_t max1(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r =
            __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

template <class E>
__device__ __forceinline__ uint4 vmax(const uint4& a, const uint4& b) {
    return make_uint4(Elem<E>::max1(a.x, b.x), Elem<E>::max1(a.y, b.y), Elem<E>::max1(a.z, b.z),
                      Elem<E>::max1(a.w, b.w));
}

template <class E>
__device__ __forceinline__ uint4 vneg_inf() {
    return make_uint4(Elem<E>::kNegInf, Elem<E>::kNegInf, Elem<E>::kNegInf, Elem<E>::kNegInf);
}

__device__ __forceinline__ uint4 ldg_once(const uint4* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "l"(p));
    return r;
}

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

// Two floats in one register pair: sm_100a multiplies or adds both in one
// instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t&>(r))
        : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Monotone map of a float to an unsigned key (-0 as +0); the 16-bit types'
// widened values differ in the bits above kKeyShift only.
__device__ __forceinline__ uint32_t ord(float f) {
    const uint32_t u = __float_as_uint(__fadd_rn(f, 0.0f));
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float unord(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
template <class E>
__device__ __forceinline__ uint32_t key_of(float f) {
    return ord(f) >> Elem<E>::kKeyShift;
}
template <class E>
__device__ __forceinline__ float value_of(uint32_t key) {
    const uint32_t top = key << Elem<E>::kKeyShift;
    // a negative value's key is complemented, its zero low bits included
    return (top & 0x80000000u) ? unord(top) : unord(top | ((1u << Elem<E>::kKeyShift) - 1u));
}

// ---------------------------------------------------------------------------
// Block reductions. `scratch` holds a value per warp; every thread gets the
// result, summed in one order.
// ---------------------------------------------------------------------------
template <int kTeam, class T, class Op>
__device__ __forceinline__ T block_reduce(T v, Op op, T* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kTeam / 32; ++w) v = op(v, scratch[w]);
    __syncthreads();
    return v;
}
struct Add {
    template <class T>
    __device__ T operator()(T a, T b) const { return a + b; }
};
struct Max {
    template <class T>
    __device__ T operator()(T a, T b) const { return a > b ? a : b; }
};
struct Min {
    template <class T>
    __device__ T operator()(T a, T b) const { return a < b ? a : b; }
};

template <class T>
__device__ __forceinline__ T shuffle_up(T v, int o) { return __shfl_up_sync(kAll, v, o); }
__device__ __forceinline__ unsigned __int128 shuffle_up(unsigned __int128 v, int o) {
    const uint64_t high = __shfl_up_sync(kAll, static_cast<uint64_t>(v >> 64), o);
    return static_cast<unsigned __int128>(high) << 64 | __shfl_up_sync(kAll, static_cast<uint64_t>(v), o);
}

// Sum of the values of the threads before this one, and (`all`) of all.
template <int kTeam, class T>
__device__ __forceinline__ T block_before(T v, T* scratch, T* all = nullptr) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T up = shuffle_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    T base = T(0), total = T(0);
#pragma unroll
    for (int w = 0; w < kTeam / 32; ++w) {
        const T of = scratch[w];
        base += w < warp ? of : T(0);
        total += of;
    }
    __syncthreads();
    if (all) *all = total;
    T excl = shuffle_up(incl, 1);
    if (lane == 0) excl = T(0);
    return base + excl;
}

__device__ __forceinline__ void cluster_sync(int size) {
    if (size > 1) {
        cg::this_cluster().sync();
    } else {
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Slices. Positions count from the 16-byte boundary at or before the row's
// first element (`phase` elements ahead of it); CTA c of the cluster holds
// positions [c*S, (c+1)*S) in `buf`, and what lies outside the row is -inf.
// ---------------------------------------------------------------------------
struct Slice {
    int nv;      // vectors in buf
    int first;   // token of buf's element 0 (negative where the row starts later)
};

// Loads the slice and adds it to the elementwise maximum `acc`. kClean: NaN
// is stored as -inf.
template <int kTeam, class E, bool kClean>
__device__ __forceinline__ Slice load_slice(const E* row, int V, int S, int c, uint4* buf, uint4& acc) {
    constexpr int kVec = Elem<E>::kVec;
    constexpr int kBatch = 8;
    const int phase = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(E));
    const int a0 = c * S;
    const int len = max(0, min(S, V + phase - a0));
    const int nv = (len + kVec - 1) / kVec;
    const int v0 = (a0 == 0 && phase > 0) ? 1 : 0;
    const int v1 = len / kVec;
    const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) -
                                                      static_cast<uintptr_t>(phase) * sizeof(E)) + a0 / kVec;
    const uint4 none = vneg_inf<E>();
    for (int base = v0 + static_cast<int>(threadIdx.x); base < v1; base += kBatch * kTeam) {
        uint4 r[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int v = base + i * kTeam;
            r[i] = v < v1 ? ldg_once(src + v) : none;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int v = base + i * kTeam;
            if (kClean) r[i] = vmax<E>(r[i], none);
            acc = vmax<E>(acc, r[i]);
            if (v < v1) buf[v] = r[i];
        }
    }
    // the row's ragged ends, element by element
    int edge = -1;
    if (threadIdx.x == 0 && v0 == 1 && nv > 0) edge = 0;
    if (threadIdx.x == 32 && v1 < nv && !(v0 == 1 && v1 == 0)) edge = v1;
    if (edge >= 0) {
        float f[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const int i = a0 + edge * kVec + e - phase;
            f[e] = (i >= 0 && i < V) ? Elem<E>::widen(row[i]) : neg_inf();
        }
        uint4 r = Elem<E>::pack(f);
        if (kClean) r = vmax<E>(r, none);
        acc = vmax<E>(acc, r);
        buf[edge] = r;
    }
    return Slice{nv, a0 - phase};
}

template <class E>
__device__ __forceinline__ float lanes_max(const uint4& v) {
    float f[Elem<E>::kVec];
    Elem<E>::unpack(v, f);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < Elem<E>::kVec; ++i) m = fmaxf(m, f[i]);
    return m;
}

// Descending sort of n keys in shared memory: a bitonic network whose runs
// all have the same direction, so n need not be a power of two. Steps of up to
// 32 places keep a warp within its own 64 keys, and wait for the warp alone.
template <int kT>
__device__ void sort_by(uint64_t* a, int n) {
    int n2 = 1;
    while (n2 < n) n2 <<= 1;
    const int half = n2 >> 1;
    __syncthreads();
    for (int size = 2; size <= n2; size <<= 1) {
        for (int st = size >> 1; st > 0; st >>= 1) {
            for (int p = threadIdx.x; p < half; p += kT) {
                const int i = ((p & ~(st - 1)) << 1) | (p & (st - 1));
                // the first step of a size compares mirrored places
                const int j = st == (size >> 1) ? (i ^ (size - 1)) : i + st;
                if (j < n) {
                    const uint64_t x = a[i], y = a[j];
                    if (x < y) {
                        a[i] = y;
                        a[j] = x;
                    }
                }
            }
            const int next = st > 1 ? st >> 1 : size;
            if (st > 32 || next > 32)
                __syncthreads();
            else
                __syncwarp();
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint64_t entry(float x, int token) {
    return (static_cast<uint64_t>(ord(x)) << 32) | static_cast<uint64_t>(~static_cast<uint32_t>(token));
}
__device__ __forceinline__ float entry_value(uint64_t e) { return unord(static_cast<uint32_t>(e >> 32)); }
__device__ __forceinline__ int entry_token(uint64_t e) {
    return static_cast<int>(~static_cast<uint32_t>(e & 0xFFFFFFFFu));
}

// ---------------------------------------------------------------------------
// What the sampling and top-list kernels keep in shared memory beside the
// slice and the two lists.
// ---------------------------------------------------------------------------
struct Packet {        // one CTA's share of what the cluster adds up
    double sum;
    float best;
    float tau;
    int index;
};
struct Shared {
    Packet box[kMaxCluster];       // written by every CTA of the cluster
    int counts[kMaxCluster];
    double masses[kMaxCluster];
    int ties[kMaxCluster];
    double d8[kMostWarps];
    unsigned __int128 u16[kMostWarps];
    float f8[kMostWarps];
    int i8[kMostWarps];
    double range_mass[kMostWarps];
    int range_ties[kMostWarps];
    __align__(16) int steps[128];
    int listed;
    int found_bin;
    unsigned __int128 found_above;
    unsigned __int128 totals[kMaxCluster];
};

struct Team {      // a CTA's place in its cluster
    int size;
    int rank;
    __device__ Team() {
        auto c = cg::this_cluster();
        size = static_cast<int>(c.num_blocks());
        rank = static_cast<int>(c.block_rank());
    }
    // Gives `value` to every CTA of the cluster, at its own place.
    template <class T>
    __device__ void tell(T* place, const T& value) const {
        if (static_cast<int>(threadIdx.x) < size)
            *cg::this_cluster().map_shared_rank(place + rank, threadIdx.x) = value;
    }
    template <class T>
    __device__ const T* of(const T* place, int other) const {
        return cg::this_cluster().map_shared_rank(const_cast<T*>(place), other);
    }
};

// 2^(d c / 32) in 64 bits, relative error below 2e-12: 2^(n/32 + r/32) with n
// the whole number nearest to d c (within -2^15 and 2^15), a table of 2^(j/32)
// (an entry per lane) and the Taylor polynomial of 2^(r/32) to the fourth
// power: what it leaves out is at most (ln 2 / 64)^5 / 120 = 1.3e-12. All 32
// lanes of a warp call it together. `up` octaves are added.
__device__ __forceinline__ double exp_table() { return exp2(static_cast<double>(threadIdx.x & 31) * 0.03125); }
__device__ __forceinline__ double exp_by(double d, double c, int n, double tab, int up = 0) {
    constexpr double kL = 0.021660849392498290;   // ln 2 / 32
    const double nd = __hiloint2double(0x43300000, n ^ static_cast<int>(0x80000000)) - 4503601774854144.0;
    const double r = fma(d, c, -nd);
    double p = fma(r, kL * kL * kL * kL / 24.0, kL * kL * kL / 6.0);
    p = fma(r, p, kL * kL / 2.0);
    p = fma(r, p, kL);
    p = fma(r, p, 1.0);
    p *= __shfl_sync(kAll, tab, n & 31);
    return __hiloint2double(__double2hiint(p) + (((n >> 5) + up) << 20), __double2loint(p));
}

// ---------------------------------------------------------------------------
// Weights of sampling: exp((x - m) / T) in 64 bits, because tokens have to be
// the ones that exact sums give: with V borders between tokens, sums in 32
// bits would pick another token about once in a hundred flat rows.
// ---------------------------------------------------------------------------
struct Weights {
    float mf;
    float cf;
    // The table's step goes by (x s - m s) (c / s): with s = 1/2 because x - m
    // itself can overflow in 32 bits, with 2^99 where T is so small that c does.
    float s, ms, cs;
    double m;
    double c;
    double tab;    // 2^(lane/32)
    // ordinary: the temperature is known to be at least 1e-36
    __device__ Weights(float best, float temperature, bool ordinary) {
        mf = best;
        m = static_cast<double>(best);
        c = 46.166241308446828384 / static_cast<double>(temperature);   // 32 / ln 2
        cf = static_cast<float>(c);
        const bool tiny = !ordinary && temperature < 1.0e-36f;
        s = tiny ? 6.338253e29f : 0.5f;
        // x <= m: where m s is below all floats, x s - m s stays negative
        ms = fmaxf(s * best, -FLT_MAX);
        cs = static_cast<float>(c * (tiny ? 1.5777218104420236e-30 : 2.0));
        tab = exp_table();
    }
    // All 32 lanes of the warp call it together. `up`: octaves by which a weight
    // other than the best one's is taken up.
    __device__ __forceinline__ double operator()(float x, int up = 0) const {
        // 0 * inf and inf - inf come out as NaN, which fmaxf drops
        const float t = fmaxf(fmaf(x, s, -ms) * cs, -40000.0f);
        const int n = __float_as_int(t + 12582912.0f) - 0x4B400000;
        const double p = exp_by(static_cast<double>(x) - m, c, n, tab, up);
        return x == mf ? 1.0 : (n < -32686 ? 0.0 : p);   // exp(-708) and below count as nothing
    }
    // For sums by a finite maximum and a temperature in [1e-36, 1e30]: exp(-690)
    // stands for all that is less (`low` = m - 690 T), which no sum notices.
    __device__ __forceinline__ double term(float x, float low) const {
        const float v = fmaxf(x, low);
        const int bits = __float_as_int(fmaf(v - mf, cf, 12582912.0f));   // 0x4B400000 + n
        const double nd = __hiloint2double(0x43300000, bits + static_cast<int>(0x80000000u - 0x4B400000u)) -
                          4503601774854144.0;
        const double r = fma(static_cast<double>(v) - m, c, -nd);
        constexpr double kL = 0.021660849392498290;   // ln 2 / 32
        double p = fma(r, kL * kL * kL * kL / 24.0, kL * kL * kL / 6.0);
        p = fma(r, p, kL * kL / 2.0);
        p = fma(r, p, kL);
        p = fma(r, p, 1.0);
        p *= __shfl_sync(kAll, tab, bits & 31);
        // n / 32 octaves; what 0x4B400000 adds to the shifted bits is beyond them
        return __hiloint2double(__double2hiint(p) + ((bits << 15) & static_cast<int>(0xFFF00000u)), __double2loint(p));
    }
};

// A weight (or one taken up by some octaves, at most about 1) as a whole number
// of 2^-43: sums of these do not depend on their order, and 2^20 of them stay
// below 2^63.
__device__ __forceinline__ unsigned long long fixed(double w) {
    return static_cast<unsigned long long>(__double_as_longlong(w + 512.0) - 0x4080000000000000LL);
}

// Adds a fixed() weight to a bin in shared memory as three limbs of 15 bits,
// kBins apart: 32-bit additions that nothing waits for (a 64-bit one is a loop
// of compare-and-swap), and a slice's elements, fewer than 2^17, do not overflow a limb.
template <bool kMass>
__device__ __forceinline__ void add_limbs(uint32_t* bin, unsigned long long w) {
    if (!kMass) {
        atomicAdd(bin, static_cast<uint32_t>(w));
        return;
    }
    const uint32_t low = static_cast<uint32_t>(w) & 0x7FFFu, mid = static_cast<uint32_t>(w >> 15) & 0x7FFFu,
                   high = static_cast<uint32_t>(w >> 30);
    if (low) atomicAdd(bin, low);
    if (mid) atomicAdd(bin + kBins, mid);
    if (high) atomicAdd(bin + 2 * kBins, high);
}

// What a search adds up: elements, or weights as whole numbers of 2^-89, so
// that weights 46 octaves below the best one still have 43 bits (a target p *
// mass may lie on the border between two equal best tokens but for the mass of
// all the small ones).
template <bool kMass>
struct SumOf {
    using T = unsigned long long;
};
template <>
struct SumOf<true> {
    using T = unsigned __int128;
};
constexpr int kOctaves = 46;
__device__ __forceinline__ double real(unsigned long long v) { return static_cast<double>(v); }
__device__ __forceinline__ double real(unsigned __int128 v) {   // times 2^-89; rounded twice, but never out of order
    return fma(static_cast<double>(static_cast<uint64_t>(v >> 64)), 0x1p-25, static_cast<double>(static_cast<uint64_t>(v)) * 0x1p-89);
}

// Where an ordered row is cut: every key above `key` is kept, and of those
// equal to it the first `ties` by index.
struct Cut {
    uint32_t key;
    int ties;
};

// Visits the slice's elements a warp at a time, all lanes together; lanes
// past the end see -inf.
template <int kTeam, class E, class F>
__device__ __forceinline__ void for_elements(const uint4* buf, const Slice& s, F&& f) {
    const int lane = threadIdx.x & 31;
    for (int base = (threadIdx.x >> 5) * 32; base < s.nv; base += kTeam) {
        const int v = base + lane;
        float x[Elem<E>::kVec];
        Elem<E>::unpack(v < s.nv ? buf[v] : vneg_inf<E>(), x);
#pragma unroll
        for (int e = 0; e < Elem<E>::kVec; ++e) f(x[e], v * Elem<E>::kVec + e);
    }
}

// Finds the value at which the descending row reaches `target`: a count of
// elements (kMass false) or a sum of fixed() weights. Elements with keys at or
// below `floor_key` stay out. A round counts or adds up the members of kBins
// bins per CTA, adds the cluster's bins and keeps the bin that reaches the
// target; the first round's bins are equal steps of the value over
// [best - span, best] (a last one holds the rest), later ones equal steps of
// the key, until a bin is one value. Weights are taken up by whole octaves, as
// many as their bin of the first round lies below the best value.
// For kMass, `target` comes in as the share p, and becomes p * (all members'
// mass + extra); where the members fall short of it, ok is false.
// Returns the key reached, and the count or mass above it.
struct Found {
    uint32_t key;
    double above;
    double target;
    double total;
    bool ok;
};

template <int kTeam, class E, bool kMass>
__device__ Found search(const Team& team, Shared& sh, uint32_t* hist, const uint4* buf, const Slice& s,
                        const Weights& weight, float span, uint32_t floor_key, double target, double extra) {
    const float scale = static_cast<float>(kBins - 1) / span;
    const float best = weight.mf;
    int lin = -1;                 // the first round's bin, once known
    uint32_t lo = floor_key + 1, hi = key_of<E>(best);
    int shift = 0;
    using Sum = typename SumOf<kMass>::T;
    Sum above = 0;
    Sum* totals = reinterpret_cast<Sum*>(sh.totals);
    Sum* found_above = reinterpret_cast<Sum*>(&sh.found_above);
    Found out;
    out.total = 0.0;
    // octaves between bins of the first round, in 2^-14, rounded down
    const int bin_octaves =
        kMass ? static_cast<int>(fmin(static_cast<double>(span) / (kBins - 1) * weight.c * 0.03125, 1.0 * kOctaves) * 16384.0) : 0;
    auto octaves = [&](int l) { return min(kOctaves, l * bin_octaves >> 14); };
    // by all lanes of the warp together; what is asked for with a bin of -1 is not used
    auto taken_up = [&](float x, int l) { return kMass ? fixed(weight(x, octaves(l))) : 1ull; };
    auto lin_bin = [&](float x) {
        // also right for infinite operands: inf - inf is NaN, and fminf drops it
        const float b = x == best ? 0.0f : fminf((best - x) * scale, static_cast<float>(kBins - 1));
        return static_cast<int>(b);
    };
    for (int round = 0;; ++round) {
        for (int b = threadIdx.x; b < 3 * kBins; b += kTeam) hist[b] = 0;
        __syncthreads();
        unsigned long long rest = 0;
        const int lane = threadIdx.x & 31;
        for (int base = (threadIdx.x >> 5) * 32; base < s.nv; base += kTeam) {
            constexpr int kVec = Elem<E>::kVec;
            float x[kVec];
            int bin[kVec];    // -1: not a member
            bool any = false;
            Elem<E>::unpack(base + lane < s.nv ? buf[base + lane] : vneg_inf<E>(), x);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const uint32_t k = key_of<E>(x[e]);
                const int l = lin_bin(x[e]);
                bool in = k > floor_key;
                if (round > 0) in = in && l == lin && k >= lo && k <= hi;
                bin[e] = in ? (round == 0 ? l : static_cast<int>((hi - k) >> shift)) : -1;
                any = any || in;
            }
            if (!__any_sync(kAll, any)) continue;
            if (round > 0) {   // one bin of many: few of a vector's elements
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    if (!__any_sync(kAll, bin[e] >= 0)) continue;
                    const unsigned long long w = taken_up(x[e], lin);
                    if (bin[e] >= 0) add_limbs<kMass>(hist + bin[e], w);
                }
                continue;
            }
            unsigned long long w[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) w[e] = taken_up(x[e], bin[e]);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                if (bin[e] < 0) continue;
                if (bin[e] == kBins - 1)
                    rest += w[e];
                else
                    add_limbs<kMass>(hist + bin[e], w[e]);
            }
        }
        if (round == 0) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) rest += __shfl_xor_sync(kAll, rest, o);
            if (lane == 0 && rest) add_limbs<kMass>(hist + kBins - 1, rest);
        }
        cluster_sync(team.size);
        // Each CTA adds up its share of the bins over the cluster (all of them
        // in each would keep the SMs' network busy for microseconds).
        const int share_bins = (kBins + team.size - 1) / team.size;
        const int each = (share_bins + kTeam - 1) / kTeam;
        const int first = team.rank * share_bins + each * static_cast<int>(threadIdx.x);
        const int last = min(min(kBins, (team.rank + 1) * share_bins), first + each);
        constexpr int kEach = kBins / kTeam;
        unsigned long long h[kEach] = {};
#pragma unroll
        for (int q = 0; q < kEach; ++q) {
            if (first + q >= last) break;
            for (int c0 = 0; c0 < team.size; c0 += 8) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {   // the loads of eight CTAs' bins in flight together
                    if (c0 + c >= team.size) continue;
                    const uint32_t* theirs = team.of(hist, c0 + c);
#pragma unroll
                    for (int k = 0; k < (kMass ? 3 : 1); ++k)
                        h[q] += static_cast<unsigned long long>(theirs[k * kBins + first + q]) << (15 * k);
                }
            }
        }
        auto in_bin = [&](int q) {
            return static_cast<Sum>(h[q]) << (kMass ? kOctaves - octaves(round == 0 ? first + q : lin) : 0);
        };
        Sum own = 0;
#pragma unroll
        for (int q = 0; q < kEach; ++q) own += in_bin(q);
        Sum of_share;
        const Sum in_share = block_before<kTeam>(own, reinterpret_cast<Sum*>(sh.u16), &of_share);
        team.tell(totals, of_share);
        cluster_sync(team.size);
        Sum total = 0, before = above + in_share;
        for (int c = 0; c < team.size; ++c) {
            if (c < team.rank) before += totals[c];
            total += totals[c];
        }
        if (round == 0) {
            if (kMass) {
                out.total = real(total) + extra;
                target *= out.total;
            }
            out.target = target;
            out.ok = real(total) >= target && total > 0;
            if (!out.ok) {
                cluster_sync(team.size);
                out.key = floor_key;
                out.above = real(total);
                return out;
            }
        }
        if (real(before) < target && real(before + own) >= target) {
            Sum run = before;
#pragma unroll
            for (int q = 0; q < kEach; ++q) {
                if (first + q >= last) break;
                const bool here = real(run) < target && real(run + in_bin(q)) >= target;
                for (int c = 0; here && c < team.size; ++c) {
                    *cg::this_cluster().map_shared_rank(&sh.found_bin, c) = first + q;
                    *cg::this_cluster().map_shared_rank(found_above, c) = run;
                }
                run += in_bin(q);
            }
        }
        cluster_sync(team.size);
        const int b = sh.found_bin;
        above = *found_above;
        __syncthreads();
        if (round == 0) {
            lin = b;
            // the bin's keys, its ends widened for the rounding of (best - x) * scale
            if (b < kBins - 1 && best < FLT_MAX) {
                const float width = span / static_cast<float>(kBins - 1);
                const float slack = 0.01f * width + 1e-5f * fmaxf(fabsf(best), span);
                if (b > 0) hi = min(hi, key_of<E>(best - static_cast<float>(b) * width + slack));
                lo = max(lo, key_of<E>(best - static_cast<float>(b + 1) * width - slack));
            }
        } else {
            if (shift == 0) {
                out.key = hi - static_cast<uint32_t>(b);
                out.above = real(above);
                return out;
            }
            hi = hi - (static_cast<uint32_t>(b) << shift);
            const uint32_t wide = (1u << shift) - 1u;
            lo = hi - lo > wide ? hi - wide : lo;
        }
        const uint32_t width = hi - lo;
        shift = 0;
        while ((width >> shift) >= static_cast<uint32_t>(kBins)) ++shift;
    }
}

// Appends every element that reaches `low` (and is above -inf) to the CTA's
// list; `listed` counts on where the list is full.
template <int kTeam, class E>
__device__ __forceinline__ void append_from(Shared& sh, const uint4* buf, const Slice& s, float low, uint64_t* list,
                                            int cap) {
    for (int v = threadIdx.x; v < s.nv; v += kTeam) {
        const uint4 r = buf[v];
        if (lanes_max<E>(r) < low) continue;
        float x[Elem<E>::kVec];
        Elem<E>::unpack(r, x);
#pragma unroll
        for (int e = 0; e < Elem<E>::kVec; ++e) {
            if (x[e] >= low && x[e] > neg_inf()) {
                const int at = atomicAdd(&sh.listed, 1);
                if (at < cap) list[at] = entry(x[e], s.first + v * Elem<E>::kVec + e);
            }
        }
    }
}

// The row's best entries, n of them (fewer where fewer are above -inf), in
// the leader's `sorted`, best first; the number of entries there, 0 in the
// other CTAs. box[] holds every CTA's `tau` below which it needs to list
// nothing. Every CTA lists what is at or above the least of these; where ties
// make that too many, the exact cut is searched.
template <int kTeam, class E>
__device__ int gather_best(const Team& team, Shared& sh, const uint4* buf, const Slice& s, float best, int n,
                           uint64_t* list, uint64_t* sorted, int cap, int leader) {
    float tau = sh.box[0].tau;
    for (int c = 1; c < team.size; ++c) tau = fminf(tau, sh.box[c].tau);
    append_from<kTeam, E>(sh, buf, s, tau, list, cap);
    __syncthreads();
    team.tell(sh.counts, sh.listed);
    cluster_sync(team.size);
    int total = 0;
    for (int c = 0; c < team.size; ++c) total += sh.counts[c];
    if (total > cap) {
        // Too many: find the n-th value itself. All of the row's elements
        // above -inf are members, and they are more than n.
        const Weights weight(best, 1.0f, true);
        float low = best;
        for_elements<kTeam, E>(buf, s, [&](float x, int) { low = x > neg_inf() ? fminf(low, x) : low; });
        low = block_reduce<kTeam>(low, Min(), sh.f8);
        cluster_sync(team.size);          // box is read by everybody
        team.tell(sh.box, Packet{0.0, 0.0f, low, 0});
        cluster_sync(team.size);
        for (int c = 0; c < team.size; ++c) low = fminf(low, sh.box[c].tau);
        float span = best - low;
        if (!(span > 0.0f)) span = 1.0f;
        if (!(span < FLT_MAX)) span = FLT_MAX;
        // both lists' space holds the bins: what was listed is listed again below
        const Found f = search<kTeam, E, false>(team, sh, reinterpret_cast<uint32_t*>(list), buf, s, weight, span,
                                         key_of<E>(neg_inf()), static_cast<double>(n), 0.0);
        const int need = n - static_cast<int>(f.above);
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        append_from<kTeam, E>(sh, buf, s, value_of<E>(f.key + 1), list, cap);
        // the first `need` of the equal ones, by index: a stretch of
        // neighbouring vectors per thread
        const int per = (s.nv + kTeam - 1) / kTeam;
        const int begin = min(s.nv, per * static_cast<int>(threadIdx.x)), end = min(s.nv, begin + per);
        int mine = 0;
        for (int v = begin; v < end; ++v) {
            float x[Elem<E>::kVec];
            Elem<E>::unpack(buf[v], x);
#pragma unroll
            for (int e = 0; e < Elem<E>::kVec; ++e) mine += key_of<E>(x[e]) == f.key;
        }
        const int all = block_reduce<kTeam>(mine, Add(), sh.i8);
        int at = block_before<kTeam>(mine, sh.i8);
        team.tell(sh.ties, all);
        cluster_sync(team.size);
        int ahead = 0;
        for (int c = 0; c < team.rank; ++c) ahead += sh.ties[c];
        const int keep = max(0, min(all, need - ahead));
        const int listed = sh.listed;
        for (int v = begin; v < end && at < keep; ++v) {
            float x[Elem<E>::kVec];
            Elem<E>::unpack(buf[v], x);
#pragma unroll
            for (int e = 0; e < Elem<E>::kVec; ++e) {
                if (key_of<E>(x[e]) == f.key && at < keep) {
                    list[listed + at] = entry(x[e], s.first + v * Elem<E>::kVec + e);
                    ++at;
                }
            }
        }
        __syncthreads();
        team.tell(sh.counts, listed + keep);
        cluster_sync(team.size);
        total = n;
    }
    if (team.rank != leader) return 0;
    int at = 0;
    for (int c = 0; c < team.size; ++c) {
        const int count = sh.counts[c];
        const uint64_t* theirs = team.of(list, c);
        for (int i = threadIdx.x; i < count; i += kTeam) sorted[at + i] = theirs[i];
        at += count;
    }
    if (total > kTeam) {
        sort_by<kTeam>(sorted, total);
        return min(n, total);
    }
    __syncthreads();   // a short list in order by counting the better ones
    const int i = threadIdx.x;
    uint64_t mine = 0;
    int rank = 0;
    if (i < total) {
        mine = sorted[i];
        int j = 0;
#pragma unroll 4
        for (; j + 2 <= total; j += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(sorted + j);
            rank += (two.x > mine ? 1 : 0) + (two.y > mine ? 1 : 0);
        }
        if (j < total) rank += sorted[j] > mine ? 1 : 0;
    }
    __syncthreads();
    if (i < total) sorted[rank] = mine;
    __syncthreads();
    return min(n, total);
}

// A value that at least t of this CTA's element-place maxima (kVec of them per
// thread) reach, and not many more; -inf where fewer than t are above -inf.
// The maxima are counted in equal steps below `best`, down to the least of the
// threads' own.
template <int kTeam, class E>
__device__ float threshold(Shared& sh, const uint4& acc, float best, int t) {
    constexpr int kSteps = 128;
    float g[Elem<E>::kVec];
    Elem<E>::unpack(acc, g);
    const float mine = lanes_max<E>(acc);
    if (threadIdx.x < kSteps) sh.steps[threadIdx.x] = 0;
    const float least = block_reduce<kTeam>(mine > neg_inf() ? mine : FLT_MAX, Min(), sh.f8);
    const float span = fmaxf(best - least, 1.0e-30f);
    const float scale = static_cast<float>(kSteps - 1) / span;
#pragma unroll
    for (int e = 0; e < Elem<E>::kVec; ++e)
        if (g[e] > neg_inf()) atomicAdd(&sh.steps[min(kSteps - 1, static_cast<int>((best - g[e]) * scale))], 1);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const int4 four = reinterpret_cast<const int4*>(sh.steps)[lane];
    int run = four.x + four.y + four.z + four.w;
    const int own = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(kAll, run, o);
        if (lane >= o) run += up;
    }
    int step = kSteps;   // the first one up to which there are enough
    if (run >= t) {
        int upto = run - own + four.x;
        step = 4 * lane;
        if (upto < t) { ++step; upto += four.y; }
        if (upto < t) { ++step; upto += four.z; }
        if (upto < t) ++step;
    }
    step = __reduce_min_sync(kAll, step);
    // the last step holds all that is further down; a hundredth of a step and
    // the rounding down cover that of (best - g) * scale
    if (!(best < FLT_MAX) || step >= kSteps - 1) return neg_inf();
    return __fsub_rd(best, (static_cast<float>(step) + 1.01f) / scale);
}

__device__ __forceinline__ void copy_async(uint4* to, const uint4* from) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}
// The cluster's barrier for threads that have nothing to show: their stores
// need not have landed.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// 2^(c2 (x - best)) for x <= best; 0 where nothing is above -inf.
__device__ __forceinline__ float share(float x, float best, float c2) {
    return best > neg_inf() || best != best ? ex2((x - best) * c2) : 0.0f;
}

// This thread's share of the slice's softmax sum, 2^(c2 (x - best)) each: the
// difference is rounded first, so the same holds for maxima of any size. Two
// sums of up to 64 terms in 32 bits at a time, and those in 64: a slice of the
// longest rows has 184 terms for each, and next to a large one as many small
// terms as that, all below half a step of the sum, would be lost.
template <int kTeam, class E>
__device__ __forceinline__ double sum_exp(const uint4* buf, int nv, float c2, float best) {
    constexpr int kVectors = 128 / Elem<E>::kVec;   // of 64 terms in each sum
    const float from = best > neg_inf() ? -best : 0.0f;
    const float2 ff = make_float2(from, from), cc = make_float2(c2, c2);
    double sum = 0.0;
    for (int v0 = threadIdx.x; v0 < nv; v0 += kVectors * kTeam) {
        float2 p = make_float2(0.0f, 0.0f);
        for (int v = v0; v < min(nv, v0 + kVectors * kTeam); v += kTeam) {
            float x[Elem<E>::kVec];
            Elem<E>::unpack(buf[v], x);
#pragma unroll
            for (int e = 0; e < Elem<E>::kVec; e += 2) {
                const float2 t = mul2(add2(make_float2(x[e], x[e + 1]), ff), cc);
                p = add2(p, make_float2(ex2(t.x), ex2(t.y)));
            }
        }
        sum += static_cast<double>(p.x + p.y);
    }
    return sum;
}

// ---------------------------------------------------------------------------
// The best log-probs of a row: x / T - log sum exp(x / T) = (x - m) / T - log Z
// with Z summed in 32 bits by each slice's maximum, 64 terms at a time (in 64
// bits from there on). Bound by latency: one pass over a slice in
// shared memory, 6 barriers of the CTA and 3 of the cluster. 8 rows of 32000
// fp32, n = 20: 9.8 us, of which a launch is 3.
// ---------------------------------------------------------------------------
template <int kTeam, class E>
__global__ void __launch_bounds__(kTeam) top_kernel(TopArgs a, int S, int cap) {
    extern __shared__ uint4 dyn[];
    __shared__ Shared sh;
    const Team team;
    uint4* buf = dyn;
    uint64_t* list = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(dyn) + static_cast<size_t>(S) * sizeof(E));
    uint64_t* sorted = list + cap;
    const int64_t step = gridDim.x / team.size;
    const int n = a.n;
    const float c2 = fminf(1.4426950408889634f / a.temperature, FLT_MAX);
    int leader = 0;
    cluster_sync(team.size);   // everybody's shared memory exists from here on
    const int64_t rows = a.left ? a.left[0] : a.in.rows;
    for (int64_t at = blockIdx.x / team.size; at < rows; at += step) {
        const int64_t row = a.left ? a.left[1 + at] : at;
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
        uint4 acc = vneg_inf<E>();
        const Slice s = load_slice<kTeam, E, true>(static_cast<const E*>(a.in.x) + row * a.in.stride, a.in.V, S, team.rank,
                                            buf, acc);
        const float mine = block_reduce<kTeam>(lanes_max<E>(acc), Max(), sh.f8);
        const double sum = block_reduce<kTeam>(sum_exp<kTeam, E>(buf, s.nv, c2, mine), Add(), sh.d8);
        const float tau = threshold<kTeam, E>(sh, acc, mine, (n + team.size - 1) / team.size);
        team.tell(sh.box, Packet{sum, mine, tau, 0});
        cluster_sync(team.size);
        float best = sh.box[0].best;
        for (int c = 1; c < team.size; ++c) best = fmaxf(best, sh.box[c].best);
        double Z = 0.0;
        for (int c = 0; c < team.size; ++c) {
            const Packet& of = sh.box[c];
            if (of.sum != 0.0)
                Z += of.sum * (of.best == best ? 1.0 : exp2(static_cast<double>(c2) * (static_cast<double>(of.best) -
                                                                                       static_cast<double>(best))));
        }
        const int got = gather_best<kTeam, E>(team, sh, buf, s, best, n, list, sorted, cap, leader);
        if (team.rank == leader) {
            const double log_z = log(Z);
            for (int i = threadIdx.x; i < n; i += kTeam) {
                float value = neg_inf();
                int token = -1;
                if (i < got) {
                    const float x = entry_value(sorted[i]);
                    token = entry_token(sorted[i]);
                    value = static_cast<float>((static_cast<double>(x) - static_cast<double>(best)) /
                                                   static_cast<double>(a.temperature) - log_z);
                }
                a.log_probs[row * n + i] = value;
                a.tokens[row * n + i] = token;
            }
        }
        leader = leader + 1 == team.size ? 0 : leader + 1;
    }
    cluster_sync(team.size);   // nobody leaves while its list is being read
}

// ---------------------------------------------------------------------------
// Sampling. One token is chosen by whole rows' order and mass: the cut is found
// as a key and a number of ties (a list for short top-k, else a search by
// bins), then the token by a sum in index order over the cluster, the CTAs'
// warps and a warp's elements. Bound by latency where a list is enough (one
// row of 32000 bf16, top_k 50: 10.0 us), else by the weights in 64 bits,
// taken three times (twice by the search, once by the choice): one row of 128256 bf16, top_p 0.9 alone, 37.7 us, of a
// floor of 0.04 (34.4 with weights as whole numbers of 2^-43, see SumOf).
// ---------------------------------------------------------------------------

// The token that index order and the uniform number give among the elements
// that the cut keeps. `out` is written by the CTA that holds it.
template <int kTeam, class E>
__device__ void pick(const Team& team, Shared& sh, const uint4* buf, const Slice& s, const Weights& weight, Cut cut,
                     double u, int32_t* out) {
    constexpr int kVec = Elem<E>::kVec;
    constexpr int kWarps = kTeam / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const double tie = weight(value_of<E>(cut.key));
    // a stretch of the slice per warp
    const int per = ((s.nv + kWarps - 1) / kWarps + 31) & ~31;
    const int begin = min(s.nv, per * warp), end = min(s.nv, begin + per);
    double mass = 0.0;
    int ties = 0;
    for (int base = begin; base < end; base += 32) {
        const int v = base + lane;
        float x[kVec];
        Elem<E>::unpack(v < end ? buf[v] : vneg_inf<E>(), x);
        bool any = false;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const uint32_t k = key_of<E>(x[e]);
            ties += k == cut.key ? 1 : 0;
            any = any || k > cut.key;
        }
        if (!__any_sync(kAll, any)) continue;
        double w[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) w[e] = weight(x[e]);
#pragma unroll
        for (int e = 0; e < kVec; ++e) mass += key_of<E>(x[e]) > cut.key ? w[e] : 0.0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mass += __shfl_xor_sync(kAll, mass, o);
        ties += __shfl_xor_sync(kAll, ties, o);
    }
    if (lane == 0) {
        sh.range_mass[warp] = mass;
        sh.range_ties[warp] = ties;
    }
    __syncthreads();
    double cta_mass = 0.0;
    int cta_ties = 0;
    for (int w = 0; w < kTeam / 32; ++w) {
        cta_mass += sh.range_mass[w];
        cta_ties += sh.range_ties[w];
    }
    team.tell(sh.masses, cta_mass);
    team.tell(sh.ties, cta_ties);
    cluster_sync(team.size);
    auto at = [&](double m, int t) { return m + static_cast<double>(min(t, cut.ties)) * tie; };
    // the first part whose running sum passes the target, else the last that adds anything
    double m_all = 0.0;
    int t_all = 0;
    for (int c = 0; c < team.size; ++c) {
        m_all += sh.masses[c];
        t_all += sh.ties[c];
    }
    // a uniform number of 1 or more lies behind every sum, whatever its rounding
    const double target = u < 1.0 ? u * at(m_all, t_all) : HUGE_VAL;
    auto adds = [&](double mass, int t_before, int count) {
        return mass > 0.0 || (tie > 0.0 && min(t_before + count, cut.ties) > min(t_before, cut.ties));
    };
    auto choose = [&](const double* masses, const int* counts, int parts, double& m, int& t) {
        double m_run = m, m_best = m;
        int t_run = t, t_best = t, chosen = -1;
        for (int i = 0; i < parts; ++i) {
            if (adds(masses[i], t_run, counts[i])) {
                chosen = i;
                m_best = m_run;
                t_best = t_run;
                if (at(m_run + masses[i], t_run + counts[i]) > target) break;
            }
            m_run += masses[i];
            t_run += counts[i];
        }
        m = m_best;
        t = t_best;
        return chosen;
    };
    double m = 0.0;
    int t = 0;
    const int owner = choose(sh.masses, sh.ties, team.size, m, t);
    if (owner == team.rank) {
        const int w = choose(sh.range_mass, sh.range_ties, kTeam / 32, m, t);
        // that stretch again, by the whole CTA: neighbouring vectors per thread
        const int w_begin = min(s.nv, per * max(w, 0)), w_end = min(s.nv, w_begin + per);
        const int each = (per + kTeam - 1) / kTeam;
        const int t_begin = min(w_end, w_begin + each * static_cast<int>(threadIdx.x));
        const int t_end = min(w_end, t_begin + each);
        double my_mass = 0.0;
        int my_ties = 0;
        for (int i = 0; i < each; ++i) {
            const int v = t_begin + i;
            float x[kVec];
            Elem<E>::unpack(v < t_end ? buf[v] : vneg_inf<E>(), x);
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                const uint32_t k = key_of<E>(x[e]);
                const double w8 = weight(x[e]);
                my_mass += k > cut.key ? w8 : 0.0;
                my_ties += k == cut.key ? 1 : 0;
            }
        }
        const double m0 = m + block_before<kTeam>(my_mass, sh.d8);
        const int t0 = t + block_before<kTeam>(my_ties, sh.i8);
        const bool mine = adds(my_mass, t0, my_ties);
        const bool past = mine && at(m0 + my_mass, t0 + my_ties) > target;
        const int none = kTeam;
        const int first = block_reduce<kTeam>(past ? static_cast<int>(threadIdx.x) : none, Min(), sh.i8);
        const int last = block_reduce<kTeam>(mine ? static_cast<int>(threadIdx.x) : -1, Max(), sh.i8);
        const int who = first < none ? first : last;
        // its warp walks along its elements
        if (warp == (who >> 5) && who >= 0) {
            double m_run = m0;
            int t_run = t0, token = -1;
            bool done = false;
            for (int i = 0; i < each; ++i) {
                const int v = t_begin + i;
                float x[kVec];
                Elem<E>::unpack(v < t_end ? buf[v] : vneg_inf<E>(), x);
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const uint32_t k = key_of<E>(x[e]);
                    const double w8 = weight(x[e]);
                    const bool some = adds(k > cut.key ? w8 : 0.0, t_run, k == cut.key ? 1 : 0);
                    if (k > cut.key) m_run += w8;
                    if (k == cut.key) ++t_run;
                    if (!done && some) {
                        token = s.first + v * kVec + e;
                        done = at(m_run, t_run) > target;
                    }
                }
            }
            if (static_cast<int>(threadIdx.x) == who) *out = token;
        }
    }
}

// A top-k row: its k best entries in order are all that is needed.
template <int kTeam>
__device__ void pick_listed(Shared& sh, const uint64_t* sorted, int count, float best, float temperature, double p,
                            double log_q, double u, double* weight, int* token, int32_t* out) {
    // weights of the ordered entries; a thread holds neighbouring ones
    const int each = (count + kTeam - 1) / kTeam;
    const int begin = min(count, each * static_cast<int>(threadIdx.x)), end = min(count, begin + each);
    double mine = 0.0;
    for (int i = begin; i < end; ++i) {
        const float x = entry_value(sorted[i]);
        const double z = x == best ? 0.0 : (static_cast<double>(x) - static_cast<double>(best)) /
                                               static_cast<double>(temperature);
        const double w = z < -708.0 ? 0.0 : exp(z);
        weight[i] = w;
        token[i] = entry_token(sorted[i]);
        mine += w;
    }
    const double total = block_reduce<kTeam>(mine, Add(), sh.d8);
    double run = block_before<kTeam>(mine, sh.d8);
    int keep = 0;
    for (int i = begin; i < end; ++i) {
        const float x = entry_value(sorted[i]);
        const double z = x == best ? 0.0 : (static_cast<double>(x) - static_cast<double>(best)) /
                                               static_cast<double>(temperature);
        keep += (i == 0 || ((!(p < 1.0) || run < p * total) && z >= log_q)) ? 1 : 0;
        run += weight[i];
    }
    keep = block_reduce<kTeam>(keep, Add(), sh.i8);   // the kept ones are the first
    mine = 0.0;
    for (int i = begin; i < min(end, keep); ++i) mine += weight[i];
    const double kept = block_reduce<kTeam>(mine, Add(), sh.d8);
    const double target = u < 1.0 ? u * kept : HUGE_VAL;   // as in pick()
    // the least kept index whose sum of weights up to it passes the target
    int first = 0x7FFFFFFF, last = -1;
    for (int i = threadIdx.x; i < keep; i += kTeam) {
        const int own = token[i];
        double sum = 0.0;
        for (int j = 0; j < keep; ++j) sum += token[j] <= own ? weight[j] : 0.0;
        if (weight[i] > 0.0) {
            last = max(last, own);
            if (sum > target) first = min(first, own);
        }
    }
    first = block_reduce<kTeam>(first, Min(), sh.i8);
    last = block_reduce<kTeam>(last, Max(), sh.i8);
    if (threadIdx.x == 0) *out = first < 0x7FFFFFFF ? first : last;
}

template <int kTeam, class E>
__global__ void __launch_bounds__(kTeam) sample_kernel(SampleArgs a, int S, int cap) {
    extern __shared__ uint4 dyn[];
    __shared__ Shared sh;
    const Team team;
    uint4* buf = dyn;
    uint64_t* list = reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(dyn) + static_cast<size_t>(S) * sizeof(E));
    uint64_t* sorted = list + cap;
    const int64_t step = gridDim.x / team.size;
    const int V = a.in.V;
    int leader = 0;
    cluster_sync(team.size);
    const int64_t rows = a.left ? a.left[0] : a.in.rows;
    for (int64_t at = blockIdx.x / team.size; at < rows; at += step) {
        const int64_t row = a.left ? a.left[1 + at] : at;
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
        const float given = a.temperature ? a.temperature[row] : a.temperature_all;
        const float temperature = given > FLT_MAX ? FLT_MAX : given;
        const int k = a.top_k ? a.top_k[row] : a.top_k_all;
        const double p = static_cast<double>(a.top_p ? a.top_p[row] : a.top_p_all);
        const float q_given = a.min_p ? a.min_p[row] : a.min_p_all;
        const double q = q_given > 1.0f ? 1.0 : static_cast<double>(q_given);
        const double u = static_cast<double>(a.uniforms[row]);
        const bool cut_k = k > 0 && k < V;
        // one token is left: no temperature, the best one alone, or no mass
        const bool greedy = !(given > 0.0f) || k == 1 || p <= 0.0;
        const bool by_list = !greedy && cut_k && k <= kSampleList;
        uint4 acc = vneg_inf<E>();
        const Slice s = load_slice<kTeam, E, true>(static_cast<const E*>(a.in.x) + row * a.in.stride, V, S, team.rank, buf,
                                            acc);
        const float mine = block_reduce<kTeam>(lanes_max<E>(acc), Max(), sh.f8);
        float tau = neg_inf();
        int index = 0x7FFFFFFF;
        if (by_list) tau = threshold<kTeam, E>(sh, acc, mine, (k + team.size - 1) / team.size);
        if (greedy) {
            for (int v = threadIdx.x; v < s.nv; v += kTeam) {
                float x[Elem<E>::kVec];
                Elem<E>::unpack(buf[v], x);
#pragma unroll
                for (int e = 0; e < Elem<E>::kVec; ++e)
                    if (x[e] == mine) index = min(index, s.first + v * Elem<E>::kVec + e);
            }
            index = block_reduce<kTeam>(index, Min(), sh.i8);
        }
        team.tell(sh.box, Packet{0.0, mine, tau, index});
        cluster_sync(team.size);
        float best = sh.box[0].best;
        for (int c = 1; c < team.size; ++c) best = fmaxf(best, sh.box[c].best);
        int32_t* out = a.tokens + row;
        if (!(best > neg_inf())) {
            if (team.rank == leader && threadIdx.x == 0) *out = -1;
            cluster_sync(team.size);   // box is free again
        } else if (greedy) {
            if (team.rank == leader && threadIdx.x == 0) {
                int token = 0x7FFFFFFF;
                for (int c = 0; c < team.size; ++c)
                    if (sh.box[c].best == best) token = min(token, sh.box[c].index);
                *out = token;
            }
            cluster_sync(team.size);
        } else if (by_list) {
            const int got = gather_best<kTeam, E>(team, sh, buf, s, best, k, list, sorted, cap, leader);
            if (team.rank == leader) {
                // the leader's own list has been copied: its space holds the weights
                double* weight = reinterpret_cast<double*>(list);
                int* token = reinterpret_cast<int*>(weight + got);
                pick_listed<kTeam>(sh, sorted, got, best, temperature, p, q > 0.0 ? log(q) : -HUGE_VAL, u, weight, token, out);
            }
        } else {
            const Weights weight(best, temperature, false);
            uint32_t* hist = reinterpret_cast<uint32_t*>(list);
            const uint32_t none = key_of<E>(neg_inf());
            Cut cut{none, 0};
            double cut_mass = 0.0;   // of the equal ones at the top-k cut
            if (cut_k) {
                float low = best;
                for_elements<kTeam, E>(buf, s, [&](float x, int) { low = x > neg_inf() ? fminf(low, x) : low; });
                low = block_reduce<kTeam>(low, Min(), sh.f8);
                cluster_sync(team.size);
                team.tell(sh.box, Packet{0.0, 0.0f, low, 0});
                cluster_sync(team.size);
                for (int c = 0; c < team.size; ++c) low = fminf(low, sh.box[c].tau);
                float span = best - low;
                if (!(span > 0.0f)) span = 1.0f;
                if (!(span < FLT_MAX)) span = FLT_MAX;
                const Found f = search<kTeam, E, false>(team, sh, hist, buf, s, weight, span, none,
                                                 static_cast<double>(k), 0.0);
                if (f.ok) {
                    cut.key = f.key;
                    cut.ties = k - static_cast<int>(f.above);
                    cut_mass = weight(value_of<E>(f.key));
                }
            }
            if (p < 1.0) {
                // (2047 / span has to stay finite)
                const float span = fminf(fmaxf(32.0f * temperature, 1.0e-35f), FLT_MAX);
                const Found f = search<kTeam, E, true>(team, sh, hist, buf, s, weight, span, cut.key, p,
                                                static_cast<double>(cut.ties) * cut_mass);
                if (f.ok) {
                    cut.key = f.key;
                    cut.ties = 0x7FFFFFFF;
                    cut_mass = weight(value_of<E>(f.key));
                }
                // of the equal ones, as many as reach the target
                const double left = ceil((f.target - f.above) / cut_mass);
                if (left < static_cast<double>(cut.ties)) cut.ties = max(1, static_cast<int>(left));
            }
            if (q > 0.0) {
                // kept: x >= m + T ln q, rounded up to a float
                const float low = __double2float_ru(static_cast<double>(best) +
                                                    static_cast<double>(temperature) * log(q));
                const uint32_t low_key = key_of<E>(fminf(low, best));
                // a 16-bit type's key drops low bits: the least key whose value reaches `low`
                const uint32_t least = value_of<E>(low_key) >= low ? low_key : low_key + 1;
                if (least > cut.key) {
                    cut.key = least - 1;
                    cut.ties = 0;
                }
            }
            pick<kTeam, E>(team, sh, buf, s, weight, cut, u, out);
            cluster_sync(team.size);
        }
        leader = leader + 1 == team.size ? 0 : leader + 1;
    }
    cluster_sync(team.size);
}

// ---------------------------------------------------------------------------
// Many rows: a scan that lists each row's candidates, then a kernel that
// finishes the rows from their lists.
//
// A row's vectors are dealt to `parts` CTAs in chunks of one vector per thread
// (chunk c to part c mod parts, so that tokens sorted by frequency spread
// evenly). A part keeps its maximum, its sum and its candidates: the elements
// at or above a threshold below which at least `take` of its threads' maxima
// do not lie. No part waits for another, so that the scan runs at the memory's
// pace. The finish accepts a list where its last wanted entry reaches every
// part's threshold: then nothing unlisted could have come before it. Rows that
// fail (or whose ties overflow a list) go to the cluster's kernel above, by
// the list `left`.
//
// A part's vectors are a thread's own from the copy to the last use, so that
// copies need no barrier, and are copied ahead by cp.async, 64 KB a CTA, three
// CTAs on an SM; the next part's begin when this part's last vector has been
// used. Bound by latency at 24 warps an SM (barriers, the loads that follow one
// another in a part) with issue next, active in 52 % of the cycles: 11
// instructions an element with the exponential (2048 rows of 128256 bf16, n =
// 64: about 160 of 185 us, 3.3 TB/s). With a weight in 64 bits it is 34, active
// in 65 % (512 rows of them, temperature alone: about 95 of 109 us). Also
// measured there, in us: a warp per part without barriers 236, the cluster's
// kernel for all rows 385 and 264.
// ---------------------------------------------------------------------------
struct PartState {
    double sum;
    float best;
    float tau;     // everything at or above it is listed
    int count;
    int unused;
};
struct ScanState {
    PartState* parts;    // [rows, parts]
    uint64_t* lists;     // [rows, parts, cap]
    double* chunks;      // [rows, parts * kHold, kWarps]: sums of a warp's vectors of a chunk
    int* left;           // [1 + rows]: the number of rows for the cluster's kernel, and which
};
struct ScanShape {
    int parts;
    int cap;
};
constexpr int kHold = 16;       // most chunks of a part, and most vectors of a slice per thread
constexpr int kScanBins = 128;
constexpr int kMaxParts = 32;   // a part per lane where they are put together
// Candidates listed for a top-p without a top-k: 64 rows of 50257 fp32, top_p
// 0.95, min_p 0.02 take 42 us with 512, 57 with 256 and 46 with 1024; 256 rows
// of 128256 with their own settings 114, 98 and 112: there 256 would be the
// better choice, and nothing known before the call separates the two.
constexpr int kNucleus = 512;

__host__ __device__ __forceinline__ ScanState scan_of(void* space, int64_t rows, ScanShape sh, bool chunks) {
    ScanState s;
    char* p = static_cast<char*>(space);
    s.parts = reinterpret_cast<PartState*>(p);
    p += rows * sh.parts * static_cast<int64_t>(sizeof(PartState));
    s.lists = reinterpret_cast<uint64_t*>(p);
    p += rows * sh.parts * sh.cap * 8;
    s.chunks = reinterpret_cast<double*>(p);
    if (chunks) p += rows * sh.parts * kHold * kWarps * 8;
    s.left = reinterpret_cast<int*>(p);
    return s;
}

// What a row needs of the scan.
struct Plan {
    int take;       // candidates; 0: none, or all from `low` on
    bool sum;       // its mass in 64 bits
    bool chunks;    // and that of each chunk
    bool by_low;    // candidates are what reaches maximum + low
    float temperature;
    double low;     // T ln(min_p), at most 0
    int k;          // 0: no cut by rank
    double p, q;
    bool left;      // the cluster's kernel takes the row
};

__device__ __forceinline__ Plan plan_of(const SampleArgs& a, int64_t row) {
    Plan r;
    const float given = a.temperature ? a.temperature[row] : a.temperature_all;
    r.temperature = given > FLT_MAX ? FLT_MAX : given;
    const int k = a.top_k ? a.top_k[row] : a.top_k_all;
    r.p = static_cast<double>(a.top_p ? a.top_p[row] : a.top_p_all);
    const float q_given = a.min_p ? a.min_p[row] : a.min_p_all;
    r.q = q_given > 1.0f ? 1.0 : static_cast<double>(q_given);
    r.k = k > 0 && k < a.in.V ? k : 0;
    const bool greedy = !(given > 0.0f) || k == 1 || r.p <= 0.0;
    const bool by_p = r.p < 1.0, by_q = r.q > 0.0;
    r.low = by_q && !greedy ? static_cast<double>(r.temperature) * log(r.q) : -HUGE_VAL;
    r.take = greedy ? 1 : r.k > 0 ? r.k : by_p ? kNucleus : 0;
    if (greedy) r.k = 1;
    r.sum = !greedy && r.k == 0 && (by_p || !by_q);
    r.chunks = r.sum && !by_p;
    // the mass of the first k needs all of them, whatever min_p leaves of them
    r.by_low = by_q && !greedy && (r.k == 0 || !by_p);
    // at such temperatures 690 T or 32 / (T ln 2) is beyond 32 bits (see Weights::term)
    r.left = r.k > kSampleList || (r.sum && !(r.temperature >= 1.0e-36f && r.temperature <= 1.0e30f));
    return r;
}
__device__ __forceinline__ Plan plan_of(const TopArgs& a, int64_t) {
    Plan r = {};
    r.take = r.k = a.n;
    r.temperature = a.temperature;
    return r;
}

template <class E, class Args, bool kTop>
__global__ void __launch_bounds__(kThreads, 3) scan_kernel(Args a, ScanShape shape, void* space, bool with_chunks) {
    constexpr int kVec = Elem<E>::kVec;
    extern __shared__ uint4 dyn[];
    __shared__ float2 part8[kWarps];
    __shared__ float low8[kWarps];
    __shared__ double d8[kWarps];
    // the bins and the list's length of this part and the next
    __shared__ __align__(16) int hist2[2 * kScanBins];
    __shared__ int listed2[2];
    const ScanState state = scan_of(space, a.in.rows, shape, with_chunks);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.in.V;
    const uint4 none = vneg_inf<E>();
    uint4* buf = dyn + tid;    // this thread's vectors, kThreads apart
    const int per = ((V + kVec - 2) / kVec + 1 + kThreads * shape.parts - 1) / (kThreads * shape.parts);   // chunks of a part
    if (blockIdx.x == 0 && tid == 0) state.left[0] = 0;
    // A part at a time: row and part, and how far the next one is.
    int64_t row = blockIdx.x / shape.parts;
    int part = static_cast<int>(blockIdx.x % shape.parts);
    const int64_t row_step = gridDim.x / shape.parts;
    const int part_step = static_cast<int>(gridDim.x % shape.parts);
    struct View {
        const E* x;
        const uint4* src;
        int phase, v0, v1;
    };
    auto view = [&](int64_t r) {
        View w;
        w.x = static_cast<const E*>(a.in.x) + r * a.in.stride;
        const uintptr_t at = reinterpret_cast<uintptr_t>(w.x);
        w.phase = static_cast<int>((at & 15u) / sizeof(E));
        w.src = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15));
        w.v0 = w.phase > 0 ? 1 : 0;
        w.v1 = (V + w.phase) / kVec;
        return w;
    };
    // a vector that the row fills only in part
    auto ragged = [&](const View& w, int v) {
        float f[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            const int token = v * kVec + e - w.phase;
            f[e] = token >= 0 && token < V ? Elem<E>::widen(w.x[token]) : neg_inf();
        }
        return Elem<E>::pack(f);
    };
    const int stride = shape.parts * kThreads;
    auto copy = [&](const View& w, int p) {
        int v = p * kThreads + tid;
        if (w.v0 == 0 && (p + 1) * kThreads + (per - 1) * stride <= w.v1) {
            const uint4* from = w.src + v;
#pragma unroll 4
            for (int i = 0; i < per; ++i, from += stride) copy_async(buf + i * kThreads, from);
        } else {
            for (int i = 0; i < per; ++i, v += stride) {
                if (v >= w.v0 && v < w.v1)
                    copy_async(buf + i * kThreads, w.src + v);
                else
                    buf[i * kThreads] = v * kVec < V + w.phase ? ragged(w, v) : none;
            }
        }
        copies_commit();
    };
    View here = view(row);
    if (tid < 2 * kScanBins) hist2[tid] = 0;
    if (tid < 2) listed2[tid] = 0;
    int parity = 0;
    if (row < a.in.rows) copy(here, part);
    __syncthreads();
    while (row < a.in.rows) {
        int64_t next_row = row + row_step;
        int next_part = part + part_step;
        if (next_part >= shape.parts) {
            next_part -= shape.parts;
            ++next_row;
        }
        const View next = view(next_row);
        const bool more = next_row < a.in.rows;
        const Plan plan = plan_of(a, row);
        const int phase = here.phase;
        int* hist = hist2 + parity * kScanBins;
        int* listed = listed2 + parity;
        parity ^= 1;
        copies_wait<0>();
        uint4 top = none;
        float mine = neg_inf(), sum = 0.0f, from = 0.0f;
        const float c2 = fminf(1.4426950408889634f / plan.temperature, FLT_MAX);
        if (kTop) {
            // The thread's exponentials by the maximum of its first vectors;
            // where the others run so far beyond it that the sum overflows, or
            // where there is a NaN, by the maximum of all and without NaN.
            auto add_up = [&](bool clean) {
                const float2 ff = make_float2(-from, -from), cc = make_float2(c2, c2);
                float2 p = make_float2(0.0f, 0.0f);
#pragma unroll 4
                for (int i = 0; i < per; ++i) {
                    uint4 r = buf[i * kThreads];
                    if (clean) r = vmax<E>(r, none);
                    float f[kVec];
                    Elem<E>::unpack(r, f);
                    // (two 16-bit values at a time would take the exponentials' pipe)
#pragma unroll
                    for (int e = 0; e < kVec; e += 2) mine = fmaxf(fmaxf(f[e], f[e + 1]), mine);
#pragma unroll
                    for (int e = 0; e < kVec; e += 2) {
                        const float2 t = mul2(add2(make_float2(f[e], f[e + 1]), ff), cc);
                        p = add2(p, make_float2(ex2(t.x), ex2(t.y)));
                    }
                }
                sum = p.x + p.y;
            };
            for (int i = 0; i < min(per, 4); ++i) top = vmax<E>(top, buf[i * kThreads]);
            const float first = lanes_max<E>(top);
            from = first > neg_inf() ? first : 0.0f;
            add_up(false);
            if (!(first > neg_inf()) || !(sum < 1.0e30f)) {
                from = mine > neg_inf() ? mine : 0.0f;
                add_up(true);
            }
        } else {
#pragma unroll 4
            for (int i = 0; i < per; ++i) top = vmax<E>(top, buf[i * kThreads]);
        }
        if (!kTop) mine = lanes_max<E>(top);
        // the sums in 64 bits go over the vectors a second time
        const bool again = !kTop && plan.sum;
        if (!again && more) copy(next, next_part);
        float2 of_warp = make_float2(mine, 0.0f);
        float least = mine > neg_inf() ? mine : FLT_MAX;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            of_warp.x = fmaxf(of_warp.x, __shfl_xor_sync(kAll, of_warp.x, o));
            least = fminf(least, __shfl_xor_sync(kAll, least, o));
        }
        if (kTop) {
            of_warp.y = sum == 0.0f ? 0.0f : sum * ex2((from - of_warp.x) * c2);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) of_warp.y += __shfl_xor_sync(kAll, of_warp.y, o);
        }
        if (lane == 0) {
            part8[warp] = of_warp;
            low8[warp] = least;
        }
        __syncthreads();
        float best = part8[0].x;
        least = low8[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            best = fmaxf(best, part8[w].x);
            least = fminf(least, low8[w]);
        }
        float tau = HUGE_VALF;   // nothing is listed
        if (plan.take > 0 && !plan.left) {
            // how many of the threads' maxima to pass: the part's share, and
            // three times the spread of such shares
            const float mean = static_cast<float>(plan.take) / static_cast<float>(shape.parts);
            const int want = static_cast<int>(ceilf(mean + 3.0f * sqrtf(mean))) + (shape.parts > 1 ? 2 : 0);
            const float span = fmaxf(best - least, 1.0e-30f);
            const float scale = static_cast<float>(kScanBins - 1) / span;
            if (mine > neg_inf()) atomicAdd(&hist[min(kScanBins - 1, static_cast<int>((best - mine) * scale))], 1);
            __syncthreads();
            const int4 four = reinterpret_cast<const int4*>(hist)[lane];
            int run = four.x + four.y + four.z + four.w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(kAll, run, o);
                if (lane >= o) run += up;
            }
            int bin = kScanBins;   // the first bin up to which there are enough
            const int before = run - (four.x + four.y + four.z + four.w);
            if (run >= want) {
                bin = 4 * lane;
                int sum4 = before + four.x;
                if (sum4 < want) { ++bin; sum4 += four.y; }
                if (sum4 < want) { ++bin; sum4 += four.z; }
                if (sum4 < want) ++bin;
            }
            bin = __reduce_min_sync(kAll, bin);
            tau = bin < kScanBins - 1 && best < FLT_MAX ? best - static_cast<float>(bin + 1) / scale : neg_inf();
        }
        if (plan.by_low && !plan.left) {
            const float low = __double2float_rd(static_cast<double>(best) + plan.low);
            tau = plan.take > 0 ? fmaxf(tau, low) : low;
        }
        double mass = 0.0;
        if (again && best > neg_inf()) {
            const Weights weight(best, plan.temperature, true);
            const float low = best - 690.0f * plan.temperature;
            for (int i = 0; i < per; ++i) {
                float f[kVec];
                Elem<E>::unpack(buf[i * kThreads], f);
                double w0 = 0.0, w1 = 0.0;
#pragma unroll
                for (int e = 0; e < kVec; e += 2) {
                    w0 += weight.term(f[e], low);
                    w1 += weight.term(f[e + 1], low);
                }
                double w = w0 + w1;
                mass += w;
                if (plan.chunks) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(kAll, w, o);
                    if (lane == 0)
                        state.chunks[(row * shape.parts * kHold + i * shape.parts + part) * kWarps + warp] = w;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(kAll, mass, o);
            if (lane == 0) d8[warp] = mass;
        }
        if (again && more) copy(next, next_part);
        // The warp looks through the vectors of those of its threads whose
        // maximum reaches tau, two threads at a time and a vector per lane;
        // they come from L2, as shared memory is on to the next rows.
        const int64_t item = row * shape.parts + part;
        uint64_t* list = state.lists + item * shape.cap;
        for (unsigned have = __ballot_sync(kAll, mine >= tau && mine > neg_inf()); have;) {
            int owner = __ffs(have) - 1;
            have &= have - 1;
            const int other = have ? __ffs(have) - 1 : -1;
            have &= have - 1;
            if (lane >= kHold) owner = other;
            const int i = lane % kHold, v = (i * shape.parts + part) * kThreads + warp * 32 + owner;
            if (owner < 0 || i >= per || v >= (V + phase + kVec - 1) / kVec) continue;
            float f[kVec];
            Elem<E>::unpack(v >= here.v0 && v < here.v1 ? ldg_once(here.src + v) : ragged(here, v), f);
            unsigned hits = 0;
#pragma unroll
            for (int e = 0; e < kVec; ++e) hits |= f[e] >= tau && f[e] > neg_inf() ? 1u << e : 0u;
            if (hits == 0) continue;
            int place = atomicAdd(listed, __popc(hits));
#pragma unroll
            for (int e = 0; e < kVec; ++e) {
                if (!(hits >> e & 1u)) continue;
                if (place < shape.cap) list[place] = entry(f[e], v * kVec + e - phase);
                ++place;
            }
        }
        float all = 0.0f;
        if (kTop && tid < 32) {   // the warps' sums, a warp per lane
            const float2 of = lane < kWarps ? part8[lane] : make_float2(neg_inf(), 0.0f);
            all = of.y == 0.0f ? 0.0f : of.y * share(of.x, best, c2);
#pragma unroll
            for (int o = kWarps / 2; o > 0; o >>= 1) all += __shfl_xor_sync(kAll, all, o);
        }
        // this part's bins were read before, the other ones are in use next
        __syncthreads();
        if (tid < kScanBins) hist[tid] = 0;
        if (tid == 0) {
            PartState out = {static_cast<double>(all), best, tau, *listed, 0};
            if (!kTop && plan.sum && best > neg_inf()) {
                out.sum = 0.0;
                for (int w = 0; w < kWarps; ++w) out.sum += d8[w];
            }
            state.parts[item] = out;
            *listed = 0;
        }
        row = next_row;
        part = next_part;
        here = next;
    }
    copies_wait<0>();
}

// The entries of the parts' lists that reach every part's threshold, in `keys`,
// best first: none is missing between them.
struct Gathered {
    int count;     // -1: a list overflowed
    float best;
    float tau;     // the highest of the parts' thresholds
    bool all;      // every element above -inf is there
};
template <int kT>
__device__ Gathered gather_parts(const ScanState& state, ScanShape shape, int64_t row, uint64_t* keys, uint64_t* other,
                                 int* counter) {
    const PartState* parts = state.parts + row * shape.parts;
    Gathered g;
    // a part per lane, by every warp
    const int lane = threadIdx.x % 32;
    PartState mine = {0.0, neg_inf(), neg_inf(), 0, 0};
    if (lane < shape.parts) mine = parts[lane];
    g.best = mine.best;
    g.tau = mine.best > neg_inf() ? mine.tau : neg_inf();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        g.best = fmaxf(g.best, __shfl_xor_sync(kAll, g.best, o));
        g.tau = fmaxf(g.tau, __shfl_xor_sync(kAll, g.tau, o));
    }
    g.all = !(g.tau > neg_inf());
    g.count = -1;
    if (__any_sync(kAll, mine.count > shape.cap)) return g;
    if (threadIdx.x == 0) *counter = 0;
    __syncthreads();
    // a part's entries by a warp
    for (int s = threadIdx.x / 32; s < shape.parts; s += kT / 32) {
        const int count = __shfl_sync(kAll, mine.count, s);
        const uint64_t* list = state.lists + (row * shape.parts + s) * shape.cap;
        for (int i = lane; i - lane < count; i += 32) {
            const uint64_t e = i < count ? list[i] : 0;
            const bool in = i < count && entry_value(e) >= g.tau;
            const unsigned all = __ballot_sync(kAll, in);
            int at = lane == 0 ? atomicAdd(counter, __popc(all)) : 0;
            at = __shfl_sync(kAll, at, 0) + __popc(all & ((1u << lane) - 1u));
            if (in) other[at] = e;
        }
    }
    __syncthreads();
    g.count = *counter;
    if (g.count > kT) {
        sort_by<kT>(other, g.count);
        for (int i = threadIdx.x; i < g.count; i += kT) keys[i] = other[i];
    }
    // a short list in order by counting the better ones
    const int i = threadIdx.x;
    if (i < g.count && g.count <= kT) {
        const uint64_t own = other[i];
        int rank = 0;
        int j = 0;
        for (; j + 2 <= g.count; j += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(other + j);
            rank += (two.x > own ? 1 : 0) + (two.y > own ? 1 : 0);
        }
        if (j < g.count) rank += other[j] > own ? 1 : 0;
        keys[rank] = own;
    }
    __syncthreads();
    return g;
}

// A row's lists in order, and its sums joined. Bound by latency: a row takes
// about 7 us, 2048 rows of n = 64 about 20 us.
__global__ void __launch_bounds__(256) top_finish_kernel(TopArgs a, ScanShape shape, void* space, bool with_chunks) {
    extern __shared__ uint4 dyn[];
    __shared__ int counter;
    constexpr int kFinish = 256;
    const ScanState state = scan_of(space, a.in.rows, shape, with_chunks);
    uint64_t* keys = reinterpret_cast<uint64_t*>(dyn);
    uint64_t* other = keys + shape.parts * shape.cap;
    const int n = a.n;
    const double c = static_cast<double>(fminf(1.4426950408889634f / a.temperature, FLT_MAX));
    for (int64_t row = blockIdx.x; row < a.in.rows; row += gridDim.x) {
        const Gathered g = gather_parts<kFinish>(state, shape, row, keys, other, &counter);
        if (g.count < 0 || (!g.all && g.count < n) || !(g.best < HUGE_VALF)) {
            if (threadIdx.x == 0) state.left[1 + atomicAdd(&state.left[0], 1)] = static_cast<int>(row);
            __syncthreads();
            continue;
        }
        double Z = 0.0;   // a part per lane, by every warp
        if (static_cast<int>(threadIdx.x) % 32 < shape.parts) {
            const PartState p = state.parts[row * shape.parts + threadIdx.x % 32];
            if (p.sum != 0.0)
                Z = p.sum * (p.best == g.best ? 1.0 : exp2(c * (static_cast<double>(p.best) - static_cast<double>(g.best))));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) Z += __shfl_xor_sync(kAll, Z, o);
        const double log_z = log(Z);
        for (int i = threadIdx.x; i < n; i += kFinish) {
            float value = neg_inf();
            int token = -1;
            if (i < g.count) {
                token = entry_token(keys[i]);
                value = static_cast<float>((static_cast<double>(entry_value(keys[i])) - static_cast<double>(g.best)) /
                                               static_cast<double>(a.temperature) - log_z);
            }
            a.log_probs[row * n + i] = value;
            a.tokens[row * n + i] = token;
        }
        __syncthreads();
    }
}

// A row's token from its lists, or from its stretches' sums where every token
// can come. Bound by latency, as above: 7 us for a row of 100 candidates (12000
// to 14000 cycles: reading the lists 4000, the cut 2800, the choice 2200), 15
// us for one of 1000, most of it for two sorts.
template <class E>
__global__ void __launch_bounds__(512) sample_finish_kernel(SampleArgs a, ScanShape shape, void* space, bool with_chunks) {
    constexpr int kVec = Elem<E>::kVec;
    constexpr int kFinish = 512;
    constexpr int kW = kFinish / 32;
    extern __shared__ uint4 dyn[];
    __shared__ int counter;
    __shared__ double d8[kW];
    __shared__ int i8[kW];
    const ScanState state = scan_of(space, a.in.rows, shape, with_chunks);
    uint64_t* keys = reinterpret_cast<uint64_t*>(dyn);
    uint64_t* other = keys + shape.parts * shape.cap;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto total_of = [&](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
        if (lane == 0) d8[warp] = v;
        __syncthreads();
        v = 0.0;
        for (int w = 0; w < kW; ++w) v += d8[w];
        __syncthreads();
        return v;
    };
    auto before_of = [&](double v) {   // the sum of the threads before this one
        double incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double up = __shfl_up_sync(kAll, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) d8[warp] = incl;
        __syncthreads();
        double base = 0.0;
        for (int w = 0; w < warp; ++w) base += d8[w];
        __syncthreads();
        const double excl = __shfl_up_sync(kAll, incl, 1);
        return base + (lane == 0 ? 0.0 : excl);
    };
    auto over_ints = [&](int v, auto op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
        if (lane == 0) i8[warp] = v;
        __syncthreads();
        v = i8[0];
        for (int w = 1; w < kW; ++w) v = op(v, i8[w]);
        __syncthreads();
        return v;
    };
    for (int64_t row = blockIdx.x; row < a.in.rows; row += gridDim.x) {
        const Plan plan = plan_of(a, row);
        const double u = static_cast<double>(a.uniforms[row]);
        const PartState* parts = state.parts + row * shape.parts;
        int32_t* out = a.tokens + row;
        auto leave = [&]() {
            if (tid == 0) state.left[1 + atomicAdd(&state.left[0], 1)] = static_cast<int>(row);
            __syncthreads();
        };
        if (plan.left) {
            leave();
            continue;
        }
        // a part per lane, by every warp
        PartState own_part = {0.0, neg_inf(), 0.0f, 0, 0};
        if (lane < shape.parts) own_part = parts[lane];
        float best = own_part.best;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(kAll, best, o));
        if (!(best > neg_inf())) {
            if (tid == 0) *out = -1;
            continue;
        }
        const double T = static_cast<double>(plan.temperature), m = static_cast<double>(best);
        // the cluster's kernel knows infinities, and maxima from which 690 T is
        // lost in a float's rounding (see Weights::term)
        if ((best > FLT_MAX && plan.take != 1) || (plan.sum && fabsf(best) > 1.0e6f * plan.temperature)) {
            leave();
            continue;
        }
        // what a part's sums are multiplied by to go by the row's maximum
        const double factor = own_part.best == best ? 1.0
                              : own_part.best > neg_inf() ? exp((static_cast<double>(own_part.best) - m) / T) : 0.0;
        double W = 0.0;
        if (plan.sum) {
            W = factor == 0.0 ? 0.0 : own_part.sum * factor;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) W += __shfl_xor_sync(kAll, W, o);
        }
        if (plan.chunks) {
            // temperature alone: the first stretch of 32 vectors at which the
            // running sum passes the target, then the element in it
            const double target = u < 1.0 ? u * W : HUGE_VAL;
            const int stretches = shape.parts * kHold * kWarps;
            const int per = ((a.in.V + kVec - 2) / kVec + 1 + kThreads * shape.parts - 1) / (kThreads * shape.parts);
            const int used = per * shape.parts * kWarps;
            const double* sums = state.chunks + row * stretches;
            if (!(u > 0.0 && u < 1.0)) {   // the first or last weight above 0 is wanted, however small
                leave();
                continue;
            }
            __shared__ double factors[kMaxParts];
            if (warp == 0) factors[lane] = factor;
            __syncthreads();
            const int each = (used + kFinish - 1) / kFinish;
            const int begin = min(used, each * tid), end = min(used, begin + each);
            auto stretch = [&](int i) {
                const double f = factors[i / kWarps % shape.parts];
                return f == 0.0 ? 0.0 : sums[i] * f;
            };
            double mine = 0.0;
            for (int i = begin; i < end; ++i) mine += stretch(i);
            double run = before_of(mine);
            int first = used, last = -1;
            double first_run = 0.0, last_run = 0.0;
            for (int i = begin; i < end; ++i) {
                const double v = stretch(i);
                if (v > 0.0) {
                    last = i;
                    last_run = run;
                    if (first == used && run + v > target) {
                        first = i;
                        first_run = run;
                    }
                }
                run += v;
            }
            const int first_all = over_ints(first, Min()), last_all = over_ints(last, Max());
            const int chosen = first_all < used ? first_all : last_all;
            if ((first_all < used && first == chosen) || (first_all >= used && last == chosen)) {
                if (chosen >= 0) {
                    d8[0] = first_all < used ? first_run : last_run;
                    counter = chosen;
                }
            }
            __syncthreads();
            if (warp == 0) {
                const int at = counter;
                double base = d8[0];
                const E* x = static_cast<const E*>(a.in.x) + row * a.in.stride;
                const int phase = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(E));
                const int64_t start = (static_cast<int64_t>(at / kWarps) * kThreads + at % kWarps * 32 + lane) * kVec - phase;
                const Weights weight(best, plan.temperature, true);
                double w[kVec], own = 0.0;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const int64_t token = start + e;
                    float v = token >= 0 && token < a.in.V ? Elem<E>::widen(x[token]) : neg_inf();
                    w[e] = weight(v == v ? v : neg_inf());
                    own += w[e];
                }
                double incl = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(kAll, incl, o);
                    if (lane >= o) incl += up;
                }
                const double up = __shfl_up_sync(kAll, incl, 1);
                double at_run = base + (lane == 0 ? 0.0 : up);
                int hit = 0x7FFFFFFF, end_token = -1;
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    at_run += w[e];
                    if (w[e] > 0.0) {
                        end_token = static_cast<int>(start) + e;
                        if (hit == 0x7FFFFFFF && at_run > target) hit = end_token;
                    }
                }
                hit = __reduce_min_sync(kAll, hit);
                end_token = __reduce_max_sync(kAll, end_token);
                if (lane == 0) *out = hit < 0x7FFFFFFF ? hit : end_token;
            }
            __syncthreads();
            continue;
        }
        const Gathered g = gather_parts<kFinish>(state, shape, row, keys, other, &counter);
        if (g.count < 0) {
            leave();
            continue;
        }
        if (plan.take == 1) {
            if (tid == 0) *out = entry_token(keys[0]);
            __syncthreads();
            continue;
        }
        // the first k, or as many as are known
        const int count = plan.k > 0 ? min(plan.k, g.count) : g.count;
        // Is what lies behind the known ranks out? By rank; as everything that
        // reaches m + T ln q is known; or as p or q cut within the known ones.
        // The mass that p goes by is the row's, or that of the first k.
        const bool mass_known = plan.k == 0 || !(plan.p < 1.0);
        const bool enough = g.all || (plan.k > 0 && g.count >= plan.k) ||
                            (mass_known && plan.q > 0.0 && static_cast<double>(g.tau) <= m + plan.low);
        double* weight = reinterpret_cast<double*>(other);
        const int each = (count + kFinish - 1) / kFinish;
        const int begin = min(count, each * tid), end = min(count, begin + each);
        double mine = 0.0;
        auto z_of = [&](int i) {
            const float x = entry_value(keys[i]);
            return x == best ? 0.0 : (static_cast<double>(x) - m) / T;
        };
        for (int i = begin; i < end; ++i) {
            const double z = z_of(i);
            weight[i] = z < -708.0 ? 0.0 : exp(z);
            mine += weight[i];
        }
        const double listed_mass = total_of(mine);
        if (plan.k > 0) W = listed_mass;
        double run = before_of(mine);
        const double log_q = plan.q > 0.0 ? log(plan.q) : -HUGE_VAL;
        int keep = 0;
        bool cut = false;   // p or q has cut within what is known
        for (int i = begin; i < end; ++i) {
            const bool in = i == 0 || ((!(plan.p < 1.0) || run < plan.p * W) && z_of(i) >= log_q);
            keep += in ? 1 : 0;
            cut = cut || !in;
            run += weight[i];
        }
        keep = over_ints(keep, Add());
        // without a top-k, the rank behind the last known one has to be out as well
        if (plan.p < 1.0 && plan.k == 0 && !(listed_mass < plan.p * W)) cut = true;
        const bool settled = __syncthreads_or(cut && mass_known) || enough;
        if (!settled) {
            leave();
            continue;
        }
        mine = 0.0;
        for (int i = begin; i < min(end, keep); ++i) mine += weight[i];
        const double kept = total_of(mine);
        const double target = u < 1.0 ? u * kept : HUGE_VAL;
        int first = 0x7FFFFFFF, last = -1;
        if (keep > kFinish / 4) {
            // by index: token and rank in one key, then running sums (by
            // pairs, as below, 64 rows of 50257 take 48 us and not 42)
            __syncthreads();
            for (int i = tid; i < keep; i += kFinish) {
                const uint64_t token = static_cast<uint64_t>(entry_token(keys[i]));
                keys[i] = ~(token << 32 | static_cast<uint64_t>(i));
            }
            sort_by<kFinish>(keys, keep);
            const int some = (keep + kFinish - 1) / kFinish;
            const int from = min(keep, some * tid), until = min(keep, from + some);
            double own = 0.0;
            for (int i = from; i < until; ++i) own += weight[~keys[i] & 0xFFFFFFFFu];
            double at = before_of(own);
            for (int i = from; i < until; ++i) {
                const double w = weight[~keys[i] & 0xFFFFFFFFu];
                at += w;
                if (w > 0.0) {
                    last = static_cast<int>(~keys[i] >> 32);
                    if (first == 0x7FFFFFFF && at > target) first = last;
                }
            }
        } else {
            for (int i = tid; i < keep; i += kFinish) {
                const int own = entry_token(keys[i]);
                double sum = 0.0;
                for (int j = 0; j < keep; ++j) sum += entry_token(keys[j]) <= own ? weight[j] : 0.0;
                if (weight[i] > 0.0) {
                    last = max(last, own);
                    if (sum > target) first = min(first, own);
                }
            }
        }
        first = over_ints(first, Min());
        last = over_ints(last, Max());
        if (tid == 0) *out = first < 0x7FFFFFFF ? first : last;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Distillation
// ---------------------------------------------------------------------------
// What a call keeps of its rows between its kernels (and for a backward).
struct SlotState {     // a teacher's slot
    int token;         // -1: empty, or another slot of this token stands for it
    float x;           // the student's logit
    float q;           // the token's probability, all its slots together
    int unused;
};
struct RowState {
    double Q;          // sum of q
    double C;          // sum of q (l - ln 2 c2 (x - best_listed)), slot by slot
    float best_listed; // maximum of the listed logits, -inf without any
    float listed;      // sum of their exponentials 2^(c2 (x - best_listed))
    float best_rest;   // the same over all other logits
    float rest;
};
struct DistillState {
    SlotState* slots;  // [rows, n]
    RowState* rows;    // [rows]
    int* any;          // [rows]: the row has slots
    int* done;         // clusters that have finished their rows
};

__host__ __device__ __forceinline__ DistillState state_of(const DistillArgs& a) {
    DistillState s;
    char* p = static_cast<char*>(a.state);
    s.slots = reinterpret_cast<SlotState*>(p);
    p += static_cast<int64_t>(a.in.rows) * a.n * static_cast<int64_t>(sizeof(SlotState));
    s.rows = reinterpret_cast<RowState*>(p);
    p += a.in.rows * static_cast<int64_t>(sizeof(RowState));
    s.any = reinterpret_cast<int*>(p);
    s.done = s.any + a.in.rows;
    return s;
}

__device__ __forceinline__ int64_t teacher_token(const DistillArgs& a, int64_t at) {
    return a.token_bytes == 8 ? static_cast<const int64_t*>(a.teacher_tokens)[at]
                              : static_cast<int64_t>(static_cast<const int32_t*>(a.teacher_tokens)[at]);
}

template <class T, class Op>
__device__ __forceinline__ T reduce_block(T v, Op op, T* scratch) {   // any number of warps; scratch: 32 values
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < static_cast<int>(blockDim.x) / 32; ++w) v = op(v, scratch[w]);
    __syncthreads();
    return v;
}

// The teacher's slots, kGroup threads a row with kPer slots each (a warp, or a
// CTA where the slots are many): everything that takes a thread a while is
// done here, for all rows at once, and not between the barriers of the rows'
// pass. The first slot of a token stands for all of its slots. Two bit maps of
// the tokens' hashes (a bit for each of `mask` + 1 values) tell that no token
// is listed twice; where they cannot (one row in 250 with 64 slots), the
// tokens are compared. Atomics of several threads may come in any order, so
// the maps are filled in three steps: all slots enter the first one; those
// that were the first on their bit enter the second; the others, of which
// every token listed twice has at least one, are looked up there and entered.
// Of two slots of a token the later one in this order meets the earlier one's
// bits in both maps. (Both maps in one step let two threads each be the first
// in one of them, and none saw the other.)
template <class E, int kGroup, int kPer>
__global__ void __launch_bounds__(256) slots_kernel(DistillArgs a, uint32_t mask) {
    constexpr int kRows = 256 / kGroup;   // of a CTA
    extern __shared__ uint4 dyn[];
    __shared__ double d8[32];
    __shared__ float f8[32];
    const int group = threadIdx.x / kGroup, tid = threadIdx.x % kGroup;
    uint32_t* map = reinterpret_cast<uint32_t*>(dyn) + group * ((mask + 1) / 16);
    uint32_t* map2 = map + (mask + 1) / 32;
    const DistillState state = state_of(a);
    const int n = a.n;
    const float c2 = fminf(1.4426950408889634f / a.temperature, FLT_MAX);
    const double tab = exp_table();
    auto sync = [&]() {
        if (kGroup == 32)
            __syncwarp();
        else
            __syncthreads();
    };
    auto over = [&](auto v, auto op, auto* scratch) {
        if (kGroup == 32) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(kAll, v, o));
            return v;
        }
        return reduce_block(v, op, scratch);
    };
    auto some = [&](bool v) { return kGroup == 32 ? __any_sync(kAll, v) != 0 : __syncthreads_or(v) != 0; };
    for (int i = tid; i < static_cast<int>((mask + 1) / 16); i += kGroup) map[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *state.done = 0;
    sync();
    for (int64_t row = blockIdx.x * static_cast<int64_t>(kRows) + group; row < a.in.rows;
         row += gridDim.x * static_cast<int64_t>(kRows)) {
        const E* x = static_cast<const E*>(a.in.x) + row * a.in.stride;
        // this thread's slots, their loads in flight together
        int64_t i[kPer];
        float l[kPer];
        SlotState slot[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int j = tid + k * kGroup;
            i[k] = -1;
            l[k] = 0.0f;
            if (j < n) {
                i[k] = teacher_token(a, row * n + j);
                l[k] = a.teacher_log_probs[row * n + j];
            }
        }
        float best = neg_inf();
        bool any = false;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            slot[k] = SlotState{-1, neg_inf(), 0.0f, 0};
            if (i[k] >= 0 && i[k] < a.in.V) {
                any = true;
                slot[k].token = static_cast<int>(i[k]);
                slot[k].x = Elem<E>::widen(x[i[k]]);
            }
        }
        double Q = 0.0;
        bool maybe = false;
        uint32_t h[kPer];
        bool met[kPer];    // not the first on its bit of the first map
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            // log-probs above 709 are infinite, those below -708 nothing
            const float t = fminf(fmaxf(l[k] * 46.16624f, -40000.0f), 40000.0f);
            const int steps = __float_as_int(t + 12582912.0f) - 0x4B400000;
            double q = exp_by(static_cast<double>(l[k]), 46.166241308446828384, steps, tab);
            if (!(l[k] >= -708.0f)) q = l[k] < -708.0f ? 0.0 : static_cast<double>(l[k]);
            if (l[k] > 709.0f) q = HUGE_VAL;
            if (slot[k].token >= 0) {
                slot[k].q = static_cast<float>(q);
                Q += q;
                h[k] = static_cast<uint32_t>(slot[k].token) * 2654435761u;
                const uint32_t h1 = h[k] >> 7 & mask;
                met[k] = atomicOr(&map[h1 >> 5], 1u << (h1 & 31u)) >> (h1 & 31u) & 1u;
            }
            best = fmaxf(best, slot[k].x);
        }
        sync();
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t h2 = h[k] >> 15 & mask;
            if (slot[k].token >= 0 && !met[k]) atomicOr(&map2[h2 >> 5], 1u << (h2 & 31u));
        }
        sync();
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t h2 = h[k] >> 15 & mask;
            if (slot[k].token >= 0 && met[k])
                maybe = (atomicOr(&map2[h2 >> 5], 1u << (h2 & 31u)) >> (h2 & 31u) & 1u) || maybe;
        }
        any = some(any);
        best = over(best, Max(), f8);
        Q = over(Q, Add(), d8);
        bool owner[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) owner[k] = slot[k].token >= 0;
        if (some(maybe)) {
            // owner: no earlier slot has the token; i: what its slots have together
#pragma unroll
            for (int k = 0; k < kPer; ++k) i[k] = 0;
            auto meet = [&](int token, float q, int o) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    if (token < 0 || token != slot[k].token) continue;
                    owner[k] = owner[k] && o >= tid + k * kGroup;
                    i[k] = __float_as_int(__int_as_float(static_cast<int>(i[k])) + q);
                }
            };
            if (kGroup == 32) {
#pragma unroll
                for (int k = 0; k < kPer; ++k)
                    for (int o = 0; o < 32; ++o)
                        meet(__shfl_sync(kAll, slot[k].token, o), __shfl_sync(kAll, slot[k].q, o), o + 32 * k);
            } else {
                for (int o = 0; o < n; ++o) {
                    const int64_t token = teacher_token(a, row * n + o);
                    if (token >= 0 && token < a.in.V)
                        meet(static_cast<int>(token),
                             static_cast<float>(exp(static_cast<double>(a.teacher_log_probs[row * n + o]))), o);
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k) i[k] = __float_as_int(slot[k].q);
        }
        double C = 0.0;
        float listed = 0.0f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (slot[k].token < 0) continue;
            map[(h[k] >> 7 & mask) >> 5] = 0;   // all bits of the maps have been looked at
            map2[(h[k] >> 15 & mask) >> 5] = 0;
            if (slot[k].q != 0.0f) {
                const double z = slot[k].x == best ? 0.0 : static_cast<double>(slot[k].x) - static_cast<double>(best);
                C += static_cast<double>(slot[k].q) *
                     (static_cast<double>(l[k]) - 0.69314718055994530942 * static_cast<double>(c2) * z);
            }
            if (owner[k]) listed += share(slot[k].x, best, c2);
            slot[k].q = __int_as_float(static_cast<int>(i[k]));
            if (!owner[k]) slot[k].token = -1;
        }
        listed = over(listed, Add(), f8);
        C = over(C, Add(), d8);
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (tid + k * kGroup < n) state.slots[row * n + tid + k * kGroup] = slot[k];
        if (tid == 0) {
            state.rows[row] = RowState{Q, C, best, listed, neg_inf(), 0.0f};
            state.any[row] = any ? 1 : 0;
        }
        sync();
    }
}

// Is there a rest's class: is P_r, a sum `rest` of exponentials by the reference
// `best_rest` beside the row's `all`, above 0? As in 64 bits: what is below
// 2^-1075 of the row's maximum (to the octave) is nothing, so that tokens
// masked by their type's lowest value make no class of their own.
__device__ __forceinline__ bool has_rest(float rest, float best_rest, float all, float c2) {
    const int octaves = (__float_as_int(rest) >> 23) - 127;
    return rest > 0.0f && (all == best_rest || (all - best_rest) * c2 < static_cast<float>(1075 + octaves));
}

// A row's loss from its sums. Other CTAs have written them: past L1.
__device__ double row_loss(const DistillArgs& a, const DistillState& state, int64_t row, double c) {
    const RowState* at = state.rows + row;
    const RowState s = {__ldcg(&at->Q), __ldcg(&at->C), __ldcg(&at->best_listed), __ldcg(&at->listed),
                        __ldcg(&at->best_rest), __ldcg(&at->rest)};
    const float all = fmaxf(s.best_listed, s.best_rest);
    auto by = [&](float best, float v) {   // a sum by the row's maximum
        return v == 0.0f ? 0.0 : static_cast<double>(v) *
                   (best == all ? 1.0 : exp(c * (static_cast<double>(best) - static_cast<double>(all))));
    };
    const double Z = by(s.best_rest, s.rest) + by(s.best_listed, s.listed);
    if (Z == 0.0) return s.Q > 0.0 ? static_cast<double>(INFINITY) : 0.0;   // nothing above -inf
    const float c2 = fminf(1.4426950408889634f / a.temperature, FLT_MAX);
    const double left = a.tail && has_rest(s.rest, s.best_rest, all, c2) ? fmax(0.0, 1.0 - s.Q) : 0.0;
    // log P = c (x - all) - log Z
    double loss = s.C;
    if (s.Q != 0.0) {
        const double up = all == s.best_listed ? 0.0 : static_cast<double>(all) - static_cast<double>(s.best_listed);
        loss += s.Q * (log(Z) + c * up);
    }
    if (left > 0.0) {
        const double down = all == s.best_rest ? 0.0 : static_cast<double>(all) - static_cast<double>(s.best_rest);
        loss += left * (log(left * Z / static_cast<double>(s.rest)) + c * down);
    }
    return loss;
}

// The losses of rows first, first + step, ..., and this CTA's part of their
// sum and number.
__device__ void add_losses(const DistillArgs& a, const DistillState& state, int64_t first, int64_t step, double* d32,
                           int* i32, double& sum, int& count) {
    const double c = static_cast<double>(fminf(1.4426950408889634f / a.temperature, FLT_MAX)) * 0.69314718055994530942;
    sum = 0.0;
    count = 0;
    for (int64_t row = first; row < a.in.rows; row += step) {
        const bool any = state.any[row] != 0;
        const double loss = any ? row_loss(a, state, row, c) : 0.0;
        count += any ? 1 : 0;
        sum += static_cast<double>(static_cast<float>(loss));
        a.row_losses[row] = static_cast<float>(a.reduction == kNone ? loss * static_cast<double>(a.scale) : loss);
    }
    sum = reduce_block(sum, Add(), d32);
    count = reduce_block(count, Add(), i32);
}

__device__ float reduced_loss(const DistillArgs& a, double sum, int count) {
    sum *= static_cast<double>(a.scale);
    return static_cast<float>(a.reduction == kMean ? sum / static_cast<double>(max(1, count)) : sum);
}

// Many rows' losses, and their sum in 64 bits and one order. One cluster of 8
// CTAs.
__global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(1024) losses_kernel(DistillArgs a) {
    __shared__ double d32[32];
    __shared__ int i32[32];
    __shared__ double sums[8];
    __shared__ int counts[8];
    const Team team;
    const DistillState state = state_of(a);
    double sum;
    int count;
    add_losses(a, state, team.rank + static_cast<int64_t>(threadIdx.x) * 8, 8 * 1024, d32, i32, sum, count);
    if (a.reduction == kNone) return;
    cluster_sync(8);   // everybody has started
    if (threadIdx.x == 0) {
        *cg::this_cluster().map_shared_rank(sums + team.rank, 0) = sum;
        *cg::this_cluster().map_shared_rank(counts + team.rank, 0) = count;
    }
    cluster_sync(8);
    if (team.rank == 0 && threadIdx.x == 0) {
        sum = 0.0;
        count = 0;
        for (int i = 0; i < 8; ++i) {
            sum += sums[i];
            count += counts[i];
        }
        *a.loss = reduced_loss(a, sum, count);
    }
}

struct DistillShared {
    float2 box[2][kMaxCluster];   // reference and sum of the CTAs' slices
    float2 part[kWarps];          // and of the warps' vectors
    uint32_t end_marks[2];        // which of these are listed
    int i32[32];
    uint4 marks[2][kThreads];     // a bit for each of a thread's elements: those that are listed
    double d32[32];
    int last;
};

// One pass over the row gives its sum and (kGrad) its gradient: the logits are
// read once and the gradient written once. A thread copies, adds up and turns
// into gradients the same vectors of its CTA's slice in shared memory, and
// starts the copy of the next row's vector as soon as it has used one, so
// there are two barriers a row: for the row's sum, and before the listed
// places are written a second time. 64 KB of slice a CTA, three CTAs on an SM.
// Bound by latency at 24 warps an SM (barriers, the exponentials' pipe), with
// 14 instructions an element for sum and gradient, issue active in half of the
// cycles; 4096 rows of 128256 bf16, a tenth of them without a teacher, take
// about 410 of the call's 435 us, 4.9 TB/s of what is read and written. A slice
// that is not full costs nearly what a full one does (1025 rows of fp32: 12
// vectors a thread, 49152 elements a row, 93 us; 16 vectors, 65536, 115 us), and
// ends out of phase with 16 bytes 7 us there (50257 against 50256 elements).
// Also measured on the 4096 rows, in us: 655 with the slots and losses in this
// kernel (20 barriers a row), 666 by one CTA a row reading it twice (9 % of the
// second reads hit L2), 582 with the exponentials kept in registers, 518 with
// slices of 48 KB.
// What the teacher lists is not part of the sum, which must not be a
// difference of two sums (a tail of 1e-6 would be lost in it): a row ahead,
// the slots' threads name the listed elements to the threads that hold them,
// which make them -inf.
template <class E, bool kGrad>
__global__ void __launch_bounds__(kThreads, 3) distill_kernel(DistillArgs a, int S) {
    constexpr int kVec = Elem<E>::kVec;
    constexpr int kT = kThreads;
    constexpr int kChunk = 4;
    extern __shared__ uint4 dyn[];
    __shared__ DistillShared sh;
    // the backward of a loss that was not multiplied by anything: all is done
    if (a.skip_unit && a.grad_loss_stride == 0 && *a.grad_loss == 1.0f) return;
    const Team team;
    const DistillState state = state_of(a);
    const int n = a.n, V = a.in.V, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t step = gridDim.x / team.size;
    const float c2 = fminf(1.4426950408889634f / a.temperature, FLT_MAX);
    const float2 cc = make_float2(c2, c2);
    float unit = a.scale / a.temperature;
    if (kGrad && a.reduction == kMean) {
        int rows = 0;
        for (int64_t r = tid; r < a.in.rows; r += kT) rows += state.any[r];
        unit /= static_cast<float>(max(1, reduce_block(rows, Add(), sh.i32)));
    }
    sh.marks[0][tid] = sh.marks[1][tid] = make_uint4(0, 0, 0, 0);
    if (tid < 2) sh.end_marks[tid] = 0;
    cluster_sync(team.size);

    uint4* buf = dyn + tid;   // this thread's vectors, kT apart
    // Where a row's slice lies: positions count from the 16-byte boundary at
    // or before the row's first element; [v0, v1) are whole vectors, counted
    // from the slice's start, and elements outside them (`head` at its start,
    // then those from tail_at on) are the last warp's.
    struct View {
        const uint4* src;
        int a0, v0, v1, len;
    };
    auto view = [&](const E* x) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(x);
        const int phase = static_cast<int>((at & 15u) / sizeof(E));
        View w;
        w.a0 = team.rank * S - phase;   // token of the slice's element 0
        w.len = max(0, min(S, V - w.a0));
        w.v0 = team.rank == 0 && phase > 0 ? 1 : 0;
        w.v1 = w.len / kVec;
        w.src = reinterpret_cast<const uint4*>(at & ~static_cast<uintptr_t>(15)) + team.rank * (S / kVec);
        return w;
    };
    const E* in = static_cast<const E*>(a.in.x);
    auto name = [&](const SlotState& s, const View& w, int par) {
        const int e = s.token - w.a0;
        if (s.token < 0 || e < 0 || e >= w.len) return;
        const int head = min(w.len, w.v0 * kVec), tail_at = max(head, w.v1 * kVec);
        if (e < head || e >= tail_at) {
            atomicOr(&sh.end_marks[par], 1u << (e < head ? e : e - tail_at + head));
        } else {
            const int v = e / kVec - w.v0, bit = v / kT * kVec + e % kVec;
            atomicOr(reinterpret_cast<uint32_t*>(&sh.marks[par][v % kT]) + (bit >> 5), 1u << (bit & 31));
        }
    };
    const uint4 none = vneg_inf<E>();
    SlotState slot = {-1, 0.0f, 0.0f, 0};   // this thread's first slot of the next row
    auto name_all = [&](int64_t r, const View& w, int par) {
        if (tid < n) name(slot, w, par);
        for (int j = tid + kT; j < n; j += kT) name(state.slots[r * n + j], w, par);
    };

    const int64_t first_row = blockIdx.x / team.size;
    bool any_next = first_row < a.in.rows && state.any[first_row] != 0;
    bool any_after = first_row + step < a.in.rows && state.any[first_row + step] != 0;
    View next = view(in + first_row * a.in.stride);
    if (any_next) {
        if (tid < n) slot = state.slots[first_row * n + tid];
        for (int i = 0, v = next.v0 + tid; i < kHold; v += kT, ++i) {
            if (v < next.v1)
                copy_async(buf + i * kT, next.src + v);
            else
                buf[i * kT] = none;
        }
        name_all(first_row, next, 0);
    }
    copies_commit();
    __syncthreads();
    int parity = 0, turn = 0;
    for (int64_t row = first_row; row < a.in.rows; row += step) {
        const int par = parity;
        parity ^= 1;
        const bool any = any_next;
        any_next = any_after;
        any_after = row + 2 * step < a.in.rows && state.any[row + 2 * step] != 0;
        const View here = next;
        const SlotState mine = slot;
        next = view(in + (row + step) * a.in.stride);
        if (any_next && tid < n) slot = state.slots[(row + step) * n + tid];
        float g = 1.0f;
        if (kGrad && a.grad_loss) g = a.grad_loss[row * a.grad_loss_stride];
        E* out = static_cast<E*>(a.grad) + (kGrad ? row * V : 0);
        uint4* dst = reinterpret_cast<uint4*>(out + here.a0);
        const bool same_phase = kGrad && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0;
        dst += here.v0 + tid;
        const int count = (here.v1 - here.v0 - tid + kT - 1) / kT;   // of this thread's vectors
        const int next_count = any_next ? (next.v1 - next.v0 - tid + kT - 1) / kT : 0;
        const uint4* src = next.src + next.v0 + tid;   // only its first next_count vectors are read
        const int head = min(here.len, here.v0 * kVec), tail_at = max(head, here.v1 * kVec);
        const int ragged = lane < head ? lane : tail_at + lane - head;
        const bool at_end = warp == kWarps - 1 && ragged < here.len && here.a0 + ragged >= 0;
        auto copy_next = [&]() {
            for (int i = 0; i < kHold; ++i) {
                if (i < next_count)
                    copy_async(buf + i * kT, src + i * kT);
                else
                    buf[i * kT] = none;
            }
        };
        if (!any || (a.skip_unit && g == 1.0f)) {   // the same for the whole cluster
            if (any) {
                sh.marks[par][tid] = make_uint4(0, 0, 0, 0);
                if (tid == 0) sh.end_marks[par] = 0;
                copies_wait<0>();
            } else if (kGrad) {
                // a row without a teacher: gradient 0 whatever its logits hold
                if (same_phase)
                    for (int i = 0; i < count; ++i) __stcs(dst + i * kT, make_uint4(0, 0, 0, 0));
                else
                    for (int e = here.v0 * kVec + tid; e < here.v1 * kVec; e += kT)
                        out[here.a0 + e] = Elem<E>::narrow(0.0f);
                if (at_end) out[here.a0 + ragged] = Elem<E>::narrow(0.0f);
            }
            copy_next();
            copies_commit();
            if (any_next) {
                __syncthreads();   // the marks of two rows ago are gone
                name_all(row + step, next, parity);
            }
            __syncthreads();
            continue;
        }
        const RowState known = state.rows[row];
        copies_wait<0>();
        const uint4 marks = sh.marks[par][tid];
        if (marks.x | marks.y | marks.z | marks.w) {
            sh.marks[par][tid] = make_uint4(0, 0, 0, 0);
            const uint32_t word[4] = {marks.x, marks.y, marks.z, marks.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                for (uint32_t left = word[k]; left; left &= left - 1) {
                    const int bit = 32 * k + __ffs(left) - 1;
                    reinterpret_cast<E*>(buf + bit / kVec * kT)[bit % kVec] = Elem<E>::narrow(neg_inf());
                }
            }
        }
        float end_x = neg_inf();
        if (at_end && !(sh.end_marks[par] >> lane & 1u)) end_x = Elem<E>::widen(in[row * a.in.stride + here.a0 + ragged]);
        // The sum goes by the maximum of the thread's first vectors; where the
        // others run so far beyond it that the sum passes 1e18, by all of them.
        // (Factors between such maxima come out as 0 below 2^-126, so what is
        // lost of the row's sum is below 2^-50.)
        auto best_of = [&](int chunks) {
            uint4 top = none;
            for (int i = 0; i < chunks * kChunk; ++i) top = vmax<E>(top, buf[i * kT]);
            return lanes_max<E>(top);
        };
        const int chunks = (count + kChunk - 1) / kChunk;   // the last one is filled up with -inf
        float best = neg_inf(), sum = 0.0f;
        auto add_up = [&]() {
            const float from = best > neg_inf() ? -best : 0.0f;
            const float2 ff = make_float2(from, from);
            float2 p = make_float2(0.0f, 0.0f);
            const uint4* at = buf;
            for (int i = 0; i < chunks; ++i, at += kChunk * kT) {
                uint4 r[kChunk];
#pragma unroll
                for (int k = 0; k < kChunk; ++k) r[k] = at[k * kT];
#pragma unroll
                for (int k = 0; k < kChunk; ++k) {
                    float f[kVec];
                    Elem<E>::unpack(r[k], f);
#pragma unroll
                    for (int m = 0; m < kVec; m += 2) {
                        const float2 t = mul2(add2(make_float2(f[m], f[m + 1]), ff), cc);
                        p = add2(p, make_float2(ex2(t.x), ex2(t.y)));
                    }
                }
            }
            sum = p.x + p.y + (at_end ? ex2((end_x + from) * c2) : 0.0f);
        };
        best = fmaxf(best_of(min(chunks, 1)), end_x);
        add_up();
        if (!(best > neg_inf()) || !(sum < 1.0e18f)) {
            best = fmaxf(best_of(chunks), end_x);
            add_up();
        }
        // over the warp, the CTA and the cluster: references, and sums by them
        float2 rest = make_float2(best, sum);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) rest.x = fmaxf(rest.x, __shfl_xor_sync(kAll, rest.x, o));
        rest.y = sum == 0.0f ? 0.0f : sum * share(best, rest.x, c2);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) rest.y += __shfl_xor_sync(kAll, rest.y, o);
        if (lane == 0) sh.part[warp] = rest;
        __syncthreads();
        auto join = [&](const float2* parts, int size) {
            float2 all = make_float2(neg_inf(), 0.0f);
            for (int i = 0; i < size; ++i) all.x = fmaxf(all.x, parts[i].x);
            const float from = all.x > neg_inf() ? -all.x : 0.0f;
            for (int i = 0; i < size; ++i) all.y += parts[i].y * ex2((parts[i].x + from) * c2);
            return all;
        };
        if (tid == 0) sh.end_marks[par] = 0;
        if (team.size == 1 || warp == 0) rest = join(sh.part, kWarps);
        if (team.size > 1) {
            if (warp == 0) {
                if (lane < team.size) *cg::this_cluster().map_shared_rank(&sh.box[turn][team.rank], lane) = rest;
                cluster_arrive();
            } else {
                cluster_arrive_relaxed();
            }
        }
        if (any_next) name_all(row + step, next, parity);
        if (team.size > 1) {
            cluster_wait();
            rest = join(sh.box[turn], team.size);
            turn ^= 1;
        }
        if (tid == 0 && team.rank == 0 && !a.skip_state) {
            state.rows[row].best_rest = rest.x;
            state.rows[row].rest = rest.y;
        }
        if (kGrad) {
            const float all = fmaxf(rest.x, known.best_listed);
            const float Z = (rest.y == 0.0f ? 0.0f : rest.y * share(rest.x, all, c2)) +
                            (known.listed == 0.0f ? 0.0f : known.listed * share(known.best_listed, all, c2));
            const float q_rest =
                a.tail && has_rest(rest.y, rest.x, all, c2) ? static_cast<float>(fmax(0.0, 1.0 - known.Q)) : 0.0f;
            const float w = unit * g;
            const float G = (static_cast<float>(known.Q) + q_rest) * (Z == 0.0f ? 0.0f : __fdividef(1.0f, Z));
            // P / P_r = exponential by the rest's reference / its sum, and P =
            // exponential by the row's / Z. With a rest's class both go by the
            // rest's, where P may be lost next to P / P_r; without one by the
            // row's, so that the smallest P stays. (By a thread's own, a factor
            // to the row's of 2^-126 took all of its elements' gradients.)
            const float by = q_rest > 0.0f ? rest.x : all;
            float scale = G;
            if (q_rest > 0.0f) scale = G * share(rest.x, all, c2) - __fdividef(q_rest, rest.y);
            scale *= w;
            const float from = by > neg_inf() ? -by : 0.0f;
            const float2 ff = make_float2(from, from), ss = make_float2(scale, scale);
            auto gradient = [&](const uint4& r) {
                float f[kVec];
                Elem<E>::unpack(r, f);
#pragma unroll
                for (int k = 0; k < kVec; k += 2) {
                    const float2 t = mul2(add2(make_float2(f[k], f[k + 1]), ff), cc);
                    const float2 y = mul2(make_float2(ex2(t.x), ex2(t.y)), ss);
                    f[k] = y.x;
                    f[k + 1] = y.y;
                }
                return Elem<E>::pack(f);
            };
            if (same_phase) {
                uint4* at = buf;
                for (int i = 0; i < kHold; i += kChunk, at += kChunk * kT, dst += kChunk * kT, src += kChunk * kT) {
                    uint4 r[kChunk];
                    if (i + kChunk <= min(count, next_count)) {
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) r[k] = at[k * kT];
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) r[k] = gradient(r[k]);
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) {
                            copy_async(at + k * kT, src + k * kT);
                            __stcs(dst + k * kT, r[k]);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) r[k] = i + k < count ? at[k * kT] : none;
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) r[k] = gradient(r[k]);
#pragma unroll
                        for (int k = 0; k < kChunk; ++k) {
                            if (i + k < next_count)
                                copy_async(at + k * kT, src + k * kT);
                            else
                                at[k * kT] = none;
                            if (i + k < count) __stcs(dst + k * kT, r[k]);
                        }
                    }
                }
            } else {
                for (int k = 0; k < count; ++k) {
                    const uint4 r = gradient(buf[k * kT]);
                    const E* f = reinterpret_cast<const E*>(&r);
#pragma unroll
                    for (int m = 0; m < kVec; ++m) out[here.a0 + (here.v0 + tid + k * kT) * kVec + m] = f[m];
                }
                copy_next();
            }
            copies_commit();
            if (at_end) out[here.a0 + ragged] = Elem<E>::narrow(ex2((end_x + from) * c2) * scale);
            __syncthreads();   // the listed places are written a second time
            auto listed = [&](const SlotState& s) {
                const int at = s.token - here.a0;
                if (s.token >= 0 && at >= 0 && at < here.len)
                    out[s.token] = Elem<E>::narrow(fmaf(share(s.x, all, c2), G * w, -s.q * w));
            };
            if (tid < n) listed(mine);
            for (int j = tid + kT; j < n; j += kT) listed(state.slots[row * n + j]);
        } else {
            copy_next();
            copies_commit();
            __syncthreads();
        }
    }
    copies_wait<0>();
    if (a.join_losses && team.rank == 0) {
        // the cluster that finishes last has every row's sums
        if (tid == 0) {
            __threadfence();
            sh.last = atomicAdd(state.done, 1) == static_cast<int>(step) - 1 ? 1 : 0;
            __threadfence();
        }
        __syncthreads();
        if (sh.last) {
            double sum;
            int rows;
            add_losses(a, state, tid, kT, sh.d32, sh.i32, sum, rows);
            if (tid == 0 && a.reduction != kNone) *a.loss = reduced_loss(a, sum, rows);
        }
    }
    cluster_sync(team.size);
}

// ---------------------------------------------------------------------------
// Launchers
// ---------------------------------------------------------------------------
std::mutex g_mu;
std::vector<std::tuple<const void*, int, size_t>> g_smem;               // kernel, device: shared memory allowed
std::vector<std::tuple<const void*, int, size_t, int, int>> g_clusters;   // kernel, device, smem, size: resident

// How a row is cut: CTAs per row and elements per slice.
struct Shape {
    int size;
    int S;
};

// Slices of up to 64 KB (distillation; 68 KB else) let two or three CTAs share
// an SM, so that one's loads, one's arithmetic and one's stores overlap. Few
// rows are cut finer, down to 8 KB, so that they reach more SMs; 16 CTAs (more
// than every GPU grants a cluster) are taken only for rows that need them (256
// rows with their own settings, of which 3 are left to clusters: 116 us with 8
// CTAs, 119 with 16).
Shape shape_of(const Rows& in, int es, int most, bool few = false) {
    const int vec = 16 / es;
    auto slice = [&](int size) {
        const int64_t per = (static_cast<int64_t>(in.V) + vec - 1 + size - 1) / size;
        return static_cast<int>((per + 63) / 64 * 64);
    };
    int size = 1;
    while (size < 8 && static_cast<int64_t>(slice(size)) * es > most) ++size;
    if (static_cast<int64_t>(slice(size)) * es > most) size = 16;
    if (few && size < 8) size = 8;   // a handful of rows out of many: one row's time counts
    while (size <= 4 && in.rows * size * 2 <= 148 && static_cast<int64_t>(slice(size)) * es > 8 * 1024) size *= 2;
    return Shape{size, slice(size)};
}

template <class Kernel, class... Args>
cudaError_t launch_rows(Kernel kernel, const Rows& in, int size, size_t smem, cudaStream_t stream, int threads,
                        Args... args) {
    const void* fn = reinterpret_cast<const void*>(kernel);
    int dev = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(size);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int resident = 0;
    {
        std::lock_guard<std::mutex> lock(g_mu);
        bool known = false;
        for (auto& e : g_smem) {
            if (std::get<0>(e) != fn || std::get<1>(e) != dev) continue;
            known = true;
            if (std::get<2>(e) < smem) {
                err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
                if (err != cudaSuccess) return err;
                std::get<2>(e) = smem;
            }
        }
        if (!known) {
            err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (err == cudaSuccess) err = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           static_cast<int>(cudaSharedmemCarveoutMaxShared));
            if (err != cudaSuccess) return err;
            g_smem.emplace_back(fn, dev, smem);
        }
        for (auto& e : g_clusters)
            if (std::get<0>(e) == fn && std::get<1>(e) == dev && std::get<2>(e) == smem && std::get<3>(e) == size)
                resident = std::get<4>(e);
        if (resident == 0) {
            cfg.gridDim = dim3(static_cast<unsigned>(size));
            err = cudaOccupancyMaxActiveClusters(&resident, fn, &cfg);
            if (err != cudaSuccess) return err;
            if (resident <= 0) return cudaErrorInvalidConfiguration;
            g_clusters.emplace_back(fn, dev, smem, size, resident);
        }
    }
    const int64_t clusters = std::min<int64_t>(in.rows, resident);
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * size));
    return dbs_dev::count_launch(cudaLaunchKernelEx(&cfg, kernel, args...));
}

int element_size(int dtype) { return dtype == kF32 ? 4 : 2; }

int list_space(int n) {
    int cap = kBins / 2;
    while (cap < 2 * n) cap *= 2;
    return std::max(cap, 3 * kBins / 4);   // both lists' space also holds the bins of a search
}

template <class E>
cudaError_t launch_distill_typed(const DistillArgs& a, cudaStream_t stream) {
    const Shape sh = shape_of(a.in, sizeof(E), kThreads * kHold * 16);
    const size_t smem = static_cast<size_t>(kThreads) * kHold * 16;
    return a.grad ? launch_rows(distill_kernel<E, true>, a.in, sh.size, smem, stream, kThreads, a, sh.S)
                  : launch_rows(distill_kernel<E, false>, a.in, sh.size, smem, stream, kThreads, a, sh.S);
}

template <class E>
cudaError_t launch_slots(const DistillArgs& a, cudaStream_t stream) {
    const unsigned warps = static_cast<unsigned>(std::min<int64_t>((a.in.rows + 7) / 8, 148 * 8));
    if (a.n <= 32) {
        slots_kernel<E, 32, 1><<<warps, 256, 8 * 2048, stream>>>(a, 8192 - 1);
    } else if (a.n <= 64) {
        slots_kernel<E, 32, 2><<<warps, 256, 8 * 2048, stream>>>(a, 8192 - 1);
    } else if (a.n <= 128) {
        slots_kernel<E, 32, 4><<<warps, 256, 8 * 2048, stream>>>(a, 8192 - 1);
    } else {
        static_assert(kMaxTop <= 4 * 256, "four slots per thread");
        const unsigned ctas = static_cast<unsigned>(std::min<int64_t>(a.in.rows, 148 * 8));
        slots_kernel<E, 256, 4><<<ctas, 256, 32768, stream>>>(a, 131072 - 1);
    }
    return dbs_dev::count_launch(cudaGetLastError());
}

cudaError_t launch_distill_any(const DistillArgs& a, cudaStream_t stream) {
    switch (a.in.dtype) {
        case kF32: return launch_distill_typed<float>(a, stream);
        case kF16: return launch_distill_typed<__half>(a, stream);
        default: return launch_distill_typed<__nv_bfloat16>(a, stream);
    }
}

}  // namespace

namespace {

constexpr int kScanTop = 256;   // the longest list of top_log_probs that a scan gathers

// Parts of at most 16 chunks; more of them where the rows are few or the lists
// long (a list of its part's share should take less than half of its threads).
ScanShape scan_shape(const Rows& in, int es, int take) {
    const int chunk = kThreads * 16 / es;
    const int chunks = (in.V + 16 / es - 1 + chunk - 1) / chunk;
    int parts = (chunks + kHold - 1) / kHold;
    while (parts < chunks && parts < kMaxParts && (parts * 100 < take || in.rows * parts < 148 * 2)) ++parts;
    const float mean = static_cast<float>(take) / static_cast<float>(parts);
    const int cap = (static_cast<int>(4.0f * mean + 12.0f * sqrtf(mean)) + 96) / 2 * 2;
    return ScanShape{parts, cap};
}

// Which batches are scanned, by three launches, and which go to the cluster's
// kernel at once. Where a list is enough (`lists`) its clusters are many on an
// SM, and only rows of more than a CTA's slice gain, once they are many, or
// where a row needs more than eight CTAs. Sums in 64 bits (a top-p without a
// top-k, temperature alone) gain earlier; with settings of each row (`both`)
// rows have to be longer. Measured in us, scan against cluster's kernel, bf16:
//   top_k 50: 512 x 32000 37 / 26, 64 x 128256 18 / 14, 128 x 128256 23 / 28, 512 x 128256 59 / 101
//   n = 64: 512 x 32000 31 / 28, 1024 x 32000 47 / 50, 2048 x 32000 79 / 89, 4096 x 32000 150 / 172, 48 x 128256 16 / 15,
//     2048 x 128256 186 / 385; one row of 256000 fp32, n = 128, 12.7 / 16.6
//   temperature alone: 128 x 32000 19 / 16, 400 x 16384 26 / 33, 512 x 128256 109 / 264; one of 200000 12.6 / 18.0
//   top_p 0.9, min_p 0.02: 64 x 32000 47 / 37, 16 x 128256 35 / 70, 32 x 128256 40 / 53, 64 x 128256 52 / 99; one of 200000 20 / 52
//   top_p 0.9 alone: 64 x 32000 92 / 38, 16 x 128256 74 / 71, 32 x 128256 82 / 54, 64 x 128256 128 / 104; one of 200000 61 / 56
//   each row's own: 1024 x 8192 142 / 131, 64 x 32000 52 / 37, 256 x 32000 84 / 89, 256 x 128256 114 / 225
// Where the rule takes the slower side: n = 64 of 1024 rows of 32000 and more (by 6 to 15 %; one border serves top_k and n,
// and top_k loses there), up to 38 rows of 128256 with top-p and min-p, and a top-p alone whose rows are flat, as these are
// (their nuclei are longer than the list, so that they are looked through twice), which a rule on sizes cannot tell.
bool scans(const Rows& in, bool lists, bool both) {
    if (in.rows > INT_MAX) return false;   // the list of rows left over holds ints
    const int es = element_size(in.dtype);
    const int64_t row = static_cast<int64_t>(in.V) * es, all = in.rows * row;
    if (row + 16 > static_cast<int64_t>(kMaxParts) * kHold * kThreads * 16) return false;
    if (lists) return row > 520 * 1024 || (row > 68 * 1024 && all >= 20000000);
    return row > 256 * 1024 || (row >= (both ? 48 : 16) * 1024 && all >= 10000000);
}

// A top-k for every row, short enough for a list.
bool by_lists(const SampleArgs& a) {
    return !a.top_k && a.top_k_all > 0 && a.top_k_all <= kSampleList && a.top_k_all < a.in.V;
}

int sample_take(const SampleArgs& a) {
    const bool by_p = a.top_p || a.top_p_all < 1.0f;
    return a.top_k ? (by_p ? 384 : 128) : a.top_k_all > 0 ? std::min(a.top_k_all, kSampleList) : by_p ? kNucleus : 1;
}

int64_t scan_bytes(const Rows& in, ScanShape sh, bool chunks) {
    return in.rows * (sh.parts * (static_cast<int64_t>(sizeof(PartState)) + sh.cap * 8LL +
                                  (chunks ? kHold * kWarps * 8LL : 0LL)) + 4) + 64;
}

template <class E, class Args, bool kTop>
cudaError_t launch_scan(const Args& a, ScanShape sh, bool chunks, cudaStream_t stream) {
    Rows items = a.in;   // a CTA takes a part at a time
    items.rows *= sh.parts;
    return launch_rows(scan_kernel<E, Args, kTop>, items, 1, static_cast<size_t>(kThreads) * kHold * 16, stream,
                       kThreads, a, sh, a.space, chunks);
}

template <class Kernel, class Args>
cudaError_t launch_finish(Kernel kernel, const Args& a, ScanShape sh, bool chunks, int threads, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(sh.parts) * sh.cap * 16;
    return launch_rows(kernel, a.in, 1, smem, stream, threads, a, sh, a.space, chunks);
}

template <int kTeam>
cudaError_t launch_sample_rows(const SampleArgs& a, Shape sh, int cap, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(sh.S) * element_size(a.in.dtype) + static_cast<size_t>(cap) * 16;
    auto launch = [&](auto kernel) { return launch_rows(kernel, a.in, sh.size, smem, stream, kTeam, a, sh.S, cap); };
    switch (a.in.dtype) {
        case kF32: return launch(sample_kernel<kTeam, float>);
        case kF16: return launch(sample_kernel<kTeam, __half>);
        default: return launch(sample_kernel<kTeam, __nv_bfloat16>);
    }
}

}  // namespace

int64_t sample_space(const SampleArgs& a) {
    // a longer top-k is the cluster's kernel's for every row
    const bool long_list = !a.top_k && a.top_k_all > kSampleList && a.top_k_all < a.in.V;
    if (long_list || !scans(a.in, by_lists(a), a.top_k != nullptr)) return 0;
    // the chunks' sums are for rows with a temperature alone
    return scan_bytes(a.in, scan_shape(a.in, element_size(a.in.dtype), sample_take(a)), !by_lists(a));
}

int64_t top_space(const TopArgs& a) {
    if (a.n > kScanTop || !scans(a.in, true, false)) return 0;
    return scan_bytes(a.in, scan_shape(a.in, element_size(a.in.dtype), a.n), false);
}

cudaError_t launch_sample(const SampleArgs& given, cudaStream_t stream) {
    SampleArgs a = given;
    // a ratio alone, or the best token, needs no sum of its row: as lists do
    const bool greedy = !a.temperature && !(a.temperature_all > 0.0f);
    const bool ratio = !a.top_k && (a.top_k_all <= 0 || a.top_k_all >= a.in.V) && !a.top_p && a.top_p_all >= 1.0f &&
                       !a.min_p && a.min_p_all > 0.0f;
    const bool lists = greedy || by_lists(a);
    if (sample_space(a) > 0 && !ratio && scans(a.in, lists, a.top_k != nullptr)) {
        const ScanShape scan = scan_shape(a.in, element_size(a.in.dtype), sample_take(a));
        const bool chunks = !by_lists(a);
        cudaError_t err;
        switch (a.in.dtype) {
            case kF32:
                err = launch_scan<float, SampleArgs, false>(a, scan, chunks, stream);
                if (err == cudaSuccess) err = launch_finish(sample_finish_kernel<float>, a, scan, chunks, 512, stream);
                break;
            case kF16:
                err = launch_scan<__half, SampleArgs, false>(a, scan, chunks, stream);
                if (err == cudaSuccess) err = launch_finish(sample_finish_kernel<__half>, a, scan, chunks, 512, stream);
                break;
            default:
                err = launch_scan<__nv_bfloat16, SampleArgs, false>(a, scan, chunks, stream);
                if (err == cudaSuccess) err = launch_finish(sample_finish_kernel<__nv_bfloat16>, a, scan, chunks, 512, stream);
        }
        if (err != cudaSuccess) return err;
        a.left = scan_of(a.space, a.in.rows, scan, chunks).left;
    }
    const int es = element_size(a.in.dtype);
    const Shape sh = shape_of(a.in, es, 68 * 1024, a.left != nullptr);
    // lists for rows that may take that path, bins for the others
    const int cap = list_space(a.top_k ? kSampleList : (a.top_k_all <= kSampleList ? std::max(a.top_k_all, 0) : 0));
    return lists || ratio ? launch_sample_rows<kListTeam>(a, sh, cap, stream) : launch_sample_rows<kMassTeam>(a, sh, cap, stream);
}

cudaError_t launch_top(const TopArgs& given, cudaStream_t stream) {
    TopArgs a = given;
    if (top_space(a) > 0) {
        const ScanShape scan = scan_shape(a.in, element_size(a.in.dtype), a.n);
        cudaError_t err = a.in.dtype == kF32   ? launch_scan<float, TopArgs, true>(a, scan, false, stream)
                          : a.in.dtype == kF16 ? launch_scan<__half, TopArgs, true>(a, scan, false, stream)
                                               : launch_scan<__nv_bfloat16, TopArgs, true>(a, scan, false, stream);
        if (err == cudaSuccess) err = launch_finish(top_finish_kernel, a, scan, false, 256, stream);
        if (err != cudaSuccess) return err;
        a.left = scan_of(a.space, a.in.rows, scan, false).left;
    }
    const int es = element_size(a.in.dtype);
    const Shape sh = shape_of(a.in, es, 68 * 1024, a.left != nullptr);
    const int cap = list_space(a.n);
    const size_t smem = static_cast<size_t>(sh.S) * es + static_cast<size_t>(cap) * 16;
    switch (a.in.dtype) {
        case kF32: return launch_rows(top_kernel<kListTeam, float>, a.in, sh.size, smem, stream, kListTeam, a, sh.S, cap);
        case kF16: return launch_rows(top_kernel<kListTeam, __half>, a.in, sh.size, smem, stream, kListTeam, a, sh.S, cap);
        default: return launch_rows(top_kernel<kListTeam, __nv_bfloat16>, a.in, sh.size, smem, stream, kListTeam, a, sh.S, cap);
    }
}

// Rows up to which the pass itself adds up the losses at its end; a kernel of
// its own does it for more (at 2048 rows one CTA takes 15 us for them, the
// launch and its kernel 7 us).
constexpr int64_t kJoinRows = 512;

cudaError_t launch_distill(const DistillArgs& given, cudaStream_t stream) {
    DistillArgs a = given;
    a.join_losses = a.in.rows <= kJoinRows ? 1 : 0;
    if (a.in.rows > 0) {
        cudaError_t err = a.in.dtype == kF32   ? launch_slots<float>(a, stream)
                          : a.in.dtype == kF16 ? launch_slots<__half>(a, stream)
                                               : launch_slots<__nv_bfloat16>(a, stream);
        if (err == cudaSuccess) err = launch_distill_any(a, stream);
        if (err != cudaSuccess || a.join_losses) return err;
    } else if (a.reduction == kNone) {
        return cudaSuccess;
    }
    losses_kernel<<<8, 1024, 0, stream>>>(a);
    return dbs_dev::count_launch(cudaGetLastError());
}

cudaError_t launch_distill_backward(const DistillArgs& a, cudaStream_t stream) {
    return launch_distill_any(a, stream);
}

int64_t distill_state_bytes(int64_t rows, int n) {
    return rows * (n * static_cast<int64_t>(sizeof(SlotState)) + static_cast<int64_t>(sizeof(RowState)) + 4) + 16;
}

}  // namespace dbs_logits
