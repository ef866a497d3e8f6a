// What the norms' forward and backward kernels share: rows held in registers by teams of threads, their sums, and how a
// call's sizes choose a kernel.
//
// A team of threads owns a row at a time: each thread holds P packs of V elements in registers, so every row is read once and
// its sums need one exchange. Teams of 32 threads or less live in a warp (a power of two of lanes); larger ones are whole
// warps that meet at a named barrier of their own, so a block's teams never wait for one another. The rows that come next
// are on their way to shared memory meanwhile. Blocks stay on their SM and take row after row.
//
// Bound by memory in principle; what is reached is the rate of instructions and the latency of a row's two or three exchanges
// (the profiled kernels issue 1.05 to 2.0 of 4 instructions a cycle at 11 to 16 warps an SM, DRAM at 27 to 54 %): see the kernels
// for the times.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include <cuda_bf16.h>

#include "../../include/lamq_b200_step.h"
#include "lamq_common.cuh"

namespace lamq {

// The checks of a call's arguments (norm.cu): LAMQ_OK, or LAMQ_ERR_INVALID with the reason set.
int norm_args_status(const lamq_norm_args *a, bool backward);

namespace {

constexpr int kNormThreads = 512;   // most threads of a block

// The kernels: vectors or elements, 16 of a row a thread in teams of up to 256 (the full join's backward: 8 of a row in teams of
// up to 512); vectors in teams of up to 512, with 16 elements a thread and with 32; rows of elements by blocks (norm_wide.cuh).
enum NormKernel { kVectors, kElements, kVectors8, kElements8, kVectorsWide, kVectorsWidest, kWide };

enum { kNormAlone, kJoinPlain, kJoinFull };  // the norm alone; a join without post and gate; any join

// Threads that an SM holds: 85 registers each where the forward reads vectors and has no post norm and gate, else 128.
constexpr int resident(NormKernel kernel, int mode, bool backward) {
    return !backward && kernel == kVectors && mode != kJoinFull ? 768 : kNormThreads;
}

template <NormKernel kKernel>
struct NormSizes {
    static constexpr int E = kKernel == kVectorsWidest ? 32 : kKernel == kVectors8 || kKernel == kElements8 ? 8 : 16;
    static constexpr int V = kKernel == kElements || kKernel == kElements8 ? 1 : 8, P = E / V;
    static constexpr bool kHold = kKernel <= kElements8;  // weights and sums stay in registers
    static constexpr int kThreads = kHold ? 4096 / E : kNormThreads;
};
constexpr int kNormMaxD = 16384;    // widest row
constexpr int kNormSums = 3;        // sums exchanged at once
constexpr int kSMs = 148;

// ---- loads
//
// As volatile assembly, which the compiler runs only where the source does. What was seen: earlier kernels, with plain loads and
// __ldg behind a test of their pointer, faulted in two calls where tensors were absent (NULL), though the source then reads none
// of them; which load it was, and why, was not found. Since then all loads are these, absent tensors have a pointer that may be
// read (the host's `present`), and the kernels were written anew; every load of an absent tensor stands behind its flag.

__device__ __forceinline__ uint4 load16(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ float load_one(const float *p) {
    float v;
    asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ float load_one(const __nv_bfloat16 *p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return __uint_as_float((uint32_t)v << 16);
}

// ---- V elements of T: 16 bytes (bf16) or 32 (fp32) where V is 8, one element where rows may begin anywhere

template <typename T, int V>
struct Raw;

template <>
struct Raw<float, 8> {
    __device__ __forceinline__ static void unpack(const uint4 (&v)[2], float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[4 * i] = __uint_as_float(v[i].x), f[4 * i + 1] = __uint_as_float(v[i].y);
            f[4 * i + 2] = __uint_as_float(v[i].z), f[4 * i + 3] = __uint_as_float(v[i].w);
        }
    }
    __device__ __forceinline__ static void load(const float *p, float (&f)[8]) {
        const uint4 v[2] = {load16(p), load16(p + 4)};
        unpack(v, f);
    }
    __device__ __forceinline__ static void store(float *p, const float (&f)[8]) {
        // 32 bytes at once: two stores of 16 would each fill half of every sector they touch
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
                     "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                     : "memory");
    }
};

template <>
struct Raw<__nv_bfloat16, 8> {
    __device__ __forceinline__ static void unpack(const uint4 (&v)[1], float (&f)[8]) {
        const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ static void load(const __nv_bfloat16 *p, float (&f)[8]) {
        const uint4 v[1] = {load16(p)};
        unpack(v, f);
    }
    __device__ __forceinline__ static void store(__nv_bfloat16 *p, const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <typename T>
struct Raw<T, 1> {
    __device__ __forceinline__ static void load(const T *p, float (&f)[1]) { f[0] = load_one(p); }
    __device__ __forceinline__ static void store(float *p, const float (&f)[1]) { *p = f[0]; }
    __device__ __forceinline__ static void store(__nv_bfloat16 *p, const float (&f)[1]) { *p = __float2bfloat16_rn(f[0]); }
};

// V elements at index i of an array whose type is known when the call is made: weights, gates and their gradients.
template <int V>
__device__ __forceinline__ void load_typed(const void *base, int dtype, int64_t i, float (&f)[V]) {
    if (dtype == LAMQ_F32)
        Raw<float, V>::load(reinterpret_cast<const float *>(base) + i, f);
    else
        Raw<__nv_bfloat16, V>::load(reinterpret_cast<const __nv_bfloat16 *>(base) + i, f);
}

template <int V>
__device__ __forceinline__ void store_typed(void *base, int dtype, int64_t i, const float (&f)[V]) {
    if (dtype == LAMQ_F32)
        Raw<float, V>::store(reinterpret_cast<float *>(base) + i, f);
    else
        Raw<__nv_bfloat16, V>::store(reinterpret_cast<__nv_bfloat16 *>(base) + i, f);
}

// ---- what a thread holds of a row: E elements, worked on in pairs (one instruction for two)

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)),
          "l"(reinterpret_cast<const uint64_t &>(c)));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
    return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<const uint64_t &>(a)), "l"(reinterpret_cast<const uint64_t &>(b)));
    return d;
}

template <int E>
struct Vec {
    static constexpr int kPairs = (E + 1) / 2;
    float2 v[kPairs];  // the last half of an odd E is zero

    __device__ __forceinline__ Vec() {
        if constexpr (E % 2) v[kPairs - 1].y = 0.f;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = make_float2(0.f, 0.f);
    }
    // N elements from the Ith on (pairs, or one element)
    template <int N>
    __device__ __forceinline__ void set(int at, const float (&f)[N]) {
        if constexpr (N == 1) {
            if (at & 1)
                v[at / 2].y = f[0];
            else
                v[at / 2].x = f[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) v[(at + i) / 2] = make_float2(f[i], f[i + 1]);
        }
    }
    template <int N>
    __device__ __forceinline__ void get(int at, float (&f)[N]) const {
        if constexpr (N == 1) {
            f[0] = at & 1 ? v[at / 2].y : v[at / 2].x;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) f[i] = v[(at + i) / 2].x, f[i + 1] = v[(at + i) / 2].y;
        }
    }
    __device__ __forceinline__ void operator*=(float f) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = mul2(v[i], make_float2(f, f));
    }
    __device__ __forceinline__ void operator*=(const Vec &b) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = mul2(v[i], b.v[i]);
    }
    __device__ __forceinline__ void operator+=(const Vec &b) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = add2(v[i], b.v[i]);
    }
    // this + a·b
    __device__ __forceinline__ void add(const Vec &a, const Vec &b) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = fma2(a.v[i], b.v[i], v[i]);
    }
    // this·f + b
    __device__ __forceinline__ void scale_add(float f, const Vec &b) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = fma2(v[i], make_float2(f, f), b.v[i]);
    }
    // (this − f·b)·r
    __device__ __forceinline__ void take(float f, const Vec &b, float r) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) v[i] = mul2(fma2(b.v[i], make_float2(-f, -f), v[i]), make_float2(r, r));
    }
    __device__ __forceinline__ float dot(const Vec &b) const {
        float2 s = mul2(v[0], b.v[0]);
#pragma unroll
        for (int i = 1; i < kPairs; ++i) s = fma2(v[i], b.v[i], s);
        return s.x + s.y;
    }
};

// i / by for 0 <= i < 2^31 and by >= 1: with 2^(l-1) < by <= 2^l, the upper bits of i · ceil(2^(31+l) / by). (The product
// exceeds i · 2^(31+l) / by by less than 2^31 · by / by <= 2^(31+l) / by, what the next multiple is away.)
struct Divisor {
    uint32_t times;
    int shift;
    __device__ __forceinline__ int of(int i) const { return (int)((uint64_t)(uint32_t)i * times >> shift); }
};

inline Divisor divisor(int64_t by) {
    int l = 0;
    while (((int64_t)1 << l) < by) ++l;
    return {(uint32_t)((((uint64_t)1 << (31 + l)) + by - 1) / by), 31 + l};
}

// A tensor's rows: at one stride of `stride` bytes, or (stride < 0) at two.
struct Rows {
    const unsigned char *data;
    int64_t row, outer;  // bytes
    int stride, inner;
    Divisor by_inner;
};

template <typename T, bool kFlat = false>
__device__ __forceinline__ const T *row_at(const Rows &r, int i) {
    if (kFlat || r.stride >= 0) return reinterpret_cast<const T *>(r.data + (int64_t)i * r.stride);
    const int o = r.by_inner.of(i);
    return reinterpret_cast<const T *>(r.data + o * r.outer + (i - o * r.inner) * r.row);
}

// ---- teams

constexpr int kNormWarps = kNormThreads / 32;

// kSub: a team of less than a warp. Its thread t holds the packs t, t + size, ...; in larger ones a warp holds its threads' packs
// one behind the other, 32 at a time, so that a thread's packs lie at a distance known to the compiler.
template <bool kSub>
struct Team {
    int size, t, slot;  // threads of a team; this one's place; the team's place in the block
    int first;          // this thread's first pack
    int turn;           // which half of the scratch the next exchange uses
    float *scratch;     // kScratch floats, 16-byte aligned

    // Teams of more than a warp are at most half as many as the block's warps; each has kNormWarps floats for a sum.
    static constexpr int kSlots = kNormWarps / 2, kHalf = kSlots * kNormSums * kNormWarps, kScratch = 2 * kHalf;

    __device__ Team(int size_, int packs, float *scratch_)
        : size(size_), t(threadIdx.x % size_), slot(threadIdx.x / size_), first(kSub ? t : (t >> 5) * 32 * packs + (t & 31)),
          turn(0), scratch(scratch_) {
        if (!kSub && size > 32) {  // the places of the warps that there are not add zeros
            for (int i = threadIdx.x; i < kScratch; i += blockDim.x) scratch[i] = 0.f;
            __syncthreads();
        }
    }

    __device__ __forceinline__ int pack(int q) const { return first + q * (kSub ? size : 32); }

    // Of the warp: whether any team's `x` holds; of a larger team, where all agree, x.
    __device__ __forceinline__ static bool any(bool x) { return kSub ? __any_sync(0xffffffffu, x) : x; }

    __device__ __forceinline__ void barrier() const {
        if (kSub || size <= 32)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(slot + 1), "r"(size) : "memory");
    }

    // The sums over the team, in every thread of it and in a fixed order. All threads of the team call it (and all of the
    // warp, where teams are parts of one). Two halves of the scratch in turn: a team's thread comes to an exchange only
    // when the whole team has read the one before the last.
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
        static_assert(K <= kNormSums, "the scratch holds kNormSums sums a team");
        if constexpr (kSub) {
            for (int o = size >> 1; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
            return;
        }
        // Half of the lanes go on with one sum, half with another: 6 exchanges for two sums (7 for three) instead of 10 (15).
        const int lane = t & 31;
        float s = v[0];
        int mine = 0;
        if constexpr (K == 3) {
            const bool up = lane & 16;
            const float keep = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
            const float last = v[2] + __shfl_xor_sync(0xffffffffu, v[2], 16);
            const bool third = lane & 8;  // lanes 8 to 15 and 24 to 31 take the third sum
            s = (third ? last : keep) + __shfl_xor_sync(0xffffffffu, third ? keep : last, 8);
            mine = third ? 2 : up;
        } else if constexpr (K == 2) {
            const bool up = lane & 16;
            s = (up ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, up ? v[0] : v[1], 16);
            mine = up;
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1)
            if (x <= (K == 3 ? 4 : K == 2 ? 8 : 16)) s += __shfl_xor_sync(0xffffffffu, s, x);
        if (size == 32) {
            v[0] = __shfl_sync(0xffffffffu, s, 0);
            if constexpr (K >= 2) v[1] = __shfl_sync(0xffffffffu, s, 16);
            if constexpr (K == 3) v[2] = __shfl_sync(0xffffffffu, s, 8);
            return;
        }
        float *const half = scratch + turn * kHalf + slot * (kNormSums * kNormWarps);
        turn ^= 1;
        if (lane == 0 || (K >= 2 && lane == 16) || (K == 3 && lane == 8)) half[mine * kNormWarps + (t >> 5)] = s;
        barrier();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float4 *const f = reinterpret_cast<const float4 *>(half + k * kNormWarps);
            float2 a = four(f[0]);
            if (size > 128) a = add2(a, four(f[1]));
            if (size > 256) a = add2(a, add2(four(f[2]), four(f[3])));
            v[k] = a.x + a.y;
        }
    }
    __device__ __forceinline__ static float2 four(float4 f) { return add2(make_float2(f.x, f.y), make_float2(f.z, f.w)); }
};

// ---- rows on their way
//
// A team's next rows are fetched into shared memory while it works on one: `stages` of them, a stage holding every tensor that
// the call reads row by row. Vectors: the threads of a warp fetch one another's packs. Elements: the team fetches the
// 16-byte pieces that hold the row (whatever lies beside it in the first and the last of them comes along and is not used), and
// meets before it reads them.

enum { kTensorH, kTensorDy, kTensorDh, kTensorBranch, kTensorGate, kTensors };

struct RingParams {
    int stages, stage_bytes, ring_bytes;  // of a block: of one stage, of all
    int at[kTensors], image[kTensors];  // where a tensor's part of a stage begins; elements: bytes of a team's row
};

__device__ __forceinline__ uint4 shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}

template <typename T>
__device__ __forceinline__ float shared_one(uint32_t at) {
    if constexpr (sizeof(T) == 4) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
        return v;
    } else {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at));
        return __uint_as_float((uint32_t)v << 16);
    }
}

// Places in it are the bytes of the shared window at which a stage begins. Vectors: a warp's pieces lie together, 512 bytes for
// each pack (fp32: two) of its threads.
template <int V, int P, bool kSub>
struct Ring {
    uint32_t base;
    const RingParams &p;
    const Team<kSub> &team;
    int packs;

    __device__ Ring(const void *shared, const RingParams &p_, const Team<kSub> &team_, int packs_)
        : base((uint32_t)__cvta_generic_to_shared(shared)), p(p_), team(team_), packs(packs_) {}

    __device__ __forceinline__ uint32_t first() const { return base; }
    __device__ __forceinline__ uint32_t after(uint32_t stage) const {
        const uint32_t next = stage + p.stage_bytes;
        return next == base + p.ring_bytes ? base : next;
    }

    // 16 bytes, or (bytes = 0) as many zeros
    __device__ __forceinline__ static void copy16(uint32_t to, const void *from, int bytes) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    }
    __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

    // The oldest row on its way has arrived, for all threads that read it. Vectors: called when the row that fills the stages is
    // on its way, too; elements: before, since this is also where the team is through with the stage that it goes to.
    __device__ __forceinline__ void wait() const {
        switch (p.stages - (V == 1 ? 1 : 0)) {
            case 1: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
            case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
            case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
            default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        }
        if (V == 1)
            team.barrier();
        else
            __syncwarp();
    }

    __device__ __forceinline__ uint32_t part(uint32_t stage, int tensor) const {
        return stage + p.at[tensor] + (V == 1 ? team.slot * p.image[tensor] : 0);
    }
    // of a thread's first piece among the vectors
    template <typename T>
    __device__ __forceinline__ static uint32_t own() {
        return (threadIdx.x >> 5) * (P * (int)sizeof(T) / 2 * 512) + (threadIdx.x & 31) * 16;
    }

    // Starts the copies of a tensor's row (bytes = 0: of a row of zeros). Of fp32 packs, a pair of 16-byte pieces each, the threads
    // of a warp (a smaller team) fetch neighbouring pieces, so that no sector is asked for twice.
    template <typename T>
    __device__ __forceinline__ void fetch(uint32_t stage, int tensor, const T *row, int bytes) const {
        uint32_t to = part(stage, tensor);
        if constexpr (V == 8 && sizeof(T) == 2) {
            to += own<T>();
#pragma unroll
            for (int q = 0; q < P; ++q) {
                int pack = team.pack(q), some = bytes;
                if (pack >= packs) pack = 0, some = 0;  // zeros behind the row's end
                copy16(to + q * 512, row + pack * 8, some);
            }
        } else if constexpr (V == 8) {
            const int width = kSub ? team.size : 32, lane = kSub ? team.t : threadIdx.x & 31;
            to += own<T>() - lane * 16;  // of the team's (the warp's) first thread
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int piece = lane + i * width;
                    int pack = team.pack(q) - lane + (piece >> 1), some = bytes;
                    if (pack >= packs) pack = 0, some = 0;
                    copy16(to + (2 * q + (piece & 1)) * 512 + (piece >> 1) * 16, row + pack * 8 + (piece & 1) * 4, some);
                }
        } else {
            const int shift = (int)(reinterpret_cast<uintptr_t>(row) & 15);
            const unsigned char *const from = reinterpret_cast<const unsigned char *>(row) - shift;
            const int pieces = (shift + packs * (int)sizeof(T) + 15) >> 4;
            for (int i = team.t; i < pieces; i += team.size) copy16(to + i * 16, from + i * 16, bytes);
        }
    }

    // This thread's elements of the row in a stage, zeros behind the row's end.
    template <typename T>
    __device__ __forceinline__ void read(uint32_t stage, int tensor, const T *row, Vec<P * V> &x) const {
        uint32_t from = part(stage, tensor);
        if constexpr (V == 8) {
            constexpr int kPieces = sizeof(T) / 2;
            from += own<T>();
#pragma unroll
            for (int q = 0; q < P; ++q) {
                uint4 v[kPieces];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) v[i] = shared16(from + (q * kPieces + i) * 512);
                float f[8];
                Raw<T, 8>::unpack(v, f);
                x.set(q * 8, f);
            }
        } else {
            from += (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15) + team.first * (uint32_t)sizeof(T);
            const int there = packs - team.first, step = kSub ? team.size : 32;
#pragma unroll
            for (int q = 0; q < P; ++q) {
                float f[1] = {shared_one<T>(from + q * step * (int)sizeof(T))};  // the image has room for all places
                if (q * step >= there) f[0] = 0.f;
                x.set(q, f);
            }
        }
    }

    __device__ __forceinline__ void fetch_typed(uint32_t stage, int tensor, const void *row, int dtype, int bytes) const {
        if (dtype == LAMQ_F32)
            fetch(stage, tensor, reinterpret_cast<const float *>(row), bytes);
        else
            fetch(stage, tensor, reinterpret_cast<const __nv_bfloat16 *>(row), bytes);
    }
    __device__ __forceinline__ void read_typed(uint32_t stage, int tensor, const void *row, int dtype, Vec<P * V> &x) const {
        if (dtype == LAMQ_F32)
            read(stage, tensor, reinterpret_cast<const float *>(row), x);
        else
            read(stage, tensor, reinterpret_cast<const __nv_bfloat16 *>(row), x);
    }
};

// v^-1/2 for a normal v: the hardware's approximation (2 units in the last place) and a Newton step. An infinite v gives 0.
__device__ __forceinline__ float reciprocal_root(float v) {
    const float r = rsqrtf(v);
    const float e = fmaf(-v * r, r, 1.f);
    return isinf(v) ? 0.f : fmaf(0.5f * r, e, r);
}

constexpr float kShrink = 0x1p-80f;  // brings fp32's largest numbers where 16384 of their squares have a sum

// The factor (mean(x²) + eps)^-1/2 of a row, from the sum of squares, for x as it stands after the call: where the sum
// overflowed, x is multiplied by kShrink and summed again (eps is then far below the mean's last bit). `shrunk` is
// kShrink or 1: the factor of x as it was is the result times `shrunk`.
template <bool kSub, int E>
__device__ __forceinline__ float unit_factor(Team<kSub> &team, Vec<E> &x, float ss, float inv_d, float eps, float &shrunk) {
    shrunk = 1.f;
    const bool over = isinf(ss);
    if (team.any(over)) {
        if (over) shrunk = kShrink;
        x *= shrunk;
        float again[1] = {x.dot(x)};
        team.sum(again);
        ss = again[0];
        if (over) eps = 0.f;
    }
    return reciprocal_root(fmaf(ss, inv_d, eps));
}

// Whether of a row's Σ h² and Σ t·h, taken of the row as it is, one may have lost something to fp32's range: past its end; or, of
// rows so small that the factor passes 2^20, products of 2^-126 and less, which are rounded to multiples of 2^-149. (Of others
// that is 2^-103 in the result at most: the mean of roundings of 2^-150, times the factor twice and ĥ <= 128.) Σ t·h is then taken
// of the normed row: an exchange more, so not for all.
__device__ __forceinline__ bool sums_lost(float hh, float th, float eps) {
    return isinf(hh) || !(fabsf(th) <= 0x1p126f) || (eps < 0x1p-40f && hh < 0x1p-26f && fabsf(th) < 0x1p-60f);
}

// ---- the host's side

// Which tensors a call has, and in the place of the others an output's memory of the same shape and no smaller a type: what
// a kernel gets may be read whether or not it is there.
enum { kHasWeight = 1, kHasPost = 2, kHasGate = 4, kHasDh = 8, kHasDy = 16 };

struct Present {
    int has;
    Rows h, branch, dh, dy;  // h: the norm's input, or what the branch is added to
    const void *weight, *post, *gate;
    int weight_dtype, post_dtype, gate_dtype, gate_span;
    Divisor by_span;
};

inline int element_size(int dtype) { return dtype == LAMQ_F32 ? 4 : 2; }

inline bool one_stride(const lamq_rows &r, int64_t rows) {
    return r.row >= 0 && (r.inner >= rows || r.outer == r.inner * r.row);
}

inline Rows rows_of(const lamq_rows &r, int64_t rows, int size) {
    Rows x;
    x.data = reinterpret_cast<const unsigned char *>(r.data);
    x.row = r.row * size, x.outer = r.outer * size, x.inner = (int)r.inner, x.by_inner = divisor(r.inner);
    x.stride = one_stride(r, rows) && x.row <= INT_MAX ? (int)x.row : -1;
    return x;
}

inline Present present(const lamq_norm_args &a, bool backward) {
    const void *const out = backward ? a.d_residual : a.branch.data ? a.h : a.y;
    const lamq_rows rows{const_cast<void *>(out), INT_MAX, a.d, 0};
    const int r = element_size(a.residual_dtype), b = element_size(a.branch_dtype);
    Present p;
    p.has = (a.weight ? kHasWeight : 0) | (a.post ? kHasPost : 0) | (a.gate ? kHasGate : 0) |
            (backward && a.dh.data ? kHasDh : 0) | (backward && a.dy.data ? kHasDy : 0);
    p.h = rows_of(a.residual, a.rows, r);
    p.branch = rows_of(a.branch.data ? a.branch : rows, a.rows, b);
    p.dh = rows_of(p.has & kHasDh ? a.dh : rows, a.rows, r);
    p.dy = rows_of(p.has & kHasDy ? a.dy : rows, a.rows, b);
    p.weight = a.weight ? a.weight : out, p.weight_dtype = a.weight ? a.weight_dtype : a.residual_dtype;
    p.post = a.post ? a.post : out, p.post_dtype = a.post ? a.post_dtype : a.residual_dtype;
    p.gate = a.gate ? a.gate : out, p.gate_dtype = a.gate ? a.gate_dtype : a.residual_dtype;
    p.gate_span = a.gate ? (int)a.gate_span : 1, p.by_span = divisor(p.gate_span);
    return p;
}

inline bool aligned_rows(const lamq_rows &r) {
    return !r.data || ((reinterpret_cast<uintptr_t>(r.data) & 15) == 0 && r.row % 8 == 0 && r.outer % 8 == 0);
}

// How many threads share a row, and P: the packs of V elements that each holds of it.
struct NormShape {
    int V, P, team, packs;
    NormKernel kernel;
};

// Vectors where every row begins on 16 bytes and every array on 32, elements elsewhere. A thread holds 16 elements of a row:
// what it does for a row beside the arithmetic (places, waits, exchanges) costs as much as the arithmetic of 16 (16384 x 2560,
// the norm's backward, us: 78 with 8, 61 with 16; the forward of a join with both norms takes the same with either). The full
// join's backward holds three sums and three tensors of a row: 8 of each (8192 x 4096: 152 with 8 and 16 warps an SM, 189 with
// 16 and 8 warps). Up to 32 threads a team is a power of two of lanes, else whole
// warps. Wider rows take teams of up to 512 threads with 16 elements, then with 32; rows wider than 4096 that may begin
// anywhere, a block each.
inline NormShape norm_shape(const lamq_norm_args &a, bool backward) {
    const void *arrays[] = {a.weight, a.post, a.gate, a.h, a.y, a.d_residual, a.d_branch, a.d_weight, a.d_post, a.d_gate};
    bool vec = a.d % 8 == 0 && aligned_rows(a.residual) && aligned_rows(a.branch);
    if (backward) vec = vec && aligned_rows(a.dh) && aligned_rows(a.dy);
    for (const void *p : arrays) vec = vec && (reinterpret_cast<uintptr_t>(p) & 31) == 0;  // 32 bytes are stored at once
    const bool full = backward && (a.post || a.gate);
    int e = full ? 8 : 16;
    NormShape s;
    s.kernel = full ? (vec ? kVectors8 : kElements8) : vec ? kVectors : kElements;
    if (a.d > 4096) {
        s.kernel = !vec ? kWide : a.d <= 8192 ? kVectorsWide : full ? kWide : kVectorsWidest;
        e = s.kernel == kVectorsWidest ? 32 : 16;
    }
    s.V = vec && s.kernel != kWide ? 8 : 1;
    s.P = e / s.V;
    s.packs = a.d / s.V;
    const int threads = (a.d + e - 1) / e;
    s.team = s.kernel == kWide ? kNormThreads : (threads + 31) / 32 * 32;
    if (threads <= 32)
        for (s.team = 1; s.team < threads;) s.team *= 2;
    return s;
}

inline bool holds(NormKernel kernel) { return kernel <= kElements8; }

// Teams of a block: blocks of about 256 threads, fewer where there are few rows, whole warps always. Threads of larger teams
// keep their sums in shared memory, where a block's teams are not added up: one team a block.
inline int norm_slots(const NormShape &s, int64_t rows) {
    if (!holds(s.kernel)) return 1;
    const int least = std::max(1, 32 / s.team), most = std::max(least, 256 / s.team);
    const int64_t wanted = (rows + 2 * kSMs - 1) / (2 * kSMs);
    return (int)std::min<int64_t>(most, std::max<int64_t>(least, (wanted + least - 1) / least * least));
}

// Lets a kernel have `dynamic` bytes of shared memory beside its own. LAMQ_OK, or an error that is set.
inline int allow_shared(const void *kernel, int dynamic) {
    if (dynamic + 24 * 1024 <= 48 * 1024) return LAMQ_OK;  // beside the kernels' static arrays, 20 KB at most
    const cudaError_t e = smem_limit_max_once(kernel);
    if (e == cudaSuccess) return LAMQ_OK;
    set_error("shared memory: %s", cudaGetErrorString(e));
    return LAMQ_ERR_CUDA;
}

// What a call runs: its shape, its blocks and their shared memory.
struct NormLayout {
    NormShape shape;
    int mode, slots, blocks;  // blocks: of an SM
    RingParams ring;
    int sums_bytes, shared;   // of the dynamic shared memory: the sums that registers do not hold, and all of it
};

constexpr int kSmemSM = 220 * 1024;  // of 228 KB; each block takes 1 KB for itself

// `gate_sums`: the gradient of the gate is wanted; `sums`: that of any parameter. Blocks are as many as their registers allow, or
// as have room for two stages each; stages fill the room, four at most (a block alone on its SM may have one). What finds no
// room (rows that begin anywhere: for two stages) is left to the wide kernels: the full join's backward of fp32 rows from 7688
// elements on with parameters' gradients (from 6664 with a gate in fp32 for each element), the plain join's from 13320 (of an
// fp32 stream with bf16 branches, 15368). More blocks with fewer registers are slower: the norm's backward of 16384 x 2560 at 96
// registers, 4 blocks of 160 threads, 93 us against 55 at 122, 3 blocks (what spills, and one stage less).
inline NormLayout norm_layout(const lamq_norm_args &a, bool backward, bool sums, bool gate_sums) {
    NormLayout l{};
    const bool join = a.branch.data, gates = a.gate && a.gate_span == 1;
    l.mode = !join ? kNormAlone : a.post || a.gate ? kJoinFull : kJoinPlain;
    l.shape = norm_shape(a, backward);
    NormShape &s = l.shape;
    const int r = element_size(a.residual_dtype), b = element_size(a.branch_dtype);
    int size[kTensors] = {r, 0, 0, join ? b : 0, gates ? element_size(a.gate_dtype) : 0};
    if (backward) {
        size[kTensorH] = a.dy.data ? r : 0, size[kTensorDy] = a.dy.data ? b : 0, size[kTensorDh] = a.dh.data ? r : 0;
        size[kTensorBranch] = a.post || gate_sums ? b : 0;
    }
    if (s.kernel != kWide) {
        const bool hold = holds(s.kernel);
        l.slots = norm_slots(s, a.rows);
        const int threads = s.team * l.slots;
        RingParams &g = l.ring;
        for (int k = 0; k < kTensors; ++k) {
            g.at[k] = g.stage_bytes;
            g.image[k] = (s.team * s.P * size[k] + 15) / 16 * 16 + 16;  // of elements: a place for each, wherever the row begins
            g.stage_bytes += size[k] == 0 ? 0 : s.V == 8 ? s.P * 8 * size[k] * threads : g.image[k] * l.slots;
        }
        l.sums_bytes = sums && !hold ? (l.mode == kJoinFull ? 3 : 1) * s.P * s.V * threads * (int)sizeof(float) : 0;
        const int own = Team<false>::kScratch * (int)sizeof(float) + 1024 + l.sums_bytes +
                        (backward && sums && hold ? 4096 * (int)sizeof(float) : 0);
        l.blocks = std::max(1, resident(s.kernel, l.mode, backward) / threads);
        for (;; --l.blocks) {
            g.stages = std::min(4, (kSmemSM / l.blocks - own) / std::max(1, g.stage_bytes));
            if (g.stages >= 2 || l.blocks == 1) break;
        }
        g.ring_bytes = g.stages * g.stage_bytes;
        l.shared = g.ring_bytes + l.sums_bytes;
        if (g.stages >= (s.V == 1 ? 2 : 1)) return l;
    }
    s.V = 1, s.kernel = kWide, s.team = kNormThreads, s.packs = a.d;
    l.slots = 1, l.blocks = 2, l.shared = a.d * (int)sizeof(float);
    return l;
}

}  // namespace
}  // namespace lamq
