// gradnorm.hip -- the global norm of many gradient tensors, and clipping by it.
//
//     norm   = (sum over all tensors k and elements i of |s_k g_ki|^p)^(1/p),  p = 1, 2;  their largest magnitude for p = infinity
//     factor = min(1, max_norm / (norm + 1e-6))
//     g      = g * factor          (clip; nothing is written when the factor is one)
//
// The gradients of a Monte-Carlo estimate carry outliers (one firefly in one view); clipping bounds the step they can cause.  Bytes bound
// all of it: the norm reads every gradient once, the scaling reads and writes it.
//
// Sums in fp64.  An fp32 gradient's square leaves the range of fp32 from 1.8e19 up and 1e-19 down, and a sum of 1e9 terms loses half of
// fp32's digits; a conversion and an fma in fp64 per element are far below what the memory can deliver in elements.  No atomics: every
// workgroup writes its sum to a place of its own and they are added in a fixed order.  The order follows from the sizes, the alignment, which
// tensors are neighbours in memory (they are cut as one) and whether one workgroup clips the list: the same call on the same places gives
// the same bits, and other places change a norm by the rounding of its fp64 sum, which is seen in fp32 once in some 1e8 times.
//
// Work split.  The tensors are cut into chunks of NVDR_GN_CHUNK bytes, and runs of chunks, whatever tensors they fall into, are dealt to the
// workgroups in turn, as many rounds of equally long runs as NVDR_GN_RUN gives: a long tensor is shared by many workgroups, many short ones
// by few, and no workgroup has more than one run more than another.  The table of the tensors travels in the kernel arguments -- by value, so
// that a captured graph keeps it and no copy to the device is needed -- which bounds the tensors of a launch; longer lists take several
// launches.  Neighbours in memory (views of one bucket) become one entry.
//
// What was measured (us a call on MI355X; 789 M fp32 = 3.16 GB | 296 M bf16 = 0.59 GB in 315 tensors | 10.7 M fp32 = 43 MB in the cache):
//   norm   one contiguous run per workgroup, plain loads          515 | 104 | 12.4
//          the same with non-temporal loads                       458 |  92 | 12.5
//          runs of 128 KB dealt in turn, non-temporal             449 |  96 | 12.4      (7.0 TB/s; 32 KB runs: 468 | 132 | 13.2)
//          finished by its own first workgroup, not by a kernel   447 |  95 | 10.8      (wavefronts joined by DPP: 10.4)
//   clip   one contiguous run per workgroup, plain               1783 | 357 | 23.4
//          the last 160 MB of the norm's pass loaded to stay,
//          the scaling from the end to the front, non-temporal   1675 | 307 | 23.4
//          runs of 128 KB dealt in turn                          1581 | 300 | 23.3
//          scaling by 256 workgroups of 1024, eight loads deep   1472 | 293 | 24.7      (6.2 TB/s of reading and writing)
// The time of a short list is that of its launches: 0.8 MB take 5.4 us on the device and 6.6 a call, clipped 4.1 + 4.2 and 10.0; one workgroup
// clips 64 KB in one launch, 6.8 us where the two launches took 8.6 (at 128 KB 8.5 against 8.7, and 8.1 against 6.7 in a captured graph).
// A list that fits the last-level cache is left there: plain loads and stores (non-temporal ones cost 29 instead of 23 us at 43 MB), for the
// scaling and for whoever reads the gradients next.
#include <stdlib.h>
#include <algorithm>
#include <atomic>
#include <chrono>

#include "common.h"
#include "gradnorm.h"
#include "nvdr_hip.h"

#define NVDR_GN_BLOCK 512               // threads of a workgroup of the norm, and of the scaling of a list that fits the cache
#define NVDR_GN_GRID 512                // workgroups of a launch at most: two per CU
#define NVDR_GN_STREAM_BLOCK 1024       // the scaling of a longer list: fewer places in memory at a time
#define NVDR_GN_STREAM_GRID 256
#define NVDR_GN_TENSORS 160             // of a launch: the kernel arguments end at 4 KB
#define NVDR_GN_CHUNK 4096              // bytes
#define NVDR_GN_RUN (128 << 10)         // bytes
#define NVDR_GN_KEEP (160ll << 20)      // bytes that stay in the last-level cache (256 MB) from one pass to the next: 96 to 256 MB within 2 %
#define NVDR_GN_ONE_BLOCK 1024          // a short list: one workgroup clips all of it
#define NVDR_GN_ONE_TENSORS 8
#define NVDR_GN_ONE_CLIP (64 << 10)     // bytes
#define NVDR_GN_PATIENCE (1 << 28)      // polls after which a workgroup no longer waits for another (minutes; the norm is then a NaN)
#define NVDR_GN_EPS 1e-6

enum { GN_INF = 0, GN_ONE = 1, GN_TWO = 2 };                // the kernels' norm types
enum { GN_F32 = NVDR_GRAD_F32, GN_BF16 = NVDR_GRAD_BF16, GN_F16 = NVDR_GRAD_F16 };

// (what a workgroup asks for first lies in front, within one load)
struct GradTable {
    int n_tensors;
    uint32_t chunks;
    uint32_t run;                               // chunks that a workgroup takes at a time
    uint32_t kept;                              // chunks from here on are loaded to stay in the last-level cache
    uint32_t first[NVDR_GN_TENSORS + 8];        // chunks in front of the tensor; from n_tensors on: all of them
    float scale[NVDR_GN_TENSORS];
    uint64_t data[NVDR_GN_TENSORS];             // address, the type in the upper two bits
    int64_t n[NVDR_GN_TENSORS];                 // elements, never zero
};
static_assert(NVDR_GN_CHUNK == 4 << 10, "gn_fill divides by shifting");
static_assert(sizeof(GradTable) <= 3900, "the kernel arguments have to fit 4 KB");

typedef uint32_t gn_u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float gn_bf16(uint32_t bits) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float gn_f16(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }

// ---- one thread's sum ------------------------------------------------------------------------------------------------------------
// p = infinity compares bit patterns: without the sign they order like the values, a NaN above infinity, so that a NaN survives.
template <int P>
struct GradSum {
    double s = 0.0;
    uint32_t m = 0;
    __device__ __forceinline__ void add(float x)
    {
        if (P == GN_TWO) { const double d = (double)x; s = fma(d, d, s); }
        else if (P == GN_ONE) s += fabs((double)x);
        else m = max(m, __float_as_uint(x) & 0x7fffffffu);
    }
    template <int T>
    __device__ __forceinline__ void add16(gn_u4 v)
    {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if (T == GN_F32) add(__uint_as_float(v[c]));
            else if (T == GN_BF16) { add(gn_bf16(v[c] & 0xffffu)); add(__uint_as_float(v[c] & 0xffff0000u)); }
            else { add(gn_f16(v[c] & 0xffffu)); add(gn_f16(v[c] >> 16)); }
        }
    }
    __device__ __forceinline__ double value() const { return P == GN_INF ? (double)__uint_as_float(m) : s; }
};

template <int P>
__device__ __forceinline__ double gn_join(double a, double b)
{
    if (P == GN_INF) return (a > b || a != a) ? a : b;
    return a + b;
}

// v joined with the value of the lane that the DPP control names (lanes it names none for: with zero, which changes no sum and no maximum)
template <int P, int CTRL, int ROWS>
__device__ __forceinline__ double gn_dpp(double v)
{
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, ROWS, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, ROWS, 0xf, false);
    return gn_join<P>(v, __longlong_as_double((long long)((unsigned long long)hi << 32 | lo)));
}

// the sum over the workgroup, in every thread; `lds`: one double per wavefront.  Within a wavefront by DPP (rows of sixteen lanes, then row to
// row into the last lane): 0.4 us less a kernel than six exchanges through the LDS hardware.
template <int P>
__device__ __forceinline__ double gn_block_join(double v, double *lds)
{
    v = gn_dpp<P, 0x111, 0xf>(v);          // row_shr:1
    v = gn_dpp<P, 0x112, 0xf>(v);          // row_shr:2
    v = gn_dpp<P, 0x114, 0xf>(v);          // row_shr:4
    v = gn_dpp<P, 0x118, 0xf>(v);          // row_shr:8
    v = gn_dpp<P, 0x142, 0xa>(v);          // row_bcast:15 into rows 1 and 3
    v = gn_dpp<P, 0x143, 0xc>(v);          // row_bcast:31 into rows 2 and 3
    __syncthreads();                                        // (a second call: the first one's values have been read)
    if ((threadIdx.x & 63) == 63) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = gn_join<P>(v, lds[w]);
    return v;
}

// ---- which part of which tensor ----------------------------------------------------------------------------------------------------
// the tensor that chunk c falls into: of a few all entries are compared, of more 64 at a time by the lanes (one round trip each; a search would
// take seven)
__device__ __forceinline__ int gn_find(const GradTable &tab, uint32_t c)
{
    if (tab.n_tensors <= 8) {
        int at = 0;
#pragma unroll
        for (int q = 1; q < 8; ++q) at += tab.first[q] <= c ? 1 : 0;
        return at;
    }
    const int lane = threadIdx.x & 63;
    int at = -1;
    for (int q = 0; q < tab.n_tensors; q += 64)
        at += __popcll(__ballot(q + lane < tab.n_tensors && tab.first[min(q + lane, NVDR_GN_TENSORS)] <= c));
    return __builtin_amdgcn_readfirstlane(at);
}

// elements per chunk
__device__ __forceinline__ int gn_chunk_len(int type) { return type == GN_F32 ? NVDR_GN_CHUNK / 4 : NVDR_GN_CHUNK / 2; }

template <bool NT>
__device__ __forceinline__ gn_u4 gn_load(const gn_u4 *p) { return NT ? __builtin_nontemporal_load(p) : *p; }

template <int P, int T, bool NT, int BLOCK>
__device__ __forceinline__ double gn_sum_part(const char *p, int64_t count)
{
    constexpr int SIZE = T == GN_F32 ? 4 : 2, VEC = 16 / SIZE;
    auto one = [&](int64_t i) -> float {
        if (T == GN_F32) return ((const float *)p)[i];
        const uint32_t h = ((const uint16_t *)p)[i];
        return T == GN_BF16 ? gn_bf16(h) : gn_f16(h);
    };
    GradSum<P> a[4];
    const int64_t head = min((int64_t)((16 - ((uintptr_t)p & 15)) & 15) / SIZE, count);     // up to the first 16-byte boundary
    const int64_t nvec = (count - head) / VEC, tail = count - head - nvec * VEC;
    if ((int64_t)threadIdx.x < head) a[0].add(one(threadIdx.x));
    if ((int64_t)threadIdx.x < tail) a[1].add(one(head + nvec * VEC + threadIdx.x));
    const gn_u4 *v = (const gn_u4 *)(p + head * SIZE);
    int64_t i = threadIdx.x;
    for (; i + 3 * BLOCK < nvec; i += 4 * BLOCK) {      // four loads in flight
        gn_u4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = gn_load<NT>(v + i + u * BLOCK);
#pragma unroll
        for (int u = 0; u < 4; ++u) a[u].template add16<T>(x[u]);
    }
    gn_u4 x[3];
#pragma unroll
    for (int u = 0; u < 3; ++u) x[u] = i + u * BLOCK < nvec ? gn_load<NT>(v + i + u * BLOCK) : gn_u4{0, 0, 0, 0};     // (a zero adds nothing)
#pragma unroll
    for (int u = 0; u < 3; ++u) a[u].template add16<T>(x[u]);
    return gn_join<P>(gn_join<P>(a[0].value(), a[1].value()), gn_join<P>(a[2].value(), a[3].value()));
}

template <int P, bool NT, int BLOCK>
__device__ __forceinline__ double gn_sum_typed(const char *p, int type, int64_t e0, int64_t e1)
{
    if (type == GN_F32) return gn_sum_part<P, GN_F32, NT, BLOCK>(p + e0 * 4, e1 - e0);
    if (type == GN_BF16) return gn_sum_part<P, GN_BF16, NT, BLOCK>(p + e0 * 2, e1 - e0);
    return gn_sum_part<P, GN_F16, NT, BLOCK>(p + e0 * 2, e1 - e0);
}

// one thread's sum over the runs of its workgroup
template <int P, int BLOCK>
__device__ __forceinline__ double gn_sum_runs(const GradTable &tab)
{
    const uint32_t chunks = tab.chunks, run = tab.run, kept = tab.kept;
    double sum = 0.0;
    for (uint64_t r = (uint64_t)blockIdx.x * run; r < chunks; r += (uint64_t)gridDim.x * run) {
        uint32_t c = (uint32_t)r;
        const uint32_t c1 = min(c + run, chunks);
        int k = gn_find(tab, c);
        while (c < c1) {
            const bool stream = c < kept;
            const uint32_t first = tab.first[k], next = tab.first[k + 1], end = min(stream ? min(kept, c1) : c1, next);
            const int type = (int)(tab.data[k] >> 62), len = gn_chunk_len(type);
            const char *p = (const char *)(tab.data[k] & ~(3ull << 62));
            const int64_t e0 = (int64_t)(c - first) * len, e1 = min((int64_t)(end - first) * len, tab.n[k]);
            const double s = stream ? gn_sum_typed<P, true, BLOCK>(p, type, e0, e1) : gn_sum_typed<P, false, BLOCK>(p, type, e0, e1);
            const double w = fabs((double)tab.scale[k]);
            sum = gn_join<P>(sum, P == GN_TWO ? s * (w * w) : s * w);
            c = end;
            k += end == next;
        }
    }
    return sum;
}

// ---- the norm of the parts, and the factor -----------------------------------------------------------------------------------------
template <int P>
__device__ __forceinline__ double gn_root(double v) { return P == GN_TWO ? sqrt(v) : v; }

template <int P>
__device__ __forceinline__ double gn_total(const double *__restrict__ part, int n_part, double *lds)
{
    double v = 0.0;
    for (int i = threadIdx.x; i < n_part; i += blockDim.x) v = gn_join<P>(v, part[i]);
    return gn_root<P>(gn_block_join<P>(v, lds));
}

// one rounding to fp32, of the quotient in fp64; a NaN stays a NaN.  An infinite max_norm never scales (inf / inf would)
__device__ __forceinline__ float gn_factor(double norm, double max_norm)
{
    if (max_norm == (double)__builtin_inff()) return 1.0f;
    const double f = max_norm / (norm + NVDR_GN_EPS);
    return (float)(f > 1.0 ? 1.0 : f);
}

struct GradOut {
    double max_norm;
    float *norm, *factor;       // factor: NULL for none
    AdamBegin adam;             // adam.state: NULL for none
};

// What one thread writes when the norm is known.  In front of an Adam step also what that needs of its counter, which moves here: the
// update reads no state, and no launch behind it is needed to move it.  (`step`: adam_begin, computed where it costs no time.)
__device__ __forceinline__ void gn_finish(double norm, const GradOut &o, AdamStep step)
{
    step.factor = gn_factor(norm, o.max_norm);
    *o.norm = (float)norm;
    if (o.factor) *o.factor = step.factor;
    if (o.adam.state) {
        *o.adam.step = step;
        adam_advance(o.adam.state, o.adam.beta1, o.adam.beta2);
    }
}

// The parts of one table.  FINISH, in the last launch of a norm: its first workgroup waits for the others and writes the norm, `before` parts
// of earlier launches included, so that no kernel has to follow for it (a launch costs 4 us, the wait about 1).
//
// The wait.  Every other workgroup stores its part as two words, its bits under one key each, and the first one polls both until they open to the
// same bits.  Nobody waits for the first workgroup, so the others end whatever it does, and its wait ends with them.  Stores and loads go
// past the caches of the XCDs; nothing else is published, so no cache has to be written back or emptied for it (with a release and a tag
// behind the part, every workgroup wrote back what kernels before it had left in its L2: 25 instead of 17 us in front of an Adam step).
// The memory needs no clearing: a pair of keys belongs to one call only -- the host makes them from a counter, scrambled -- so that what
// another call or another tensor has left there does not open, and the first workgroup erases the words it has read, so that a captured
// launch finds none of its own when it is replayed.
struct GradKeys {
    unsigned long long a, b;
};

template <int P, bool FINISH>
__global__ void __launch_bounds__(NVDR_GN_BLOCK) grad_norm_kernel(GradTable tab, double *part, unsigned long long *words, GradKeys keys, int before, GradOut out)
{
    __shared__ double lds[NVDR_GN_BLOCK / 64];
    const double sum = gn_block_join<P>(gn_sum_runs<P, NVDR_GN_BLOCK>(tab), lds);
    if (!FINISH) {
        if (threadIdx.x == 0) part[before + blockIdx.x] = sum;
        return;
    }
    if (blockIdx.x != 0) {
        if (threadIdx.x == 0) {
            const unsigned long long bits = (unsigned long long)__double_as_longlong(sum);
            __hip_atomic_store(words + 2 * blockIdx.x, bits ^ keys.a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(words + 2 * blockIdx.x + 1, bits ^ keys.b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        return;
    }
    AdamStep step = {};
    if (out.adam.state && threadIdx.x == 0) step = adam_begin(out.adam.state, out.adam.lr, out.adam.beta1, out.adam.beta2);
    double v = 0.0;
    for (int i = threadIdx.x; i < before + (int)gridDim.x; i += NVDR_GN_BLOCK) {
        double x = sum;
        if (i < before) x = part[i];
        else if (i > before) {
            unsigned long long *w = words + 2 * (i - before), p, q;
            int left = NVDR_GN_PATIENCE;
            for (;;) {
                p = __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ^ keys.a;
                q = __hip_atomic_load(w + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ^ keys.b;
                if (p == q || --left == 0) break;
                __builtin_amdgcn_s_sleep(1);
            }
            x = p == q ? __longlong_as_double((long long)p) : (double)__builtin_nanf("");
            __hip_atomic_store(w, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(w + 1, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        v = gn_join<P>(v, x);
    }
    v = gn_root<P>(gn_block_join<P>(v, lds));
    if (threadIdx.x == 0) gn_finish(v, out, step);
}

// ---- scaling -------------------------------------------------------------------------------------------------------------------------
template <int T>
__device__ __forceinline__ uint32_t gn_scaled(uint32_t w, float f)
{
    if (T == GN_F32) return __float_as_uint(__uint_as_float(w) * f);
    if (T == GN_BF16) {
        const uint32_t lo = __builtin_bit_cast(unsigned short, (__bf16)(gn_bf16(w & 0xffffu) * f));
        return lo | ((uint32_t)__builtin_bit_cast(unsigned short, (__bf16)(__uint_as_float(w & 0xffff0000u) * f)) << 16);
    }
    const uint32_t lo = __builtin_bit_cast(unsigned short, (_Float16)(gn_f16(w & 0xffffu) * f));
    return lo | ((uint32_t)__builtin_bit_cast(unsigned short, (_Float16)(gn_f16(w >> 16) * f)) << 16);
}

// from the end to the front: the norm's pass went the other way, and what it read last is still in the last-level cache
template <int T, bool NT, int BLOCK>
__device__ __forceinline__ void gn_scale_part(char *p, int64_t count, float f)
{
    constexpr int SIZE = T == GN_F32 ? 4 : 2, VEC = 16 / SIZE, DEEP = NT ? 8 : 4;
    auto one = [&](int64_t i) {
        if (T == GN_F32) ((float *)p)[i] *= f;
        else ((uint16_t *)p)[i] = (uint16_t)gn_scaled<T>(((uint16_t *)p)[i], f);
    };
    const int64_t head = min((int64_t)((16 - ((uintptr_t)p & 15)) & 15) / SIZE, count);
    const int64_t nvec = (count - head) / VEC, tail = count - head - nvec * VEC;
    gn_u4 *v = (gn_u4 *)(p + head * SIZE);
    for (int64_t b = (nvec + DEEP * BLOCK - 1) / (DEEP * BLOCK) - 1; b >= 0; --b) {
        const int64_t i = b * (DEEP * BLOCK) + threadIdx.x;
        gn_u4 x[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u)
            if (i + u * BLOCK < nvec) x[u] = gn_load<NT>(v + i + u * BLOCK);
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            if (i + u * BLOCK >= nvec) break;
            gn_u4 y;
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = gn_scaled<T>(x[u][c], f);
            if (NT) __builtin_nontemporal_store(y, v + i + u * BLOCK);
            else v[i + u * BLOCK] = y;
        }
    }
    if ((int64_t)threadIdx.x < head) one(threadIdx.x);
    if ((int64_t)threadIdx.x < tail) one(head + nvec * VEC + threadIdx.x);
}

template <bool NT, int BLOCK>
__device__ __forceinline__ void gn_scale_runs(const GradTable &tab, float f)
{
    const uint32_t chunks = tab.chunks, run = tab.run, runs = (chunks - 1) / run + 1;
    for (int64_t r = (int64_t)((runs - 1 - blockIdx.x) / gridDim.x) * gridDim.x + blockIdx.x; r >= 0; r -= gridDim.x) {
        const uint32_t c0 = (uint32_t)r * run;
        uint32_t c = min(c0 + run, chunks);
        for (int k = gn_find(tab, c - 1); c > c0; --k) {
            const uint32_t first = tab.first[k], begin = max(c0, first);
            const int type = (int)(tab.data[k] >> 62), len = gn_chunk_len(type);
            char *p = (char *)(tab.data[k] & ~(3ull << 62));
            const int64_t e0 = (int64_t)(begin - first) * len, e1 = min((int64_t)(c - first) * len, tab.n[k]);
            if (type == GN_F32) gn_scale_part<GN_F32, NT, BLOCK>(p + e0 * 4, e1 - e0, f);
            else if (type == GN_BF16) gn_scale_part<GN_BF16, NT, BLOCK>(p + e0 * 2, e1 - e0, f);
            else gn_scale_part<GN_F16, NT, BLOCK>(p + e0 * 2, e1 - e0, f);
            c = begin;
        }
    }
}

// n_part > 0: every workgroup adds the parts up itself, in the same order, and the first one writes the norm; n_part = 0: the factor is there.
// NT: the list is longer than what stays in the cache.
template <int P, bool NT>
__global__ void __launch_bounds__(NT ? NVDR_GN_STREAM_BLOCK : NVDR_GN_BLOCK)
grad_scale_kernel(GradTable tab, const double *__restrict__ part, int n_part, double max_norm, float *__restrict__ norm, const float *__restrict__ factor)
{
    __shared__ double lds[NVDR_GN_STREAM_BLOCK / 64];
    float f;
    if (n_part > 0) {
        const double v = gn_total<P>(part, n_part, lds);
        f = gn_factor(v, max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
    } else f = *factor;
    if (f == 1.0f) return;
    gn_scale_runs<NT, NT ? NVDR_GN_STREAM_BLOCK : NVDR_GN_BLOCK>(tab, f);
}

// a short list: the norm and the scaling by one workgroup.  The barriers of the sum lie between the last read and the first write.
template <int P>
__global__ void __launch_bounds__(NVDR_GN_ONE_BLOCK) grad_clip_one_kernel(GradTable tab, double max_norm, float *__restrict__ norm)
{
    __shared__ double lds[NVDR_GN_ONE_BLOCK / 64];
    const double v = gn_root<P>(gn_block_join<P>(gn_sum_runs<P, NVDR_GN_ONE_BLOCK>(tab), lds));
    if (threadIdx.x == 0) *norm = (float)v;
    const float f = gn_factor(v, max_norm);
    if (f != 1.0f && tab.n_tensors) gn_scale_runs<false, NVDR_GN_ONE_BLOCK>(tab, f);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
struct GradList {
    const void *const *data;
    const int64_t *n;
    const uint8_t *type;
    const float *scale;         // NULL: one
    int64_t count;
};

static int64_t gn_size(int type) { return type == GN_F32 ? 4 : 2; }

static int64_t gn_bytes(const GradList &l)
{
    int64_t bytes = 0;
    for (int64_t k = 0; k < l.count; ++k) bytes += l.n[k] * gn_size(l.type[k]);
    return bytes;
}

static bool gn_one(const GradList &l, int64_t bytes) { return l.count <= NVDR_GN_ONE_TENSORS && bytes <= NVDR_GN_ONE_CLIP; }

// in doubles: the parts, the words of the last launch, the factor of nvdr_grad_clip.  (A launch ends with the list or with a full table; the split by
// the number of chunks needs more than 2^31 of them, 8 TB.)
static int64_t gn_part_room(int64_t count) { return ((count + NVDR_GN_TENSORS - 1) / NVDR_GN_TENSORS + 1) * NVDR_GN_GRID; }
static int64_t gn_workspace(const GradList &l, bool clip)
{
    // (a long list is not walked for its bytes)
    return clip && l.count <= NVDR_GN_ONE_TENSORS && gn_one(l, gn_bytes(l)) ? 0 : gn_part_room(l.count) + 2 * NVDR_GN_GRID + 1;
}

static int gn_check(const GradList &l, int norm_type, double max_norm, bool clip, const double *workspace, int64_t workspace_len, const float *norm, const char *who)
{
    NVDR_REQUIRE(l.count >= 0 && l.count < (1ll << 24), "%s: %lld tensors", who, (long long)l.count);
    NVDR_REQUIRE(l.count == 0 || (l.data && l.n && l.type), "%s: NULL argument", who);
    NVDR_REQUIRE(norm, "%s: room for the norm is needed", who);
    NVDR_REQUIRE(norm_type == NVDR_NORM_INF || norm_type == NVDR_NORM_1 || norm_type == NVDR_NORM_2, "%s: norm type %d", who, norm_type);
    NVDR_REQUIRE(max_norm >= 0.0, "%s: max_norm has to be zero or more", who);       // (a NaN fails too)
    for (int64_t k = 0; k < l.count; ++k) {
        NVDR_REQUIRE(l.type[k] <= GN_F16, "%s: tensor %lld has type %d", who, (long long)k, (int)l.type[k]);
        NVDR_REQUIRE(l.n[k] >= 0 && l.n[k] < (1ll << 40), "%s: tensor %lld has %lld elements", who, (long long)k, (long long)l.n[k]);
        NVDR_REQUIRE(l.n[k] == 0 || (l.data[k] && (uintptr_t)l.data[k] < (1ull << 62)), "%s: tensor %lld has no memory", who, (long long)k);
        NVDR_REQUIRE(((uintptr_t)l.data[k] & (uintptr_t)(gn_size(l.type[k]) - 1)) == 0, "%s: tensor %lld is not aligned to its elements", who, (long long)k);
    }
    const int64_t need = gn_workspace(l, clip);
    NVDR_REQUIRE(need == 0 || (workspace && ((uintptr_t)workspace & 7) == 0 && workspace_len >= need), "%s: an 8-byte aligned workspace of %lld doubles is needed, there are %lld",
                 who, (long long)need, (long long)(workspace ? workspace_len : 0));
    return 0;
}

// in place: no byte may belong to two tensors (two workgroups would scale it, or one read what the other has scaled)
static int gn_check_apart(const GradList &l, const char *who)
{
    typedef std::pair<uintptr_t, uintptr_t> Span;
    uintptr_t last = 0;
    bool ordered = true;
    for (int64_t k = 0; k < l.count && ordered; ++k) {
        if (l.n[k] == 0) continue;
        ordered = (uintptr_t)l.data[k] >= last;
        last = (uintptr_t)l.data[k] + (uintptr_t)(l.n[k] * gn_size(l.type[k]));
    }
    if (ordered) return 0;
    Span *s = (Span *)malloc(sizeof(Span) * (size_t)l.count);
    NVDR_REQUIRE(s, "%s: out of host memory", who);
    int64_t m = 0;
    for (int64_t k = 0; k < l.count; ++k)
        if (l.n[k]) s[m++] = Span((uintptr_t)l.data[k], (uintptr_t)l.data[k] + (uintptr_t)(l.n[k] * gn_size(l.type[k])));
    std::sort(s, s + m, [](const Span &a, const Span &b) { return a.first < b.first; });      // (none is empty: equal beginnings overlap)
    bool apart = true;
    for (int64_t k = 1; k < m; ++k) apart = apart && s[k].first >= s[k - 1].second;
    free(s);
    NVDR_REQUIRE(apart, "%s: two gradients share memory (the same tensor twice, or overlapping views)", who);
    return 0;
}

// fills `tab` with tensors from *at on, moves *at behind them and takes their bytes from *left; returns the workgroups of the launch, `most` at
// most (0: nothing left)
static unsigned gn_fill(const GradList &l, int64_t *at, int64_t *left, uint64_t most, GradTable &tab)
{
    int m = 0;
    uint64_t chunks = 0;
    tab.first[0] = 0;
    while (*at < l.count) {
        const int64_t k = *at, n = l.n[k];
        const int type = l.type[k];
        const uint64_t word = (uint64_t)(uintptr_t)l.data[k] | ((uint64_t)type << 62);
        const float scale = l.scale ? l.scale[k] : 1.0f;
        const int64_t size = gn_size(type), len = NVDR_GN_CHUNK / size;
        if (n == 0) { ++*at; continue; }
        // directly behind the one before, same type and scale: one tensor
        const bool more = m && tab.data[m - 1] + (uint64_t)(tab.n[m - 1] * size) == word && tab.scale[m - 1] == scale;
        const uint64_t front = more ? tab.first[m - 1] : chunks, c = front + (((uint64_t)((more ? tab.n[m - 1] : 0) + n + len - 1)) >> (type == GN_F32 ? 10 : 11));
        if ((!more && m == NVDR_GN_TENSORS) || (m && c >= (1ull << 31))) break;
        if (more) tab.n[m - 1] += n;
        else {
            tab.data[m] = word; tab.n[m] = n; tab.scale[m] = scale;
            ++m;
        }
        chunks = c;
        tab.first[m] = (uint32_t)chunks;
        *left -= n * size;
        ++*at;
    }
    tab.n_tensors = m;
    tab.chunks = (uint32_t)chunks;
    for (int q = m; q < 9; ++q) tab.first[q] = (uint32_t)chunks;           // (gn_find compares eight)
    tab.run = 1;
    tab.kept = 0;
    if (chunks == 0) return 0;
    // as few rounds as runs of NVDR_GN_RUN bytes give, all of the same length
    const uint64_t grid = chunks < most ? chunks : most, per = NVDR_GN_RUN / NVDR_GN_CHUNK;
    const uint64_t rounds = (chunks + grid * per - 1) / (grid * per);
    tab.run = (uint32_t)((chunks + grid * rounds - 1) / (grid * rounds));
    const uint64_t stay = *left >= NVDR_GN_KEEP ? 0 : (uint64_t)(NVDR_GN_KEEP - *left) / NVDR_GN_CHUNK;      // of this launch, given what follows it
    tab.kept = (uint32_t)(stay >= chunks ? 0 : chunks - stay);
    const uint64_t runs = (chunks + tab.run - 1) / tab.run;
    return (unsigned)(runs < grid ? runs : grid);
}

extern "C" int64_t nvdr_grad_norm_workspace(const int64_t *n, const uint8_t *type, int64_t n_tensors, int clip)
{
    const GradList l = {nullptr, n, type, nullptr, n_tensors};
    if (n_tensors < 0 || (n_tensors && (!n || !type))) return 0;
    return gn_workspace(l, clip != 0);
}

#define NVDR_GN_STARTS 64
struct GradLaunches {
    int64_t start[NVDR_GN_STARTS], left[NVDR_GN_STARTS];        // of the first launches: the scaling takes them in reverse
    int64_t count = 0;
    int n_part = 0;
};

// keys of its own for every norm: splitmix64 of a counter, a bijection
static GradKeys gn_keys()
{
    static std::atomic<unsigned long long> counter{(unsigned long long)std::chrono::steady_clock::now().time_since_epoch().count() << 20};
    const unsigned long long at = counter.fetch_add(2, std::memory_order_relaxed);
    auto mix = [](unsigned long long z) {
        z *= 0x9e3779b97f4a7c15ull;
        z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
        z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
        return z ^ (z >> 31);
    };
    return {mix(at), mix(at + 1)};          // (of two different counts: never equal, so that erased words do not open)
}

// the launches of the norm; finish: the last one writes it.  tab: as the last one had it
template <int P>
static int gn_parts(const GradList &l, int64_t bytes, double *part, bool finish, const GradOut &out, GradLaunches &g, GradTable &tab, hipStream_t st)
{
    unsigned long long *words = (unsigned long long *)(part + gn_part_room(l.count));
    int64_t at = 0, left = bytes;
    do {
        if (g.count < NVDR_GN_STARTS) { g.start[g.count] = at; g.left[g.count] = left; }
        unsigned blocks = gn_fill(l, &at, &left, NVDR_GN_GRID, tab);
        while (at < l.count && l.n[at] == 0) ++at;                  // (nothing but empty tensors left: this is the last launch)
        if (finish && at == l.count) {
            if (!blocks) blocks = 1;                                // (nothing at all: a norm of zero)
            grad_norm_kernel<P, true><<<blocks, NVDR_GN_BLOCK, 0, st>>>(tab, part, words, gn_keys(), g.n_part, out);
        } else if (blocks) grad_norm_kernel<P, false><<<blocks, NVDR_GN_BLOCK, 0, st>>>(tab, part, words, GradKeys{}, g.n_part, out);
        NVDR_LAUNCH_CHECK();
        g.n_part += (int)blocks;
        ++g.count;
    } while (at < l.count);
    return 0;
}

template <int P>
static int gn_norm(const GradList &l, double *part, const GradOut &out, hipStream_t st)
{
    GradLaunches g;
    GradTable tab;
    return gn_parts<P>(l, gn_bytes(l), part, true, out, g, tab, st);
}

static int gn_norm_typed(const GradList &l, int norm_type, double *part, const GradOut &out, hipStream_t st)
{
    return norm_type == NVDR_NORM_INF ? gn_norm<GN_INF>(l, part, out, st) : norm_type == NVDR_NORM_1 ? gn_norm<GN_ONE>(l, part, out, st) : gn_norm<GN_TWO>(l, part, out, st);
}

template <int P>
static int gn_clip(const GradList &l, double max_norm, double *part, float *norm, float *factor, hipStream_t st)
{
    const int64_t bytes = gn_bytes(l);
    GradTable tab;
    if (gn_one(l, bytes)) {
        int64_t at = 0, left = bytes;
        gn_fill(l, &at, &left, 1, tab);
        grad_clip_one_kernel<P><<<1, NVDR_GN_ONE_BLOCK, 0, st>>>(tab, max_norm, norm);
        NVDR_LAUNCH_CHECK();
        return 0;
    }
    // one table: the scaling adds the parts up itself; several, or nothing to scale: the last launch of the norm leaves the norm and the factor
    const bool finish = l.count > NVDR_GN_TENSORS || bytes == 0;
    GradLaunches g;
    GradOut out = {};
    out.max_norm = max_norm; out.norm = norm; out.factor = factor;
    if (int r = gn_parts<P>(l, bytes, part, finish, out, g, tab, st)) return r;
    const int n_part = finish ? 0 : g.n_part;
    const bool stream = bytes > NVDR_GN_KEEP;
    if (g.count == 1 && !stream) {                                  // the table of the norm's one launch is the scaling's
        if (bytes) grad_scale_kernel<P, false><<<(unsigned)g.n_part, NVDR_GN_BLOCK, 0, st>>>(tab, part, n_part, max_norm, norm, factor);
        NVDR_LAUNCH_CHECK();
        return 0;
    }
    auto launch = [&](int64_t at, int64_t left, int64_t *behind, int64_t *after) -> bool {
        const unsigned blocks = gn_fill(l, &at, &left, stream ? NVDR_GN_STREAM_GRID : NVDR_GN_GRID, tab);
        if (blocks && stream) grad_scale_kernel<P, true><<<blocks, NVDR_GN_STREAM_BLOCK, 0, st>>>(tab, part, n_part, max_norm, norm, factor);
        else if (blocks) grad_scale_kernel<P, false><<<blocks, NVDR_GN_BLOCK, 0, st>>>(tab, part, n_part, max_norm, norm, factor);
        *behind = at; *after = left;
        return blocks != 0;
    };
    int64_t at = 0, left = bytes;
    const int64_t known = g.count < NVDR_GN_STARTS ? g.count : NVDR_GN_STARTS;
    for (int64_t k = known - 1; k >= 0; --k) {
        int64_t a, b;
        launch(g.start[k], g.left[k], &a, &b);
        NVDR_LAUNCH_CHECK();
        if (k == known - 1) { at = a; left = b; }
    }
    while (launch(at, left, &at, &left)) NVDR_LAUNCH_CHECK();
    return 0;
}

extern "C" int nvdr_grad_norm(const void *const *data, const int64_t *n, const uint8_t *type, const float *scale, int64_t n_tensors, int norm_type, double max_norm,
                              double *workspace, int64_t workspace_len, float *norm, float *factor, void *stream)
{
    NvdrRange range("nvdr_grad_norm");
    const GradList l = {data, n, type, scale, n_tensors};
    if (int r = gn_check(l, norm_type, max_norm, false, workspace, workspace_len, norm, "nvdr_grad_norm")) return r;
    GradOut out = {};
    out.max_norm = max_norm; out.norm = norm; out.factor = factor;
    return gn_norm_typed(l, norm_type, workspace, out, (hipStream_t)stream);
}

int nvdr_adam_norm(const nvdr_adam_tensor *tensors, int n_tensors, int norm_type, double max_norm, double *workspace, int64_t workspace_len, float *norm,
                   const AdamBegin &adam, hipStream_t stream)
{
    const void *data[NVDR_ADAM_MAX_TENSORS];
    int64_t n[NVDR_ADAM_MAX_TENSORS];
    uint8_t type[NVDR_ADAM_MAX_TENSORS];
    float scale[NVDR_ADAM_MAX_TENSORS];
    int m = 0;
    for (int k = 0; k < n_tensors; ++k) {
        if (tensors[k].frozen) continue;
        data[m] = tensors[k].grad; n[m] = tensors[k].n; type[m] = GN_F32; scale[m] = tensors[k].grad_scale;
        ++m;
    }
    const GradList l = {data, n, type, scale, m};
    if (int r = gn_check(l, norm_type, max_norm, false, workspace, workspace_len, norm, "nvdr_adam_step_clipped")) return r;
    GradOut out = {};
    out.max_norm = max_norm; out.norm = norm; out.adam = adam;
    return gn_norm_typed(l, norm_type, workspace, out, stream);
}

extern "C" int nvdr_grad_clip(void *const *data, const int64_t *n, const uint8_t *type, int64_t n_tensors, int norm_type, double max_norm, double *workspace,
                              int64_t workspace_len, float *norm, void *stream)
{
    NvdrRange range("nvdr_grad_clip");
    const GradList l = {(const void *const *)data, n, type, nullptr, n_tensors};
    if (int r = gn_check(l, norm_type, max_norm, true, workspace, workspace_len, norm, "nvdr_grad_clip")) return r;
    if (int r = gn_check_apart(l, "nvdr_grad_clip")) return r;
    float *factor = workspace ? (float *)(workspace + workspace_len - 1) : nullptr;
    switch (norm_type) {
    case NVDR_NORM_INF: return gn_clip<GN_INF>(l, max_norm, workspace, norm, factor, (hipStream_t)stream);
    case NVDR_NORM_1: return gn_clip<GN_ONE>(l, max_norm, workspace, norm, factor, (hipStream_t)stream);
    default: return gn_clip<GN_TWO>(l, max_norm, workspace, norm, factor, (hipStream_t)stream);
    }
}
