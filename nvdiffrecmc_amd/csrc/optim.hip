// optim.hip -- the parameter update of one training iteration as ONE launch.
//
// Replaces, for the three tensors the direct-lighting iteration trains (kd texture, ks, light probe), the sequence
//     lgt.base.grad *= 64                      train.py:439-440
//     optimizer.step()                         train.py:452-461  (torch.optim.Adam, no weight decay, no amsgrad)
//     clamps of the parameters                 train.py:470-476 / material clamps
// which on ROCm is a multi-tensor Adam launch that puts ~1 M elements on 16 workgroups (45 us on a 256-CU part) plus five
// small elementwise kernels.  All tensors in one launch, the step counter in device memory (the launch can be
// captured in a HIP graph and replayed), same arithmetic and the same order of operations as torch's single-tensor Adam:
//     m = m + (g - m) * (1 - b1);  v = v * b2 + (1 - b2) * g * g
//     p = p - (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps);  p = max(min(p, hi), lo)
//
// With clipping (nvdr_adam_step_clipped) the norm of the effective gradients comes first (gradnorm.hip) and its factor enters g, as one product
// with the scale (an outlier times the scale alone can leave fp32 where its clipped value does not): the gradients are read once more, not written, and no launch follows for the step counter.
//
// Bytes bound it: 28 per parameter.  10.7 M parameters of the scene's set, 298 MB: 72 us with one element a lane and access, 64 us with
// sixteen bytes, 48 us (6.2 TB/s, what a large copy reaches) with the moments past the caches.  Textures by tiles (12 bytes a texel where
// nothing is to do): 3 x 1024^2 at a quarter of the tiles 23.7 -> 19 us, at a twentieth 15.0 -> 12.5 us.
#include "common.h"
#include "gradnorm.h"
#include "nvdr_hip.h"

#define ADAM_TILE 64             // texels of a tile of the sparse-texture path
#define ADAM_TILES 4             // tiles of a wavefront
#define ADAM_BLOCK 256
#define ADAM_ROUNDS 2            // groups of four elements that a thread of the plain path takes, all their loads in flight
// Bytes of a step from which on the moments go past the caches: a step of fewer leaves all it touches in the 256 MB last-level cache for the
// next one; of more, the moments only push out the parameters, which the next forward pass reads, and the gradients, which the norm has just
// read.  (10.7 M parameters = 298 MB a step: 51 us with non-temporal moments, 64 us without.)
#define NVDR_ADAM_KEEP (160ll << 20)
struct AdamTable {
    nvdr_adam_tensor t[NVDR_ADAM_MAX_TENSORS];
    int first_block[NVDR_ADAM_MAX_TENSORS + 1];     // workgroups [first_block[k], first_block[k + 1]) work on tensor k
    int n;
};

typedef float adam_f4 __attribute__((ext_vector_type(4)));

// Four elements from e on; behind the end of the tensor zeros are loaded and nothing is stored.  `wide`: the buffer is 16-byte aligned (e is a
// multiple of four); one that is not -- a gradient inside an exchange bucket -- goes element by element
// NT: past the caches (see NVDR_ADAM_KEEP)
template <bool NT>
__device__ __forceinline__ void adam_load(float (&x)[4], const float *p, int64_t e, int64_t n, bool wide)
{
    if (wide && e + 4 <= n) {
        const adam_f4 *q = (const adam_f4 *)(p + e);
        const adam_f4 v = NT ? __builtin_nontemporal_load(q) : *q;
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = e + c < n ? p[e + c] : 0.0f;
    }
}

template <bool NT>
__device__ __forceinline__ void adam_store(const float (&x)[4], float *p, int64_t e, int64_t n, bool wide)
{
    if (wide && e + 4 <= n) {
        const adam_f4 v = {x[0], x[1], x[2], x[3]};
        if (NT) __builtin_nontemporal_store(v, (adam_f4 *)(p + e));
        else *(adam_f4 *)(p + e) = v;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (e + c < n) p[e + c] = x[c];
    }
}

// a texel of three channels: one access of twelve bytes, whatever the alignment
template <bool NT>
__device__ __forceinline__ void adam_load(float (&x)[3], const float *p)
{
#pragma unroll
    for (int c = 0; c < 3; ++c) x[c] = NT ? __builtin_nontemporal_load(p + c) : p[c];
}

template <bool NT>
__device__ __forceinline__ void adam_store(const float (&x)[3], float *p)
{
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        if (NT) __builtin_nontemporal_store(x[c], p + c);
        else p[c] = x[c];
    }
}

struct AdamConst {
    float scale, step_size, bc2_sqrt, beta2, omb1, omb2, eps;
};

// the moments and the parameter of N elements from e on
template <int N>
__device__ __forceinline__ void adam_update(const nvdr_adam_tensor &T, const AdamConst &k, int64_t e, const float (&g)[N], float (&m)[N], float (&v)[N], float (&p)[N])
{
    float lo[N], hi[N];
#pragma unroll
    for (int c = 0; c < N; ++c) { lo[c] = T.lo; hi[c] = T.hi; }
    if (T.lo_vec) {
        int64_t i = e % T.lo_vec_n;
#pragma unroll
        for (int c = 0; c < N; ++c) { lo[c] = fmaxf(lo[c], T.lo_vec[i]); i = i + 1 == T.lo_vec_n ? 0 : i + 1; }
    }
    if (T.hi_vec) {
        int64_t i = e % T.hi_vec_n;
#pragma unroll
        for (int c = 0; c < N; ++c) { hi[c] = fminf(hi[c], T.hi_vec[i]); i = i + 1 == T.hi_vec_n ? 0 : i + 1; }
    }
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const float gg = g[c] * k.scale;
        m[c] = m[c] + (gg - m[c]) * k.omb1;                         // lerp_(grad, 1 - beta1)
        v[c] = v[c] * k.beta2 + (k.omb2 * gg) * gg;                 // mul_(beta2).addcmul_(grad, grad, value = 1 - beta2)
        const float denom = sqrtf(v[c]) / k.bc2_sqrt + k.eps;
        const float q = p[c] - k.step_size * (m[c] / denom);        // addcdiv_(exp_avg, denom, value = -step_size)
        p[c] = q < lo[c] ? lo[c] : (q > hi[c] ? hi[c] : q);         // torch.clamp semantics: a NaN parameter stays NaN
    }
}

template <bool NT>
__device__ __forceinline__ void adam_texel(const nvdr_adam_tensor &T, const AdamConst &k, int64_t e, const float (&g)[3])
{
    float m[3], v[3], p[3];
    adam_load<NT>(m, T.exp_avg + e);
    adam_load<NT>(v, T.exp_avg_sq + e);
    adam_load<NT>(p, T.param + e);
    adam_update(T, k, e, g, m, v, p);
    if (T.normalize3) {             // Texture2D.clamp_ + normalize_ of the normal map, train.py:470-474, render/texture.py:86-96
        const float len = sqrtf(fmaxf((p[0] * p[0] + p[1] * p[1]) + p[2] * p[2], 1e-20f));      // util.safe_normalize
        p[0] /= len; p[1] /= len; p[2] /= len;
    }
    adam_store<NT>(m, T.exp_avg + e);
    adam_store<NT>(v, T.exp_avg_sq + e);
    adam_store<false>(p, T.param + e);
}

// begin: what the kernel that finished the norm has prepared of this step (the counter has moved already); NULL: from state, with *grad_factor
template <bool STREAM>
__global__ void __launch_bounds__(ADAM_BLOCK) adam_step_kernel(AdamTable tab, double lr, double beta1d, double beta2d, float eps, const int *state,
                                                                const float *grad_factor, const AdamStep *begin)
{
    // state[0] = steps taken so far, state[1] unused, then two doubles: beta1^step, beta2^step (kept as running products: pow() in
    // double costs a workgroup ~10 us of latency); read-only here
    // the tensor of this workgroup: uniform, and all of its entry at once (a field read where it is used is a round trip of its own; first_block
    // of the entries behind the last tensor is the number of workgroups)
    int k = 0;
#pragma unroll
    for (int q = 1; q < NVDR_ADAM_MAX_TENSORS; ++q) k += (int)blockIdx.x >= tab.first_block[q] ? 1 : 0;
    const nvdr_adam_tensor T = tab.t[k];
    AdamStep S;
    if (begin) S = *begin;
    else {
        __shared__ AdamStep shared;
        if (threadIdx.x == 0) {
            shared = adam_begin(state, lr, beta1d, beta2d);
            if (grad_factor) shared.factor = *grad_factor;
        }
        __syncthreads();
        S = shared;
    }
    const int64_t block = (int64_t)((int)blockIdx.x - tab.first_block[k]);
    // the hyper-parameters arrive as doubles, like the Python floats torch's Adam computes 1 - beta from: (float)(1 - 0.999) is
    // 0.001f, 1 - 0.999f is 1.3e-5 off (visible in the parameters after ten steps)
    // lr_scale: this tensor's learning rate (train.py:336-338: position / material / light; a zero-initialised block: the plain rate)
    // grad_scale and the factor as one product: an outlier times the scale alone may be infinite where clipping bounds it
    const AdamConst c = {T.grad_scale * S.factor, S.step_size * (T.lr_scale == 0.0f ? 1.0f : T.lr_scale), S.bc2_sqrt, (float)beta2d, (float)(1.0 - beta1d), (float)(1.0 - beta2d), eps};
    const bool wide_g = ((uintptr_t)T.grad & 15) == 0, wide_m = ((uintptr_t)T.exp_avg & 15) == 0, wide_v = ((uintptr_t)T.exp_avg_sq & 15) == 0,
               wide_p = ((uintptr_t)T.param & 15) == 0;
    if (T.frozen && !(T.active && T.zero_grad)) return;
    if (T.active || T.normalize3) {
        // TEXELS of three channels: a lane takes one, a wavefront ADAM_TILES tiles of 64.
        //
        // Sparse textures (T.active).  A trained texture of 1024^2 texels receives gradient only at the texels some covered pixel
        // looked up -- ~5 % of them with the fixed benchmark views -- and a texel that has never received any still has zero moments:
        // its update is p - step * 0 / (0 + eps) = p, a clamp of a value the first step already clamped.  Tiles with an all-zero
        // gradient and no history are therefore skipped after reading the gradient alone: 12 instead of 84 bytes per texel, EXACTLY
        // the same parameters (step 1 visits every tile, so that the clamps / the normalisation have been applied to whatever the
        // initial values were; a step whose factor is a NaN or infinite makes 0 * factor a NaN, as in a dense tensor, and visits every tile
        // too; a normal is not normalised again where nothing else is done, a rounding or two of it).  `active[tile]` remembers history.  zero_grad: the gradient of a visited tile is zeroed behind the
        // update, so that a scatter-add backward (nvdr_texture_lookup_bwd into a persistent buffer) needs no memset of 3 x 12.6 MB per
        // iteration.
        //
        // The loop over the tiles is NOT unrolled: what a wavefront runs once has to be fetched, and straight-line code for all the
        // tiles took 10 us more at a twentieth of the tiles touched.
        const int lane = threadIdx.x & 63;
        const int64_t texels = T.n / 3, tile0 = (block * (ADAM_BLOCK / 64) + (threadIdx.x >> 6)) * ADAM_TILES;
        unsigned any = 0, visit = (1u << ADAM_TILES) - 1;
        if (T.active) {
            const int64_t tiles = (texels + ADAM_TILE - 1) / ADAM_TILE;
            float g[ADAM_TILES][3];
            unsigned history = 0;
#pragma unroll
            for (int j = 0; j < ADAM_TILES; ++j) {              // the gradients (and histories) of all tiles of this wavefront first: one round trip
                const int64_t t = (tile0 + j) * ADAM_TILE + lane;
                g[j][0] = g[j][1] = g[j][2] = 0.0f;
                if (t < texels) adam_load<false>(g[j], T.grad + 3 * t);
            }
            const bool mine = lane < ADAM_TILES && tile0 + lane < tiles;
            history = (unsigned)__ballot(mine && T.active[mine ? tile0 + lane : 0] != 0);
#pragma unroll
            for (int j = 0; j < ADAM_TILES; ++j)
                any |= (__ballot(g[j][0] != 0.0f || g[j][1] != 0.0f || g[j][2] != 0.0f) != 0ull ? 1u : 0u) << j;      // (a NaN compares unequal to zero)
            const bool spoiled = !(c.scale * 0.0f == 0.0f);
            if (T.frozen) visit = 0;
            else if (S.step > 1 && !spoiled) visit = any | history;
            if (!T.frozen && mine && (((spoiled ? visit : any) & ~history) >> lane & 1u)) T.active[tile0 + lane] = 1;
        }
#pragma unroll 1
        for (int j = 0; j < ADAM_TILES; ++j) {
            const int64_t t = (tile0 + j) * ADAM_TILE + lane;
            if (!((visit | any) >> j & 1u) || t >= texels) continue;
            float g[3];
            adam_load<false>(g, T.grad + 3 * t);                // (again: out of the cache)
            if (visit >> j & 1u) {
                if (STREAM && !T.active) adam_texel<true>(T, c, 3 * t, g);
                else adam_texel<false>(T, c, 3 * t, g);
            }
            // A frozen tensor (lr_scale 0 on the host) takes no update, but its gradient is still CONSUMED: with zero_grad the producer
            // scatter-adds into a persistent buffer that nobody else clears -- and with several ranks that buffer is the exchange bucket,
            // all-reduced in place every step: left alone its content would grow by the world size per iteration until it overflows.
            if (T.zero_grad && (any >> j & 1u)) {
                const float zero[3] = {0.0f, 0.0f, 0.0f};
                adam_store<false>(zero, const_cast<float *>(T.grad) + 3 * t);
            }
        }
        return;
    }
    const int64_t e0 = block * (ADAM_BLOCK * 4 * ADAM_ROUNDS) + threadIdx.x * 4;
    float g[ADAM_ROUNDS][4], m[ADAM_ROUNDS][4], v[ADAM_ROUNDS][4], p[ADAM_ROUNDS][4];
#pragma unroll
    for (int u = 0; u < ADAM_ROUNDS; ++u) {
        const int64_t e = e0 + u * (ADAM_BLOCK * 4);
        adam_load<false>(g[u], T.grad, e, T.n, wide_g);
        adam_load<STREAM>(m[u], T.exp_avg, e, T.n, wide_m);
        adam_load<STREAM>(v[u], T.exp_avg_sq, e, T.n, wide_v);
        adam_load<STREAM>(p[u], T.param, e, T.n, wide_p);
    }
#pragma unroll
    for (int u = 0; u < ADAM_ROUNDS; ++u) {
        const int64_t e = e0 + u * (ADAM_BLOCK * 4);
        adam_update(T, c, e, g[u], m[u], v[u], p[u]);
        adam_store<STREAM>(m[u], T.exp_avg, e, T.n, wide_m);
        adam_store<STREAM>(v[u], T.exp_avg_sq, e, T.n, wide_v);
        adam_store<false>(p[u], T.param, e, T.n, wide_p);
    }
}

// The step counter and the running powers move in a launch of their own (one thread, ~4 us) behind the update: every workgroup of the
// update has read them by then (stream order).  Tickets that the workgroups of the update draw on ONE word, the last one
// publishing the state, cost more: up to 2 048 same-address atomics, which retire one every ~12 ns -- 25 us of a 33 us kernel.  (A clipped step of all
// tensors needs no launch for it: the kernel that finishes the norm prepares the step and moves the counter.)
__global__ void adam_advance_kernel(int *state, double beta1d, double beta2d) { adam_advance(state, beta1d, beta2d); }

static bool adam_overlap(const float *a, int64_t na, const float *b, int64_t nb) { return na > 0 && nb > 0 && a < b + nb && b < a + na; }

// checks the tensors of a step and deals the workgroups; *blocks_out = how many, *stream_out = whether the moments go past the caches (a sparse
// texture does not count: what a step touches of it is few tiles, and known to the device alone)
static int adam_table(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps, const int *state, AdamTable &tab, unsigned *blocks_out,
                      bool *stream_out)
{
    NVDR_REQUIRE(tensors && state, "adam_step: NULL argument");
    NVDR_REQUIRE(n_tensors >= 1 && n_tensors <= NVDR_ADAM_MAX_TENSORS, "adam_step: %d tensors (1..%d supported)", n_tensors, NVDR_ADAM_MAX_TENSORS);
    NVDR_REQUIRE(lr >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "adam_step: bad hyper-parameters");
    memset(&tab, 0, sizeof(tab));
    tab.n = n_tensors;
    int64_t total = 0, dense = 0;
    for (int k = 0; k < n_tensors; ++k) {
        const nvdr_adam_tensor &t = tensors[k];
        NVDR_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq && t.n >= 0, "adam_step: tensor %d has a NULL buffer", k);
        for (int j = 0; j < k; ++j) {
            const nvdr_adam_tensor &o = tensors[j];
            const float *const mine[3] = {t.param, t.exp_avg, t.exp_avg_sq}, *const others[3] = {o.param, o.exp_avg, o.exp_avg_sq};
            for (int a = 0; a < 9; ++a)
                NVDR_REQUIRE(!adam_overlap(mine[a / 3], t.n, others[a % 3], o.n), "adam_step: tensors %d and %d are the same or overlap (two workgroups would update them)", j, k);
            NVDR_REQUIRE(!(o.zero_grad || t.zero_grad) || !adam_overlap(o.grad, o.n, t.grad, t.n), "adam_step: tensors %d and %d share a gradient that zero_grad clears", j, k);
        }
        NVDR_REQUIRE(!t.lo_vec || t.lo_vec_n > 0, "adam_step: tensor %d: lo_vec without length", k);
        NVDR_REQUIRE(!t.hi_vec || t.hi_vec_n > 0, "adam_step: tensor %d: hi_vec without length", k);
        NVDR_REQUIRE(!t.normalize3 || t.n % 3 == 0, "adam_step: tensor %d: normalize3 needs a multiple of three elements", k);
        NVDR_REQUIRE(t.lr_scale >= 0.0f, "adam_step: tensor %d: negative lr_scale (0 = the plain rate; `frozen` freezes)", k);
        NVDR_REQUIRE(!t.active || t.n % 3 == 0, "adam_step: tensor %d: the sparse path works on texels of three channels", k);
        NVDR_REQUIRE(!t.zero_grad || t.active, "adam_step: tensor %d: zero_grad needs the sparse path (active)", k);
        tab.t[k] = t;
        total += t.n;
        if (!t.active && !t.frozen) dense += t.n;
    }
    NVDR_REQUIRE(total < (1ll << 40), "adam_step: too many elements");
    int64_t blocks = 0;
    for (int k = 0; k < n_tensors; ++k) {
        tab.first_block[k] = (int)blocks;
        blocks += tensors[k].active || tensors[k].normalize3 ? div_up(tensors[k].n, ADAM_BLOCK * ADAM_TILES * 3) : div_up(tensors[k].n, ADAM_BLOCK * 4 * ADAM_ROUNDS);
    }
    for (int k = n_tensors; k <= NVDR_ADAM_MAX_TENSORS; ++k) tab.first_block[k] = (int)blocks;
    *blocks_out = (unsigned)(blocks < 1 ? 1 : blocks);
    *stream_out = 28 * dense > NVDR_ADAM_KEEP;
    return 0;
}

static void adam_launch(const AdamTable &tab, unsigned blocks, bool past, double lr, double beta1, double beta2, double eps, const int *state, const float *grad_factor,
                        const AdamStep *begin, hipStream_t st)
{
    if (past) adam_step_kernel<true><<<blocks, ADAM_BLOCK, 0, st>>>(tab, lr, beta1, beta2, (float)eps, state, grad_factor, begin);
    else adam_step_kernel<false><<<blocks, ADAM_BLOCK, 0, st>>>(tab, lr, beta1, beta2, (float)eps, state, grad_factor, begin);
}

extern "C" int nvdr_adam_step(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps,
                              int *state, void *stream_)
{
    return nvdr_adam_step_partial(tensors, n_tensors, lr, beta1, beta2, eps, state, 1, stream_);
}

extern "C" int nvdr_adam_step_partial(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps,
                                      int *state, int advance, void *stream_)
{
    return nvdr_adam_step_factor(tensors, n_tensors, lr, beta1, beta2, eps, state, advance, nullptr, stream_);
}

extern "C" int nvdr_adam_step_factor(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps,
                                     int *state, int advance, const float *grad_factor, void *stream_)
{
    NvdrRange range("nvdr_adam_step");
    AdamTable tab;
    unsigned blocks;
    bool past;
    if (int r = adam_table(tensors, n_tensors, lr, beta1, beta2, eps, state, tab, &blocks, &past)) return r;
    adam_launch(tab, blocks, past, lr, beta1, beta2, eps, state, grad_factor, nullptr, (hipStream_t)stream_);
    if (advance) adam_advance_kernel<<<1, 1, 0, (hipStream_t)stream_>>>(state, beta1, beta2);
    NVDR_LAUNCH_CHECK();
    return 0;
}

extern "C" int nvdr_adam_step_clipped(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps,
                                      int *state, int norm_type, double max_norm, double *workspace, int64_t workspace_len, float *norm, void *stream_)
{
    NvdrRange range("nvdr_adam_step");
    AdamTable tab;
    unsigned blocks;
    bool past;
    if (int r = adam_table(tensors, n_tensors, lr, beta1, beta2, eps, state, tab, &blocks, &past)) return r;
    NVDR_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_len >= 2, "adam_step: a 16-byte aligned workspace is needed");
    AdamStep *begin = (AdamStep *)workspace;
    const AdamBegin adam = {state, lr, beta1, beta2, begin};
    if (int r = nvdr_adam_norm(tensors, n_tensors, norm_type, max_norm, workspace + 2, workspace_len - 2, norm, adam, (hipStream_t)stream_)) return r;
    adam_launch(tab, blocks, past, lr, beta1, beta2, eps, state, nullptr, begin, (hipStream_t)stream_);
    NVDR_LAUNCH_CHECK();
    return 0;
}
