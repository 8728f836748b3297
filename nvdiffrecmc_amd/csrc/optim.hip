// optim.hip -- the parameter update of one training iteration as ONE launch.
//
// Replaces, for the three tensors the direct-lighting iteration trains (kd texture, ks, light probe), the sequence
//     lgt.base.grad *= 64                      train.py:439-440
//     optimizer.step()                         train.py:452-461  (torch.optim.Adam, no weight decay, no amsgrad)
//     clamps of the parameters                 train.py:470-476 / material clamps
// which on ROCm is a multi-tensor Adam launch that puts ~1 M elements on 16 workgroups (45 us on a 256-CU part) plus five
// small elementwise kernels.  One thread per element over all tensors, the step counter in device memory (the launch can be
// captured in a HIP graph and replayed), same arithmetic and the same order of operations as torch's single-tensor Adam:
//     m = m + (g - m) * (1 - b1);  v = v * b2 + (1 - b2) * g * g
//     p = p - (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps);  p = max(min(p, hi), lo)
#include "common.h"
#include "gradnorm.h"
#include "nvdr_hip.h"

#define ADAM_TILE 64             // texels of a tile of the sparse-texture path
#define ADAM_BLOCK 256
#define ADAM_ROUNDS 2            // groups of four elements that a thread of the plain path takes, all their loads in flight
struct AdamTable {
    nvdr_adam_tensor t[NVDR_ADAM_MAX_TENSORS];
    int first_block[NVDR_ADAM_MAX_TENSORS + 1];     // workgroups [first_block[k], first_block[k + 1]) work on tensor k
    int n;
};
static_assert(NVDR_ADAM_MAX_TENSORS <= 32, "the kernel compares first_block one by one");

// N elements from e on; behind the end of the tensor zeros are loaded and nothing is stored.  `wide`: the buffer is 16-byte aligned (e is a
// multiple of four); one that is not -- a gradient inside an exchange bucket -- goes element by element
template <int N>
__device__ __forceinline__ void adam_load(float (&x)[N], const float *p, int64_t e, int64_t n, bool wide)
{
    if (wide && e + N <= n) {
#pragma unroll
        for (int c = 0; c < N; c += 4) {
            const float4 v = *(const float4 *)(p + e + c);
            x[c] = v.x; x[c + 1] = v.y; x[c + 2] = v.z; x[c + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) x[c] = e + c < n ? p[e + c] : 0.0f;
    }
}

template <int N>
__device__ __forceinline__ void adam_store(const float (&x)[N], float *p, int64_t e, int64_t n, bool wide)
{
    if (wide && e + N <= n) {
#pragma unroll
        for (int c = 0; c < N; c += 4) *(float4 *)(p + e + c) = make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]);
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c)
            if (e + c < n) p[e + c] = x[c];
    }
}

struct AdamConst {
    float factor, step_size, bc2_sqrt, beta2, omb1, omb2, eps;
};

// the moments and the parameter of N elements from e on
template <int N>
__device__ __forceinline__ void adam_update(const nvdr_adam_tensor &T, const AdamConst &k, int64_t e, const float (&g)[N], float (&m)[N], float (&v)[N], float (&p)[N])
{
    int64_t il = T.lo_vec ? e % T.lo_vec_n : 0, ih = T.hi_vec ? e % T.hi_vec_n : 0;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const float gg = g[c] * T.grad_scale * k.factor;
        m[c] = m[c] + (gg - m[c]) * k.omb1;                         // lerp_(grad, 1 - beta1)
        v[c] = v[c] * k.beta2 + (k.omb2 * gg) * gg;                 // mul_(beta2).addcmul_(grad, grad, value = 1 - beta2)
        const float denom = sqrtf(v[c]) / k.bc2_sqrt + k.eps;
        const float q = p[c] - k.step_size * (m[c] / denom);        // addcdiv_(exp_avg, denom, value = -step_size)
        float lo = T.lo, hi = T.hi;
        if (T.lo_vec) { lo = fmaxf(lo, T.lo_vec[il]); if (++il == T.lo_vec_n) il = 0; }
        if (T.hi_vec) { hi = fminf(hi, T.hi_vec[ih]); if (++ih == T.hi_vec_n) ih = 0; }
        p[c] = q < lo ? lo : (q > hi ? hi : q);                     // torch.clamp semantics: a NaN parameter stays NaN
    }
}

// begin: what grad_norm_final_kernel has prepared of this step (the counter has moved already); NULL: from state, with *grad_factor
__global__ void __launch_bounds__(ADAM_BLOCK) adam_step_kernel(AdamTable tab, double lr, double beta1d, double beta2d, float eps, const int *state,
                                                                const float *grad_factor, const AdamStep *begin)
{
    // state[0] = steps taken so far, state[1] unused, then two doubles: beta1^step, beta2^step (kept as running products: pow() in
    // double costs a workgroup ~10 us of latency); read-only here
    __shared__ AdamStep shared;
    if (!begin) {
        if (threadIdx.x == 0) {
            shared = adam_begin(state, lr, beta1d, beta2d);
            if (grad_factor) shared.factor = *grad_factor;
        }
        __syncthreads();
    }
    const AdamStep S = begin ? *begin : shared;
    // the tensor of this workgroup (uniform: the table entry is read with scalar loads)
    int k = 0;
    for (int q = 1; q < tab.n; ++q)
        if ((int)blockIdx.x >= tab.first_block[q]) k = q;
    const nvdr_adam_tensor &T = tab.t[k];
    const int64_t block = (int64_t)((int)blockIdx.x - tab.first_block[k]);
    // the hyper-parameters arrive as doubles, like the Python floats torch's Adam computes 1 - beta from: (float)(1 - 0.999) is
    // 0.001f, 1 - 0.999f is 1.3e-5 off (visible in the parameters after ten steps)
    // lr_scale: this tensor's learning rate (train.py:336-338: position / material / light; a zero-initialised block: the plain rate)
    const AdamConst c = {S.factor, S.step_size * (T.lr_scale == 0.0f ? 1.0f : T.lr_scale), S.bc2_sqrt, (float)beta2d, (float)(1.0 - beta1d), (float)(1.0 - beta2d), eps};
    const bool wide_g = ((uintptr_t)T.grad & 15) == 0, wide_m = ((uintptr_t)T.exp_avg & 15) == 0, wide_v = ((uintptr_t)T.exp_avg_sq & 15) == 0,
               wide_p = ((uintptr_t)T.param & 15) == 0;
    if (T.frozen && !(T.active && T.zero_grad)) return;
    if (T.active || T.normalize3) {
        // TEXELS of three channels: a lane takes four of them (twelve floats, three wide accesses a buffer), sixteen lanes a tile of 64.
        //
        // Sparse textures (T.active).  A trained texture of 1024^2 texels receives gradient only at the texels some covered pixel
        // looked up -- ~5 % of them with the fixed benchmark views -- and a texel that has never received any still has zero moments:
        // its update is p - step * 0 / (0 + eps) = p, a clamp of a value the first step already clamped.  Tiles with an all-zero
        // gradient and no history are therefore skipped after reading the gradient alone: 12 instead of 84 bytes per texel, EXACTLY
        // the same parameters (step 1 visits every tile, so that the clamps / the normalisation have been applied to whatever the
        // initial values were).  `active[tile]` remembers history.  zero_grad: the gradient of a visited tile is zeroed behind the
        // update, so that a scatter-add backward (nvdr_texture_lookup_bwd into a persistent buffer) needs no memset of 3 x 12.6 MB per
        // iteration.
        // Normal maps (T.normalize3): every texel is renormalised after the clamps (Texture2D.clamp_ + normalize_, train.py:470-474,
        // render/texture.py:86-96).
        const int lane = threadIdx.x & 63;
        const int64_t wave = block * (ADAM_BLOCK / 64) + (threadIdx.x >> 6), e = wave * (4 * ADAM_TILE * 3) + lane * 12;
        float g[12];
        adam_load(g, T.grad, e, T.n, wide_g);
        if (T.active) {
            const int64_t tile = wave * 4 + (lane >> 4), tiles = (T.n / 3 + ADAM_TILE - 1) / ADAM_TILE;
            const bool history = tile < tiles && T.active[tile] != 0;
            bool nonzero = false;
#pragma unroll
            for (int i = 0; i < 12; ++i) nonzero |= g[i] != 0.0f;       // (a NaN is)
            const bool any = (__ballot(nonzero) >> (lane & 48) & 0xffffull) != 0;
            const float zero[12] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (T.zero_grad && any) adam_store(zero, const_cast<float *>(T.grad), e, T.n, wide_g);
            // A frozen tensor (lr_scale 0 on the host) takes no update, but its gradient is still CONSUMED: with zero_grad the producer
            // scatter-adds into a persistent buffer that nobody else clears -- and with several ranks that buffer is the exchange bucket,
            // all-reduced in place every step: left alone its content would grow by the world size per iteration until it overflows.
            if (T.frozen || (!any && !history && S.step > 1)) return;
            if (any && !history && (lane & 15) == 0 && tile < tiles) T.active[tile] = 1;
        }
        float m[12], v[12], p[12];
        adam_load(m, T.exp_avg, e, T.n, wide_m);
        adam_load(v, T.exp_avg_sq, e, T.n, wide_v);
        adam_load(p, T.param, e, T.n, wide_p);
        adam_update(T, c, e, g, m, v, p);
        if (T.normalize3) {
#pragma unroll
            for (int i = 0; i < 12; i += 3) {
                const float len = sqrtf(fmaxf((p[i] * p[i] + p[i + 1] * p[i + 1]) + p[i + 2] * p[i + 2], 1e-20f));      // util.safe_normalize
                p[i] /= len; p[i + 1] /= len; p[i + 2] /= len;
            }
        }
        adam_store(m, T.exp_avg, e, T.n, wide_m);
        adam_store(v, T.exp_avg_sq, e, T.n, wide_v);
        adam_store(p, T.param, e, T.n, wide_p);
        return;
    }
    const int64_t e0 = block * (ADAM_BLOCK * 4 * ADAM_ROUNDS) + threadIdx.x * 4;
    float g[ADAM_ROUNDS][4], m[ADAM_ROUNDS][4], v[ADAM_ROUNDS][4], p[ADAM_ROUNDS][4];
#pragma unroll
    for (int u = 0; u < ADAM_ROUNDS; ++u) {
        const int64_t e = e0 + u * (ADAM_BLOCK * 4);
        adam_load(g[u], T.grad, e, T.n, wide_g);
        adam_load(m[u], T.exp_avg, e, T.n, wide_m);
        adam_load(v[u], T.exp_avg_sq, e, T.n, wide_v);
        adam_load(p[u], T.param, e, T.n, wide_p);
    }
#pragma unroll
    for (int u = 0; u < ADAM_ROUNDS; ++u) {
        const int64_t e = e0 + u * (ADAM_BLOCK * 4);
        adam_update(T, c, e, g[u], m[u], v[u], p[u]);
        adam_store(m[u], T.exp_avg, e, T.n, wide_m);
        adam_store(v[u], T.exp_avg_sq, e, T.n, wide_v);
        adam_store(p[u], T.param, e, T.n, wide_p);
    }
}

// The step counter and the running powers move in a launch of their own (one thread, ~4 us) behind the update: every workgroup of the
// update has read them by then (stream order).  Rounds 2-3 let the workgroups of the update draw tickets on ONE word and the last
// one publish the state: up to 2 048 same-address atomics, which retire one every ~12 ns -- 25 us of a 33 us kernel.  (A clipped step of all
// tensors needs no launch for it: the kernel that finishes the norm prepares the step and moves the counter.)
__global__ void adam_advance_kernel(int *state, double beta1d, double beta2d) { adam_advance(state, beta1d, beta2d); }

// checks the tensors of a step and deals the workgroups; *blocks = how many
static int adam_table(const nvdr_adam_tensor *tensors, int n_tensors, double lr, double beta1, double beta2, double eps, const int *state, AdamTable &tab, unsigned *blocks_out)
{
    NVDR_REQUIRE(tensors && state, "adam_step: NULL argument");
    NVDR_REQUIRE(n_tensors >= 1 && n_tensors <= NVDR_ADAM_MAX_TENSORS, "adam_step: %d tensors (1..%d supported)", n_tensors, NVDR_ADAM_MAX_TENSORS);
    NVDR_REQUIRE(lr >= 0.0 && beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "adam_step: bad hyper-parameters");
    memset(&tab, 0, sizeof(tab));
    tab.n = n_tensors;
    int64_t total = 0;
    for (int k = 0; k < n_tensors; ++k) {
        const nvdr_adam_tensor &t = tensors[k];
        NVDR_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq && t.n >= 0, "adam_step: tensor %d has a NULL buffer", k);
        NVDR_REQUIRE(!t.lo_vec || t.lo_vec_n > 0, "adam_step: tensor %d: lo_vec without length", k);
        NVDR_REQUIRE(!t.hi_vec || t.hi_vec_n > 0, "adam_step: tensor %d: hi_vec without length", k);
        NVDR_REQUIRE(!t.normalize3 || t.n % 3 == 0, "adam_step: tensor %d: normalize3 needs a multiple of three elements", k);
        NVDR_REQUIRE(t.lr_scale >= 0.0f, "adam_step: tensor %d: negative lr_scale (0 = the plain rate; `frozen` freezes)", k);
        NVDR_REQUIRE(!t.active || t.n % 3 == 0, "adam_step: tensor %d: the sparse path works on texels of three channels", k);
        NVDR_REQUIRE(!t.zero_grad || t.active, "adam_step: tensor %d: zero_grad needs the sparse path (active)", k);
        tab.t[k] = t;
        total += t.n;
    }
    NVDR_REQUIRE(total < (1ll << 40), "adam_step: too many elements");
    int64_t blocks = 0;
    for (int k = 0; k < n_tensors; ++k) {
        tab.first_block[k] = (int)blocks;
        blocks += tensors[k].active || tensors[k].normalize3 ? div_up(tensors[k].n, ADAM_BLOCK * 12) : div_up(tensors[k].n, ADAM_BLOCK * 4 * ADAM_ROUNDS);
    }
    for (int k = n_tensors; k <= NVDR_ADAM_MAX_TENSORS; ++k) tab.first_block[k] = (int)blocks;
    *blocks_out = (unsigned)(blocks < 1 ? 1 : blocks);
    return 0;
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
    if (int r = adam_table(tensors, n_tensors, lr, beta1, beta2, eps, state, tab, &blocks)) return r;
    adam_step_kernel<<<blocks, ADAM_BLOCK, 0, (hipStream_t)stream_>>>(tab, lr, beta1, beta2, (float)eps, state, grad_factor, nullptr);
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
    if (int r = adam_table(tensors, n_tensors, lr, beta1, beta2, eps, state, tab, &blocks)) return r;
    NVDR_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0 && workspace_len >= 2, "adam_step: a 16-byte aligned workspace is needed");
    AdamStep *begin = (AdamStep *)workspace;
    const AdamBegin adam = {state, lr, beta1, beta2, begin};
    if (int r = nvdr_adam_norm(tensors, n_tensors, norm_type, max_norm, workspace + 2, workspace_len - 2, norm, adam, (hipStream_t)stream_)) return r;
    adam_step_kernel<<<blocks, ADAM_BLOCK, 0, (hipStream_t)stream_>>>(tab, lr, beta1, beta2, (float)eps, state, nullptr, begin);
    NVDR_LAUNCH_CHECK();
    return 0;
}
