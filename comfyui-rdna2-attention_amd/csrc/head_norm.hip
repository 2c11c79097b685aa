// Norms of query and key heads with their turn by position in the same pass, and the gradients.
//
// A head x of D values becomes y = R(n) (w * x r), r = (mean of x^2 + eps)^-1/2, w the tensor's weights (one of D values for all query heads, one for
// all key heads), R(n) the turn of rotary.h by the token's position n. All of it is done in 32 bits, rounded once.
//
// Backward, with g the gradient of y, turned back (R is orthogonal up to its factor, so that R^T g is the turn by -n times the same factor), and
// u = x r: the gradient of x is r (w g - u mean(w g u)), that of w the sum of g u over all tokens and heads.
//
// Both passes move each value once, as rotate does, and are laid out like it (rotary.hip): a wave takes a token and a slice of one tensor's heads, its lanes
// make the token's angles once, a head's sum crosses the D / 16 lanes that hold it. The weights' gradient stays in a lane's registers over all of the
// tokens that its wave takes; workgroups leave their sums of it in a workspace, which a second launch adds up in a fixed order.
//
// 8192 tokens of 32 + 8 heads of 128 bf16: forward 36 us (168 MB, 4.7 TB/s), backward 45 (252 MB, 5.6 TB/s) and 4 for the weights' sums. One token: 4.3 us, a launch's and three
// accesses' latency.
#include "rotary.h"

#define BACK_PASSES 2  // heads per lane and token of the backward pass: two hold a head's values and its gradient's

struct NormArgs {
    RotaryArgs r;
    const void *x[2], *g[2];  // queries and keys; their outputs' gradients
    void* y[2];               // the outputs, contiguous (the inputs' gradients)
    const void* w[2];
    void* gw[2];
    float* ws;
    const void* positions;
    int wide, wtype;
    float eps;
    int L, H[2], slices;  // heads; slices of the query heads
    long tokens, sx[2][3], sg[2][3];
};

template <class X>
__global__ __launch_bounds__(ROW_WAVES * 64) void norm_rotate_kernel(NormArgs p) {
    __shared__ __attribute__((aligned(16))) f2 cs_all[ROW_WAVES][MAX_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long token = (long)blockIdx.x * ROW_WAVES + wave;
    if (token >= p.tokens) return;
    f2* cs = cs_all[wave];
    const Place pl = place(p.r, lane);
    const int which = (int)blockIdx.y >= p.slices, per = p.r.D / 16;
    const long b = token / p.L, l = token % p.L;
    const double n = p.wide ? (double)((const long*)p.positions)[token] : (double)((const int*)p.positions)[token];
    const int pairs = p.r.R / 2;
    const double f0 = p.r.turns[min(lane, pairs - 1)], f1 = p.r.turns[min(lane + 64, pairs - 1)];
    const X* x = (const X*)p.x[which] + b * p.sx[which][0] + l * p.sx[which][1];
    X* y = (X*)p.y[which] + token * p.H[which] * p.r.D;
    const int first = ((int)blockIdx.y - (which ? p.slices : 0)) * pl.heads * PASSES + pl.head, end = pl.head < pl.heads ? p.H[which] : 0;
    f8 lo[PASSES], hi[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = first + i * pl.heads;
        const X* src = x + (long)(h < end ? h : 0) * p.sx[which][2];
        lo[i] = load8(src + pl.at);
        hi[i] = load8(src + pl.to);
    }
    const f8 wl = weights8(p.w[which], p.wtype, pl.at), wh = weights8(p.w[which], p.wtype, pl.to);
    make_angles(p.r, f0, f1, n, cs, lane);
    f8 c, s;
    angles_of(pl, cs, c, s);
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int h = first + i * pl.heads;
        const float inv = inverse_rms(lo[i], hi[i], p.r.D, p.eps, per, lane);
        lo[i] = lo[i] * inv * wl;
        hi[i] = hi[i] * inv * wh;
        if (pl.pair >= 0) turn(lo[i], hi[i], c, s, p.r.interleaved);
        if (h < end) {
            store8(y + (long)h * p.r.D + pl.at, lo[i]);
            store8(y + (long)h * p.r.D + pl.to, hi[i]);
        }
    }
}

// Workgroup (x, y) takes the tokens 4 x + wave, 4 (x + grid) + wave and so on, of slice y's heads.
template <class X>
__global__ __launch_bounds__(ROW_WAVES * 64) void norm_rotate_back_kernel(NormArgs p) {
    __shared__ __attribute__((aligned(16))) f2 cs_all[ROW_WAVES][MAX_PAIRS];
    __shared__ float sums[ROW_WAVES * 64][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    f2* cs = cs_all[wave];
    const Place pl = place(p.r, lane);
    const int which = (int)blockIdx.y >= p.slices, per = p.r.D / 16, pairs = p.r.R / 2;
    const double f0 = p.r.turns[min(lane, pairs - 1)], f1 = p.r.turns[min(lane + 64, pairs - 1)];
    const f8 wl = weights8(p.w[which], p.wtype, pl.at), wh = weights8(p.w[which], p.wtype, pl.to);
    const int first = ((int)blockIdx.y - (which ? p.slices : 0)) * pl.heads * BACK_PASSES + pl.head, end = pl.head < pl.heads ? p.H[which] : 0;
    f8 dl = {}, dh = {};
    for (long token = (long)blockIdx.x * ROW_WAVES + wave; token < p.tokens; token += (long)gridDim.x * ROW_WAVES) {
        const long b = token / p.L, l = token % p.L;
        const double n = p.wide ? (double)((const long*)p.positions)[token] : (double)((const int*)p.positions)[token];
        const X* x = (const X*)p.x[which] + b * p.sx[which][0] + l * p.sx[which][1];
        const X* g = (const X*)p.g[which] + b * p.sg[which][0] + l * p.sg[which][1];
        X* y = (X*)p.y[which] + token * p.H[which] * p.r.D;
        f8 xl[BACK_PASSES], xh[BACK_PASSES], gl[BACK_PASSES], gh[BACK_PASSES];
#pragma unroll
        for (int i = 0; i < BACK_PASSES; i++) {
            const int h = first + i * pl.heads;
            const X *src = x + (long)(h < end ? h : 0) * p.sx[which][2], *grad = g + (long)(h < end ? h : 0) * p.sg[which][2];
            xl[i] = load8(src + pl.at);
            xh[i] = load8(src + pl.to);
            gl[i] = load8(grad + pl.at);
            gh[i] = load8(grad + pl.to);
        }
        make_angles(p.r, f0, f1, n, cs, lane);
        f8 c, s;
        angles_of(pl, cs, c, s);
#pragma unroll
        for (int i = 0; i < BACK_PASSES; i++) {
            const int h = first + i * pl.heads;
            const float inv = inverse_rms(xl[i], xh[i], p.r.D, p.eps, per, lane);
            if (pl.pair >= 0) turn(gl[i], gh[i], c, s, p.r.interleaved);
            const f8 ul = xl[i] * inv, uh = xh[i] * inv;
            if (h < end) {
                dl += gl[i] * ul;
                dh += gh[i] * uh;
            }
            gl[i] *= wl;
            gh[i] *= wh;
            const float mean = head_sum(dot16(gl[i], ul, gh[i], uh), per, lane) * (1.f / (float)p.r.D);
            if (h < end) {
                store8(y + (long)h * p.r.D + pl.at, (gl[i] - ul * mean) * inv);
                store8(y + (long)h * p.r.D + pl.to, (gh[i] - uh * mean) * inv);
            }
        }
        __builtin_amdgcn_wave_barrier();  // the next token's angles go where these were
    }
    // The workgroup's sums: thread d adds value d of every lane that holds one.
#pragma unroll
    for (int e = 0; e < 8; e++) {
        sums[threadIdx.x][e] = dl[e];
        sums[threadIdx.x][8 + e] = dh[e];
    }
    __syncthreads();
    const int d = threadIdx.x, half = p.r.R / 2;
    if (d < p.r.D) {
        const bool split = !p.r.interleaved && d < p.r.R;
        const int u = split ? d % half / 8 : d / 16, e = split ? d / half * 8 + d % 8 : d % 16;
        float sum = 0.f;
        for (int w = 0; w < ROW_WAVES; w++)
            for (int i = 0; i < pl.heads; i++) sum += sums[w * 64 + i * per + u][e];
        p.ws[((long)blockIdx.y * gridDim.x + blockIdx.x) * p.r.D + d] = sum;
    }
}

// Adds up the workgroups' sums: workgroup (x, t) values 16 x .. 16 x + 15 of tensor t's weights, 64 rows at a time.
__global__ __launch_bounds__(1024) void norm_weights_kernel(NormArgs p, int grid, int slices) {
    __shared__ float sums[64][17];
    const int t = blockIdx.y, c = threadIdx.x & 15, r = threadIdx.x >> 4, d = blockIdx.x * 16 + c;
    const int from = t ? p.slices * grid : 0, to = t ? slices * grid : p.slices * grid;
    float sum = 0.f;
#pragma unroll 4
    for (int i = from + r; i < to; i += 64) sum += p.ws[(long)i * p.r.D + d];
    sums[r][c] = sum;
    __syncthreads();
    for (int n = 32; n; n >>= 1) {
        if (r < n) sums[r][c] += sums[r + n][c];
        __syncthreads();
    }
    if (r == 0) {
        if (p.wtype == RDA_FP16) ((half_t*)p.gw[t])[d] = (half_t)sums[0][c];
        else if (p.wtype == RDA_BF16) ((bf16_t*)p.gw[t])[d] = (bf16_t)sums[0][c];
        else ((float*)p.gw[t])[d] = sums[0][c];
    }
}

#define BACK_GRID 768  // workgroups of the backward pass at most: three on each of 256 CUs

// B, L, H, Hkv, D, R of dims; slices of a tensor's heads.
static bool norm_sizes_ok(const double* turns, const long* dims, int type, int wtype) {
    const long B = dims[0], L = dims[1], H = dims[2], Hkv = dims[3];
    if (B <= 0 || L <= 0 || H <= 0 || H > 65535 || Hkv <= 0 || Hkv > 65535 || !rotary_ok(turns, dims[4], dims[5]) || dims[5] == 0) return false;
    return B <= MAX_ROWS && L <= MAX_ROWS && B * L <= MAX_ROWS && type >= RDA_FP16 && type <= RDA_FP32 && wtype >= RDA_FP16 && wtype <= RDA_FP32;
}
static int norm_slices(long H, long D, int passes) { return (int)((H + 64 / (D / 16) * passes - 1) / (64 / (D / 16) * passes)); }
static NormArgs norm_args(const void* q, const void* k, void* q_out, void* k_out, const void* positions, int wide, const void* qw, const void* kw, int wtype, float eps,
                          const double* turns, float factor, float sign, int interleaved, const long* dims) {
    NormArgs a = {};
    a.r = {turns, (int)dims[4], (int)dims[5], interleaved & 1, factor, sign};
    a.x[0] = q; a.x[1] = k; a.y[0] = q_out; a.y[1] = k_out; a.w[0] = qw; a.w[1] = kw;
    a.positions = positions; a.wide = wide; a.wtype = wtype; a.eps = eps;
    a.L = (int)dims[1]; a.H[0] = (int)dims[2]; a.H[1] = (int)dims[3]; a.tokens = dims[0] * dims[1];
    for (int i = 0; i < 6; i++) a.sx[i / 3][i % 3] = dims[6 + i];
    return a;
}
static long back_grid(long tokens, long slices) {
    const long most = (BACK_GRID + slices - 1) / slices, all = (tokens + ROW_WAVES - 1) / ROW_WAVES;
    return all < most ? all : most;
}

extern "C" {

int rda_norm_rotate(const void* q, const void* k, void* q_out, void* k_out, const void* positions, int wide, const void* q_weight, const void* k_weight,
                    int weight_type, float eps, const double* turns, float factor, int interleaved, int type, const long* dims, void* stream) {
    if (!norm_sizes_ok(turns, dims, type, weight_type) || !vector_rows(q, dims + 6, 3, type) || !vector_rows(k, dims + 9, 3, type) || !vector_rows(q_out, dims, 0, type) ||
        !vector_rows(k_out, dims, 0, type) || !vector_rows(q_weight, dims, 0, type) || !vector_rows(k_weight, dims, 0, type))
        return RDA_ERR_INVALID;
    NormArgs a = norm_args(q, k, q_out, k_out, positions, wide, q_weight, k_weight, weight_type, eps, turns, factor, 1.f, interleaved, dims);
    a.slices = norm_slices(dims[2], dims[4], PASSES);
    const dim3 grid((unsigned)((a.tokens + ROW_WAVES - 1) / ROW_WAVES), (unsigned)(a.slices + norm_slices(dims[3], dims[4], PASSES)));
    const auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(ROW_WAVES * 64), 0, (hipStream_t)stream, a);
        return (int)hipGetLastError();
    };
    return type == RDA_FP16 ? launch(norm_rotate_kernel<half_t>) : type == RDA_BF16 ? launch(norm_rotate_kernel<bf16_t>) : launch(norm_rotate_kernel<float>);
}

size_t rda_norm_rotate_back_workspace(long tokens, long H, long Hkv, long D) {
    if (tokens <= 0 || tokens > MAX_ROWS || H <= 0 || H > 65535 || Hkv <= 0 || Hkv > 65535 || D <= 0 || D % 16 || D > 2 * MAX_PAIRS) return 0;
    const long slices = norm_slices(H, D, BACK_PASSES) + norm_slices(Hkv, D, BACK_PASSES);
    return (size_t)(back_grid(tokens, slices) * slices * D) * 4;
}

int rda_norm_rotate_back(const void* q, const void* k, const void* q_grad, const void* k_grad, void* q_out, void* k_out, void* q_weight_out, void* k_weight_out,
                         const void* positions, int wide, const void* q_weight, const void* k_weight, int weight_type, float eps, const double* turns, float factor,
                         int interleaved, void* workspace, int type, const long* dims, void* stream) {
    if (!norm_sizes_ok(turns, dims, type, weight_type) || !vector_rows(q, dims + 6, 3, type) || !vector_rows(k, dims + 9, 3, type) ||
        !vector_rows(q_grad, dims + 12, 3, type) || !vector_rows(k_grad, dims + 15, 3, type) || !vector_rows(q_out, dims, 0, type) || !vector_rows(k_out, dims, 0, type) ||
        !vector_rows(q_weight, dims, 0, type) || !vector_rows(k_weight, dims, 0, type))
        return RDA_ERR_INVALID;
    NormArgs a = norm_args(q, k, q_out, k_out, positions, wide, q_weight, k_weight, weight_type, eps, turns, factor, -1.f, interleaved, dims);
    a.g[0] = q_grad; a.g[1] = k_grad; a.gw[0] = q_weight_out; a.gw[1] = k_weight_out; a.ws = (float*)workspace;
    for (int i = 0; i < 6; i++) a.sg[i / 3][i % 3] = dims[12 + i];
    a.slices = norm_slices(dims[2], dims[4], BACK_PASSES);
    const int slices = a.slices + norm_slices(dims[3], dims[4], BACK_PASSES), grid = (int)back_grid(a.tokens, slices);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid, slices), dim3(ROW_WAVES * 64), 0, (hipStream_t)stream, a); };
    type == RDA_FP16 ? launch(norm_rotate_back_kernel<half_t>) : type == RDA_BF16 ? launch(norm_rotate_back_kernel<bf16_t>) : launch(norm_rotate_back_kernel<float>);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL(norm_weights_kernel, dim3((unsigned)(dims[4] / 16), 2), dim3(1024), 0, (hipStream_t)stream, a, grid, slices);
    return (int)hipGetLastError();
}

}  // extern "C"
