// Short causal depthwise convolution: y_t[d] = act(bias[d] + sum_k w[d][k] x_{t-K+1+k}[d]), its backward pass and its
// form for one more token on a pool of states (tgru_conv_* of include/tgru.h).
//
// Bound: HBM.  A tap costs one FMA per element against two to four bytes read and written, so what counts is that
// every row is fetched once, 16 bytes a lane, with enough loads in flight.  A thread owns VEC neighbouring channels
// (16 bytes of them) and a RUN of consecutive steps, which it walks with the last K - 1 rows in registers, eight rows
// requested together; only the K - 1 rows in front of a run are read twice (out of the cache: the run before has them).
// Lanes run over channels first, so a wave's loads are consecutive.
#include "ssm_common.h"
#include <algorithm>
#include <type_traits>

namespace tgru {
namespace ssm {

constexpr int kConvThreads = 256;
constexpr int kRows = 8, kRowsBack = 2;      // rows requested together

// Neighbouring channels of a row, loaded and stored by one instruction wherever they start (the chip takes wide accesses at
// any element's alignment).
template <typename X, int VEC>
struct alignas(sizeof(X)) Pack { X v[VEC]; };

template <typename X, int VEC>
__device__ __forceinline__ Pack<X, VEC> load_pack(const void *base, long elem) {
    return *reinterpret_cast<const Pack<X, VEC> *>(static_cast<const X *>(base) + elem);
}
template <typename X, int VEC>
__device__ __forceinline__ void store_pack(void *base, long elem, const float (&v)[VEC]) {
    Pack<X, VEC> p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.v[i] = from_float<X>(v[i]);
    *reinterpret_cast<Pack<X, VEC> *>(static_cast<X *>(base) + elem) = p;
}

// Where a thread stands: channels [d, d + VEC) of sequence b, steps [t0, t1) of its n, run number `row` of all runs.  The
// last pack of a row ends with the row: where VEC does not divide D, it and the pack before it both compute, and write,
// what they share.
struct Place { int b, d, t0, t1, n, run; long row; bool live; };

template <int VEC>
__device__ __forceinline__ Place place_of(const tgru_conv_args &a, int nvec, int runs, int run_len) {
    Place p;
    const unsigned id = blockIdx.x * kConvThreads + threadIdx.x;
    const unsigned r = id / (unsigned)nvec;
    p.live = r < (unsigned)a.B * (unsigned)runs;
    p.d = min((int)(id - r * (unsigned)nvec) * VEC, a.D - VEC);
    p.b = (int)(r / (unsigned)runs);
    p.run = (int)(r - (unsigned)p.b * (unsigned)runs);
    p.row = r;
    p.t0 = p.run * run_len;
    p.t1 = min(a.T, p.t0 + run_len);
    p.n = p.live ? clamped_length(a.lengths, p.b, a.T) : 0;
    return p;
}

// Row `t` of the input as the convolution sees it: t >= 0 from x (the caller knows that the sequence has it), t < 0
// from the initial state, zero where there is none.
template <typename X, int K, int VEC>
__device__ __forceinline__ void input_row(const tgru_conv_args &a, const Place &p, int t, float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = 0.f;
    if (t < 0 && !a.initial_state) return;
    const Pack<X, VEC> r = t >= 0 ? load_pack<X, VEC>(a.x, p.b * a.x_stride[0] + t * a.x_stride[1] + p.d)
                                  : load_pack<X, VEC>(a.initial_state, ((long)p.b * (K - 1) + t + K - 1) * a.D + p.d);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_float(r.v[i]);
}

// The taps of VEC channels lie next to each other.
template <int K, int VEC>
__device__ __forceinline__ void load_taps(const float *weight, const float *bias, int d, float (&w)[K][VEC], float (&b)[VEC]) {
    float flat[K * VEC];
    const float *from = weight + (long)d * K;
    if constexpr (VEC >= 4) {
#pragma unroll
        for (int j = 0; j < K * VEC / 4; ++j) {
            const Pack<float, 4> four = reinterpret_cast<const Pack<float, 4> *>(from)[j];
#pragma unroll
            for (int i = 0; i < 4; ++i) flat[4 * j + i] = four.v[i];
        }
    } else {
#pragma unroll
        for (int j = 0; j < K * VEC; ++j) flat[j] = from[j];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        b[i] = bias ? bias[d + i] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = flat[i * K + k];
    }
}

template <typename X, int K, int VEC>
__global__ __launch_bounds__(kConvThreads) void conv_fwd_kernel(tgru_conv_args a, int nvec, int runs, int run_len) {
    const Place p = place_of<VEC>(a, nvec, runs, run_len);
    if (!p.live) return;
    float w[K][VEC], bias[VEC], win[K - 1 + kRows][VEC];
    load_taps<K, VEC>(a.weight, a.bias, p.d, w, bias);
    const int tv = min(p.t1, p.n);
    const long xo = p.b * a.x_stride[0] + p.d, yo = p.b * a.y_stride[0] + p.d;
    if (p.t0 < tv) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) input_row<X, K, VEC>(a, p, p.t0 - (K - 1) + k, win[k]);
    }
    for (int t = p.t0; t < tv; t += kRows) {
        Pack<X, VEC> raw[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) raw[r] = load_pack<X, VEC>(a.x, xo + (long)min(t + r, tv - 1) * a.x_stride[1]);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int i = 0; i < VEC; ++i) win[K - 1 + r][i] = to_float(raw[r].v[i]);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float y[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float s = bias[i];
#pragma unroll
                for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][i], win[r + k][i], s);
                y[i] = a.silu ? s * sigmoid(s) : s;
            }
            if (t + r < tv) store_pack<X, VEC>(a.y, yo + (long)(t + r) * a.y_stride[1], y);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int i = 0; i < VEC; ++i) win[k][i] = win[kRows + k][i];
    }
    const float zero[VEC] = {};
    for (int t = max(p.t0, p.n); t < p.t1; ++t) store_pack<X, VEC>(a.y, yo + (long)t * a.y_stride[1], zero);
    if (a.final_state && p.run == runs - 1) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float v[VEC];
            input_row<X, K, VEC>(a, p, p.n + j - (K - 1), v);
            store_pack<X, VEC>(a.final_state, ((long)p.b * (K - 1) + j) * a.D + p.d, v);
        }
    }
}

// Backward: the pre-activation is formed again from x, dpre_t = dy_t act'(pre_t), and then
//     dx_s = sum_k w[k] dpre_{s+K-1-k},   dw[k] = sum_t dpre_t x_{t-K+1+k},   dbias = sum_t dpre_t.
// A run looks K - 1 steps past its end (dx there needs them; they count towards dw in the run that owns them).  The
// sums over a run's steps stay in registers; every run leaves one row (K + 1, D) of them, which a second kernel adds
// up in a fixed order.  Registers decide here (taps, two windows and the sums are 140 floats a lane): two rows at a time
// and the next two on their way took 95 us where, in the same run, four rows without that took 107 and eight 150.
template <typename X, int K, int VEC>
__global__ __launch_bounds__(kConvThreads) void conv_bwd_kernel(tgru_conv_args a, int nvec, int runs, int run_len) {
    const Place p = place_of<VEC>(a, nvec, runs, run_len);
    if (!p.live) return;
    float w[K][VEC], bias[VEC], win[K][VEC], dpre[K][VEC], dw[K][VEC], db[VEC];
    load_taps<K, VEC>(a.weight, a.bias, p.d, w, bias);
    const int te = min(p.n, p.t1 + K - 1);      // steps looked at: [t0, te)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) win[k][i] = dpre[k][i] = dw[k][i] = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) db[i] = 0.f;
    if (p.t0 < te) {
#pragma unroll
        for (int k = 1; k < K; ++k) input_row<X, K, VEC>(a, p, p.t0 - K + k, win[k]);
    }
    const long xo = p.b * a.x_stride[0] + p.d, go = p.b * a.dy_stride[0] + p.d, dxo = p.b * a.dx_stride[0] + p.d;
    Pack<X, VEC> nx[kRowsBack], ng[kRowsBack];      // the next rows, requested while these are worked on
    auto request = [&](int t) {
        if (t >= te) return;
#pragma unroll
        for (int r = 0; r < kRowsBack; ++r) nx[r] = load_pack<X, VEC>(a.x, xo + (long)min(t + r, te - 1) * a.x_stride[1]);
        if (a.dy) {
#pragma unroll
            for (int r = 0; r < kRowsBack; ++r) ng[r] = load_pack<X, VEC>(a.dy, go + (long)min(t + r, te - 1) * a.dy_stride[1]);
        }
    };
#pragma unroll
    for (int r = 0; r < kRowsBack; ++r)
#pragma unroll
        for (int i = 0; i < VEC; ++i) nx[r].v[i] = ng[r].v[i] = from_float<X>(0.f);
    request(p.t0);
    for (int t = p.t0; t < p.t1 + K - 1; t += kRowsBack) {
        Pack<X, VEC> rx[kRowsBack], rg[kRowsBack];
#pragma unroll
        for (int r = 0; r < kRowsBack; ++r) { rx[r] = nx[r]; rg[r] = ng[r]; }
        request(t + kRowsBack);
        // Rows that are this run's own, are there, and whose dx is this run's own too need no selection.
        auto rows = [&](auto inside) {
#pragma unroll
            for (int r = 0; r < kRowsBack; ++r) {
                const int now = t + r, s = now - (K - 1);
                const bool on = inside.value || now < te, mine = inside.value || (on && now < p.t1);
                float dx[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) { win[k][i] = win[k + 1][i]; dpre[k][i] = dpre[k + 1][i]; }
                    win[K - 1][i] = to_float(rx[r].v[i]);
                    float pre = bias[i], d = to_float(rg[r].v[i]);
#pragma unroll
                    for (int k = 0; k < K; ++k) pre = __builtin_fmaf(w[k][i], win[k][i], pre);
                    if (a.silu) {
                        const float sg = sigmoid(pre);
                        d *= sg * __builtin_fmaf(pre, 1.f - sg, 1.f);
                    }
                    d = on ? d : 0.f;
                    dpre[K - 1][i] = d;
                    if (mine) {
                        db[i] += d;
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][i] = __builtin_fmaf(d, win[k][i], dw[k][i]);
                    }
                    float v = w[K - 1][i] * dpre[0][i];      // dpre[j] is that of step s + j: tap K - 1 - j
#pragma unroll
                    for (int k = 1; k < K; ++k) v = __builtin_fmaf(w[K - 1 - k][i], dpre[k][i], v);
                    dx[i] = v;
                }
                if (inside.value) {
                    if (a.dx) store_pack<X, VEC>(a.dx, dxo + (long)s * a.dx_stride[1], dx);
                    continue;
                }
                const bool in_run = s >= p.t0 && s < p.t1, before = s < 0 && p.run == 0 && now < p.t1 + K - 1;
                if (!in_run && !before) continue;
                const int j = s - p.n + K - 1;      // row of the final state that x_s is
                if (a.dfinal && j >= 0 && j < K - 1) {
                    const Pack<X, VEC> f = load_pack<X, VEC>(a.dfinal, ((long)p.b * (K - 1) + j) * a.D + p.d);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) dx[i] += to_float(f.v[i]);
                }
                if (in_run) {
                    if (a.dx) store_pack<X, VEC>(a.dx, dxo + (long)s * a.dx_stride[1], dx);
                } else if (a.dinitial) {
                    store_pack<X, VEC>(a.dinitial, ((long)p.b * (K - 1) + s + K - 1) * a.D + p.d, dx);
                }
            }
        };
        if (t >= p.t0 + K - 1 && t + kRowsBack <= min(te, p.t1)) rows(std::true_type{});
        else rows(std::false_type{});
    }
    if (!a.dweight && !a.dbias) return;
    float *part = a.workspace + p.row * (long)(K + 1) * a.D + p.d;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[(long)k * a.D + i] = dw[k][i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[(long)K * a.D + i] = db[i];
}

// Sums of the rows part[rows][K + 1][D]: 32 columns x 32 groups of rows per workgroup, a group adds a contiguous range, the
// groups are joined in order.  FOLD: workgroup row y of the launch leaves the sums of rows [y, y + 1) * fold in row y of
// `folded`; otherwise they are dweight (D, K) and dbias (D).  Many rows of few columns are folded first, because a column
// block is one workgroup: 16384 rows of 240 columns take 9.5 us, 36 in one launch.
constexpr int kFold = 512, kMaxFolds = 4096;
template <bool FOLD>
__global__ __launch_bounds__(1024) void conv_param_grad_kernel(const float *__restrict__ part, int rows, int D, int K, float *dweight, float *dbias,
                                                               float *folded, int fold) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const long cols = (long)(K + 1) * D, col = (long)blockIdx.x * 32 + c;
    const int first = FOLD ? (int)blockIdx.y * fold : 0, end = FOLD ? min(rows - first, fold) + first : rows;
    const int per = (end - first + 31) / 32, r0 = min(end, first + grp * per), r1 = min(end, r0 + per);
    red[grp][c] = col < cols ? sum_rows(part + col, cols, r0, r1) : 0.f;
    __syncthreads();
    if (grp != 0 || col >= cols) return;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) v += red[q][c];
    if (FOLD) {
        folded[blockIdx.y * cols + col] = v;
        return;
    }
    const int k = (int)(col / D), d = (int)(col - (long)k * D);
    if (k == K) { if (dbias) dbias[d] = v; }
    else if (dweight) dweight[(long)d * K + k] = v;
}

// One token: a wave takes 64 VEC channels of one row (256 rows of 4096 channels in 16 bits: 7 us; one row of 1024: 2.2 us,
// a chain of two or three loads).  Of the rows with one slot the first takes them all, in order,
// with the state in registers between them; the others' waves find that they are not the first and leave.
template <typename X, int K, int VEC>
__global__ __launch_bounds__(64) void conv_step_kernel(tgru_conv_step_args a, int nvec, int nblk) {
    const int row0 = blockIdx.x / nblk;
    const int cv = (blockIdx.x - row0 * nblk) * 64 + (int)threadIdx.x;
    const bool on = cv < nvec;
    const int d = (on ? cv : 0) * VEC;
    const int my_slot = a.slots ? a.slots[row0] : row0;
    __builtin_amdgcn_sched_barrier(0);       // what does not depend on the slot is requested behind the slot's own load
    float w[K][VEC], bias[VEC], win[K][VEC];
    load_taps<K, VEC>(a.weight, a.bias, d, w, bias);
    Pack<X, VEC> x = load_pack<X, VEC>(a.x, row0 * a.x_stride + d);
    __builtin_amdgcn_sched_barrier(0);
    const int slot = __builtin_amdgcn_readfirstlane(my_slot);
    if (slot < 0 || slot >= a.P) {
        const float zero[VEC] = {};
        if (on) store_pack<X, VEC>(a.y, row0 * a.y_stride + d, zero);
        return;
    }
    const long so = (long)slot * (K - 1) * a.D + d;
    Pack<X, VEC> st[K > 1 ? K - 1 : 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) st[k] = load_pack<X, VEC>(a.state, so + (long)k * a.D);
    __builtin_amdgcn_sched_barrier(0);       // on its way while the search waits for its own loads
    if (a.slots && find_slot(a.slots, 0, row0, slot) < row0) return;
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < VEC; ++i) win[k][i] = to_float(st[k].v[i]);
    for (int row = row0;;) {
        float y[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            win[K - 1][i] = to_float(x.v[i]);
            float s = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) s = __builtin_fmaf(w[k][i], win[k][i], s);
            y[i] = a.silu ? s * sigmoid(s) : s;
#pragma unroll
            for (int k = 0; k < K - 1; ++k) win[k][i] = win[k + 1][i];
        }
        if (on) store_pack<X, VEC>(a.y, row * a.y_stride + d, y);
        if (!a.slots) break;
        row = find_slot(a.slots, row + 1, a.B, slot);
        if (row >= a.B) break;
        x = load_pack<X, VEC>(a.x, row * a.x_stride + d);
    }
    if (!on) return;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store_pack<X, VEC>(a.state_out, so + (long)k * a.D, win[k]);
}

// Steps per run: as long as the launch still has about `waves` waves, because the K - 1 rows around a run are read twice; 8 at
// least (one group of loads), 64 at most.  Measured, 8 x 4096 steps of 2048 channels in 16 bits: forward 55 us with 2048
// waves (4.9 TB/s), a fifth more with 4096, half as much again with 8192; backward 106 us with 2048 (3.8 TB/s).
int conv_run_len(int B, int T, int nvec, long waves) {
    int len = 64;
    while (len > 8 && (long)B * ((T + len - 1) / len) * nvec < waves * 64) len >>= 1;
    return len;
}
constexpr long kConvWaves = 2048;

// Packs of 16 bytes wherever a row has as many channels, single elements otherwise.  (8 x 4096 steps of 2003 channels in 16 bits
// with single elements, forward 59 us, with packs 51; 64 x 256 steps of 1021: 20 and 17.)
int conv_vec(int D, int dtype) {
    const int vec = 16 / (int)dtype_bytes(dtype);
    return D >= vec ? vec : 1;
}

// Whether the rows of partial sums are folded first: more than four round trips a thread otherwise, and columns for less than
// half of the chip.  Measured, in one launch / folded: 2048 rows of 240 columns 6.2 / 7.7 us, half as many again of 960 columns 8.8 / 7.6.
bool conv_folds(long rows, long cols) { return rows > 4 * kFold && cols < 128 * 32; }
int conv_fold(long rows) { return (int)std::max<long>(kFold, (rows + kMaxFolds - 1) / kMaxFolds); }

template <typename X, int K>
int run_conv(const tgru_conv_args &a, bool backward, hipStream_t s) {
    const int vec = conv_vec(a.D, a.dtype), nvec = (a.D + vec - 1) / vec;
    const bool packs = vec > 1;
    const int len = conv_run_len(a.B, a.T, nvec, kConvWaves), runs = (a.T + len - 1) / len;
    const dim3 grid((unsigned)(((long)a.B * runs * nvec + kConvThreads - 1) / kConvThreads)), block(kConvThreads);
    constexpr int VEC = 16 / (int)sizeof(X);
    if (!backward) {
        if (packs) TGRU_LAUNCH((conv_fwd_kernel<X, K, VEC>), grid, block, 0, s, a, nvec, runs, len);
        else TGRU_LAUNCH((conv_fwd_kernel<X, K, 1>), grid, block, 0, s, a, nvec, runs, len);
        return hipGetLastError() == hipSuccess ? TGRU_OK : TGRU_E_LAUNCH;
    }
    if (packs) TGRU_LAUNCH((conv_bwd_kernel<X, K, VEC>), grid, block, 0, s, a, nvec, runs, len);
    else TGRU_LAUNCH((conv_bwd_kernel<X, K, 1>), grid, block, 0, s, a, nvec, runs, len);
    if (hipGetLastError() != hipSuccess) return TGRU_E_LAUNCH;
    if (a.dweight || a.dbias) {
        const long cols = (long)(K + 1) * a.D;
        const unsigned blocks = (unsigned)((cols + 31) / 32);
        const float *part = a.workspace;
        int rows = a.B * runs;
        if (conv_folds(rows, cols)) {
            const int fold = conv_fold(rows), folds = (int)(((long)rows + fold - 1) / fold);
            float *folded = a.workspace + rows * cols;
            TGRU_LAUNCH(conv_param_grad_kernel<true>, dim3(blocks, (unsigned)folds), dim3(1024), 0, s, part, rows, a.D, K, nullptr, nullptr, folded,
                        fold);
            if (hipGetLastError() != hipSuccess) return TGRU_E_LAUNCH;
            part = folded;
            rows = folds;
        }
        TGRU_LAUNCH(conv_param_grad_kernel<false>, dim3(blocks), dim3(1024), 0, s, part, rows, a.D, K, a.dweight, a.dbias, nullptr,
                    0);
    }
    return hipGetLastError() == hipSuccess ? TGRU_OK : TGRU_E_LAUNCH;
}

// Waves a row of the one-token form: packs where they divide D (no shared channels: the state may be updated where it lies),
// else single channels.  Measured, 256 rows in 16 bits: 4096 channels 6.4 us, 4095 10.5; 1024 and 1023 4.8 and 5.0.
int step_blocks(int D, int dtype) {
    const int vec = 16 / (int)dtype_bytes(dtype);
    return ((D % vec == 0 ? D / vec : D) + 63) / 64;
}

template <typename X, int K>
int run_conv_step(const tgru_conv_step_args &a, hipStream_t s) {
    constexpr int VEC = 16 / (int)sizeof(X);
    const bool packs = a.D % VEC == 0;
    const int nvec = packs ? a.D / VEC : a.D, nblk = step_blocks(a.D, a.dtype);
    const dim3 grid((unsigned)((long)a.B * nblk)), block(64);
    if (packs) TGRU_LAUNCH((conv_step_kernel<X, K, VEC>), grid, block, 0, s, a, nvec, nblk);
    else TGRU_LAUNCH((conv_step_kernel<X, K, 1>), grid, block, 0, s, a, nvec, nblk);
    return hipGetLastError() == hipSuccess ? TGRU_OK : TGRU_E_LAUNCH;
}

// f<X, K>() for the call's element type and number of taps
#define TGRU_CONV_DISPATCH(DTYPE, TAPS, CALL)                                                     \
    switch (TAPS) {                                                                               \
    case 1: return CALL(DTYPE, 1); case 2: return CALL(DTYPE, 2); case 3: return CALL(DTYPE, 3);  \
    case 4: return CALL(DTYPE, 4); case 5: return CALL(DTYPE, 5); case 6: return CALL(DTYPE, 6);  \
    case 7: return CALL(DTYPE, 7); default: return CALL(DTYPE, 8);                                \
    }

int dispatch_conv(const tgru_conv_args &a, bool backward, hipStream_t s) {
#define TGRU_CALL(X, K) run_conv<X, K>(a, backward, s)
    if (a.dtype == TGRU_DTYPE_F32) { TGRU_CONV_DISPATCH(float, a.K, TGRU_CALL) }
    if (a.dtype == TGRU_DTYPE_BF16) { TGRU_CONV_DISPATCH(__bf16, a.K, TGRU_CALL) }
    TGRU_CONV_DISPATCH(_Float16, a.K, TGRU_CALL)
#undef TGRU_CALL
}

int dispatch_conv_step(const tgru_conv_step_args &a, hipStream_t s) {
#define TGRU_CALL(X, K) run_conv_step<X, K>(a, s)
    if (a.dtype == TGRU_DTYPE_F32) { TGRU_CONV_DISPATCH(float, a.K, TGRU_CALL) }
    if (a.dtype == TGRU_DTYPE_BF16) { TGRU_CONV_DISPATCH(__bf16, a.K, TGRU_CALL) }
    TGRU_CONV_DISPATCH(_Float16, a.K, TGRU_CALL)
#undef TGRU_CALL
}

// A launch has a thread for every run and pack, numbered in 32 bits, and the runs (rows of partial sums) are counted in 31, with
// room for a step beyond the last.
int conv_dims(int B, int T, int D, int K, int dtype) {
    if (B <= 0 || T <= 0 || D <= 0 || K <= 0 || K > TGRU_CONV_MAX_TAPS) return TGRU_E_DIMS;
    if (T > (1 << 30) || D > INT32_MAX - kConvThreads + 1) return TGRU_E_DIMS;
    const int vec = conv_vec(D, dtype), nvec = (D + vec - 1) / vec, len = conv_run_len(B, T, nvec, kConvWaves);
    const double runs = (double)B * ((T + len - 1) / len);
    return runs <= 2147483648.0 - kConvThreads && runs * nvec < 4294967296.0 - kConvThreads ? TGRU_OK : TGRU_E_DIMS;
}

}  // namespace ssm
}  // namespace tgru

using namespace tgru::ssm;

extern "C" {

size_t tgru_conv_backward_workspace_bytes(int B, int T, int D, int K) {
    // the element type is not known here: room for the shorter runs of the two sizes of packs
    size_t rows = 0;
    for (int dtype : {TGRU_DTYPE_F32, TGRU_DTYPE_BF16}) {
        if (conv_dims(B, T, D, K, dtype) != TGRU_OK) continue;
        const int vec = conv_vec(D, dtype), len = conv_run_len(B, T, (D + vec - 1) / vec, kConvWaves);
        rows = std::max(rows, (size_t)B * ((T + len - 1) / len));
    }
    if (!rows) return 0;
    if (conv_folds((long)rows, (long)(K + 1) * D)) rows += std::min<size_t>((rows + kFold - 1) / kFold, kMaxFolds);
    return rows * (size_t)(K + 1) * D * sizeof(float);
}

int tgru_conv_forward(const tgru_conv_args *a, tgru_stream_t stream) {
    if (!a) return TGRU_E_NULL;
    if (int rc = conv_dims(a->B, a->T, a->D, a->K, a->dtype)) return rc;
    if (!known_dtype(a->dtype)) return TGRU_E_DTYPE;
    if (!a->x || !a->weight || !a->y) return TGRU_E_NULL;
    if (int rc = tgru::check_device()) return rc;
    tgru_conv_args c = *a;
    if (c.K == 1) c.initial_state = c.final_state = nullptr;
    return dispatch_conv(c, false, (hipStream_t)stream);
}

int tgru_conv_backward(const tgru_conv_args *a, tgru_stream_t stream) {
    if (!a) return TGRU_E_NULL;
    if (int rc = conv_dims(a->B, a->T, a->D, a->K, a->dtype)) return rc;
    if (!known_dtype(a->dtype)) return TGRU_E_DTYPE;
    // the parameter gradients' launch holds less than 2^32 threads, 32 a column
    if ((a->dweight || a->dbias) && (double)(a->K + 1) * a->D >= 134217696.0) return TGRU_E_DIMS;
    if (!a->x || !a->weight || ((a->dweight || a->dbias) && !a->workspace)) return TGRU_E_NULL;
    if (int rc = tgru::check_device()) return rc;
    tgru_conv_args c = *a;
    if (c.K == 1) { c.initial_state = nullptr; c.dinitial = nullptr; c.dfinal = nullptr; }
    return dispatch_conv(c, true, (hipStream_t)stream);
}

int tgru_conv_step(const tgru_conv_step_args *a, tgru_stream_t stream) {
    if (!a) return TGRU_E_NULL;
    if (a->B <= 0 || a->P <= 0 || a->D <= 0 || a->K <= 0 || a->K > TGRU_CONV_MAX_TAPS) return TGRU_E_DIMS;
    // less than 2^32 threads
    if (a->D > (1 << 30) || (long)a->B * ((a->D + 63) / 64) >= (1L << 26) || (!a->slots && a->P < a->B)) return TGRU_E_DIMS;
    if (!known_dtype(a->dtype)) return TGRU_E_DTYPE;
    if (search_too_long(a->slots, a->B, step_blocks(a->D, a->dtype))) return TGRU_E_DIMS;
    if (!a->x || !a->weight || !a->y || (a->K > 1 && (!a->state || !a->state_out))) return TGRU_E_NULL;
    if (int rc = tgru::check_device()) return rc;
    return dispatch_conv_step(*a, (hipStream_t)stream);
}

}  // extern "C"
