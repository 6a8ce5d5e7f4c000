// Selective scan: h_t = exp(dt_t A) h_{t-1} + dt_t u_t b_t, y_t = (c_t . h_t + skip u_t) silu(z_t) for every channel (N
// states each), its backward pass, and its form for one more token on a pool of states (tgru_scan_* of
// include/tgru.h).
//
// What bounds it.  A step costs, per channel AND STATE, one exponential and four multiply-adds forward, and about
// eighteen operations and the exponential backward, against a few bytes per channel: with 16 states the vector ALU and
// not HBM is the limit.  The matrix instructions do not apply: every (channel, state) pair has a decay of its own at
// every step, so no product of two matrices is shared by two steps.  What the vector ALU of this chip does in how many
// cycles per wave (measured, two or more waves per SIMD): multiplies, adds and multiply-adds 2.3 (4 where both factors are one
// register), DPP adds 4.3, exp2 / reciprocal 8.2, permlane swaps 8.3; with one wave, 4.6 at least.  Between exponentials the
// short ones gain less: three and an exponential take 18.8, not 15.  The four states' arithmetic of a step, measured alone with
// everything in registers, takes a SIMD 37 ns a wave forward (88 cycles), 35 in the pass for the chunks' ends and 155 backward.
// So: enough waves, operands that fit the short encodings, few selects, and no instruction for what is the same in a
// whole wave.
//
// Layout.  A wave owns CH = 64 / S channels of one group: S lanes per channel, four states each (S = 2, 4, 8, 16 covers
// 64 states; states beyond N are zeros throughout), lane = channel * S + part.  A block of Q = 16 steps is staged in LDS:
// what is per channel only (softplus, dt u, the gate) is computed once per (step, channel) by lanes that split the block
// among themselves, the maps' rows are brought to fp32; the next block's rows are requested before the recurrence runs
// over this one.  (Tried instead: a lane with all 16 states of a channel and the maps through the scalar cache -- an eighth
// fewer instructions, but a quarter of the waves: half as slow again on a batch of 64 windows of 256 steps with 1024
// channels, equal on one sequence of 16384.)
//
// scan_bwd_kernel needs the states of every step in reverse.  The forward pass saves the state in front of every block
// (4 bytes per step, channel and 16 states); inside a block the states are computed again, R steps in registers at a time.
// Sums over the states of a channel and over the channels of a group are joined inside the wave with DPP adds and permlane
// swaps.
//
// Time is split into chunks when there are too few channels to fill the chip (make_plan): a first pass leaves each
// chunk's end state from a zero start and its sum of dt -- the chunk multiplies an incoming state by exp(A sum dt) --, a
// second kernel joins the chunks in order, and the main pass starts every chunk from its joined state.  The backward
// pass does the same from the other end.
#include "ssm_common.h"
#include <algorithm>
#include <type_traits>

namespace tgru {
namespace ssm {

constexpr int Q = 16;                // steps per block
constexpr int R = Q / 2;             // steps whose states the backward pass keeps in registers at a time
constexpr int kWaves = 4;            // per workgroup
constexpr int64_t kMaxRowStride = TGRU_SCAN_MAX_ROW_STRIDE;

struct Plan {                        // how a pass is cut up; made on the host
    int NP, CH, Dg;                  // states with padding (8 .. 64), channels per wave, channels per group
    int tpg, tiles, wpg;             // waves per group, per sequence and chunk; workgroups per group (scan_bwd_kernel)
    int nblk;                        // blocks of Q steps
    int nchunks, chunk;              // chunks of time, steps of one (a multiple of Q)
    int quads;                       // the maps' rows can be loaded four values at a time
};

// What goes between kernels, all fp32: ckpt [b][block][d][NP] (the state in front of each block), carry [b][chunk][d][NP],
// sdt [b][chunk][d].

// LDS written by some lanes of a wave and read by others: the LDS unit takes a wave's accesses in order, so all that
// has to be held back is the compiler.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A barrier of the workgroup for what it exchanges through LDS.  Unlike __syncthreads() it does not wait for the wave's
// loads and stores in flight (the next block's rows, this block's gradients).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Sum over the S lanes of a channel, in every one of them.
template <int S>
__device__ __forceinline__ float sum_parts(float v) {
    if constexpr (S >= 2) v = dpp_add<0xB1>(v);      // quad_perm [1,0,3,2]
    if constexpr (S >= 4) v = dpp_add<0x4E>(v);      // quad_perm [2,3,0,1]
    if constexpr (S >= 8) v = dpp_add<0x141>(v);     // row_half_mirror
    if constexpr (S >= 16) v = dpp_add<0x140>(v);    // row_mirror
    return v;
}
// Sums over the CH channels of a wave of four values v[0..3] per lane.  The lanes' two top bits are taken by swapping
// halves and quarters (which leaves one of the four values per quarter of the wave: value 2 * (bit 4) + (bit 5)), the
// channel bits below by rotations of the row.
template <int S>
__device__ __forceinline__ float sum_channels(const float (&v)[4]) {
    auto swap_add32 = [](float x, float y) {
        const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
        return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    };
    auto swap_add16 = [](float x, float y) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
        return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    };
    float s = swap_add16(swap_add32(v[0], v[1]), swap_add32(v[2], v[3]));
    if constexpr (S <= 8) s = dpp_add<0x128>(s);     // row_ror 8
    if constexpr (S <= 4) s = dpp_add<0x124>(s);     // row_ror 4
    if constexpr (S <= 2) s = dpp_add<0x122>(s);     // row_ror 2
    if constexpr (S <= 1) s = dpp_add<0x121>(s);     // row_ror 1
    return s;
}

// A wave's place: channels [d0, d0 + nch) of group g of sequence b, steps [t_lo, t_hi) of which [t_lo, tv) exist.
struct Wave { int b, chunk, g, d0, nch, t_lo, t_hi, tv; };

__device__ __forceinline__ void set_time(Wave &w, const Plan &pl, int T, const int32_t *lengths) {
    w.t_lo = w.chunk * pl.chunk;
    w.t_hi = min(T, w.t_lo + pl.chunk);
    w.tv = min(w.t_hi, clamped_length(lengths, w.b, T));
}

// Rows of a tensor of one block, split over the lanes.  A whole block is read and written by buffer instructions: their
// address is a base that is the same for the wave (it moves by whole blocks), a scalar offset for the row and a 32-bit byte
// offset of the lane, so it costs no vector arithmetic (row strides are below 2^25 elements for that, kMaxRowStride: 15 rows
// of 4-byte elements are offsets below 2^31), and
// the compiler cannot join them with the loads of a block in which the sequence ends, which hold every lane back from the
// rows behind the end.  (Joined, all of them form 64-bit addresses per lane, a tenth of the forward kernel's instructions.)
using Block = __amdgpu_buffer_rsrc_t;
__device__ __forceinline__ Block block_at(const char *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), 0, -1, 0x00020000);
}
template <typename X>
__device__ __forceinline__ X load_elem(Block at, unsigned lane_off, long row_off) {
    if constexpr (sizeof(X) == 2) return __builtin_bit_cast(X, __builtin_amdgcn_raw_buffer_load_b16(at, (int)lane_off, (int)row_off, 0));
    else return __builtin_bit_cast(X, __builtin_amdgcn_raw_buffer_load_b32(at, (int)lane_off, (int)row_off, 0));
}

// A (B, T, D) tensor: element j of a lane is step lane / CH + j S of the block, channel lane % CH of the wave.
template <typename X, int S>
struct Rows {
    static constexpr int CH = 64 / S, E = Q * CH / 64;
    const char *base;                // step 0 of the wave's channels
    long row;                        // bytes from step to step
    unsigned lane_off, col;
    __device__ __forceinline__ void init(const void *p, const int64_t *stride, int b, int d0, int nch) {
        const int lane = threadIdx.x & 63;
        base = reinterpret_cast<const char *>(static_cast<const X *>(p) + b * stride[0] + d0);
        row = stride[1] * (long)sizeof(X);
        col = min(lane % CH, nch - 1) * (unsigned)sizeof(X);
        lane_off = (unsigned)(lane / CH) * (unsigned)row + col;
    }
    // rows t0 .. t0 + Q - 1 of which `left` exist
    __device__ __forceinline__ void load(X (&v)[E], int t0, int left) const {
        const char *p = base + t0 * row;
        if (left >= Q) {
            const Block at = block_at(p);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = load_elem<X>(at, lane_off, j * S * row);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j)
                v[j] = *reinterpret_cast<const X *>(p + ((unsigned)min((int)(threadIdx.x & 63) / CH + j * S, left - 1) * (unsigned)row + col));
        }
    }
    // element j of a block; `whole`: a block and a wave without anything missing
    template <bool whole>
    __device__ __forceinline__ void store(int t0, int j, float v) const {
        const X x = from_float<X>(v);
        if constexpr (!whole) *reinterpret_cast<X *>(const_cast<char *>(base) + (t0 + j * S) * row + lane_off) = x;
        else if constexpr (sizeof(X) == 2)
            __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, x), block_at(base + t0 * row), (int)lane_off, (int)(j * S * row), 0);
        else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), block_at(base + t0 * row), (int)lane_off, (int)(j * S * row), 0);
    }
};

// Rows of b or c of a block on their way to LDS, in fp32, zeros beyond N and behind the end: Q rows of S quads of values,
// a quad per lane and element.
template <typename X, int S>
struct Maps {
    static constexpr int F = Q * S, V = F < 64 ? 1 : F / 64;           // quads in all, per lane
    struct alignas(4 * sizeof(X)) Quad { X v[4]; };
    // A quad as it is in registers: words, since two ways of loading the same four values are joined by the compiler into
    // the slower one.
    typedef unsigned Words __attribute__((ext_vector_type(sizeof(X)), may_alias));
    const char *base;
    long row;
    unsigned lane_off;
    Words q[V];
    __device__ __forceinline__ void init(const void *p, const int64_t *stride, int b, int g, int N) {
        const int lane = threadIdx.x & 63;
        base = reinterpret_cast<const char *>(static_cast<const X *>(p) + b * stride[0] + g * stride[2]);
        row = stride[1] * (long)sizeof(X);
        lane_off = (unsigned)min(lane / S, Q - 1) * (unsigned)row + (unsigned)max(min(4 * (lane % S), N - 4), 0) * (unsigned)sizeof(X);
    }
    // quads: every row starts on a quad and N is a multiple of 4 -- one load instead of four
    __device__ __forceinline__ void load(int t0, int left, int N, int quads) {
        const int lane = threadIdx.x & 63;
        const char *p = base + t0 * row;
        if (quads && left >= Q) {
            const Block at = block_at(p);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (sizeof(X) == 2)
                    q[j] = __builtin_bit_cast(Words, __builtin_amdgcn_raw_buffer_load_b64(at, (int)lane_off, (int)(j * (64 / S) * row), 0));
                else
                    q[j] = __builtin_bit_cast(Words, __builtin_amdgcn_raw_buffer_load_b128(at, (int)lane_off, (int)(j * (64 / S) * row), 0));
            }
            return;
        }
        const int first = lane / S, rows = min(left, Q) - 1;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const char *r = p + (unsigned)min(first + j * (64 / S), rows) * (unsigned)row;
            if (quads) {
                q[j] = *reinterpret_cast<const Words *>(r + min(4 * (lane % S), N - 4) * (unsigned)sizeof(X));
            } else {
                Quad one;
#pragma unroll
                for (int k = 0; k < 4; ++k) one.v[k] = *reinterpret_cast<const X *>(r + min(4 * (lane % S) + k, N - 1) * (unsigned)sizeof(X));
                q[j] = __builtin_bit_cast(Words, one);
            }
        }
    }
    __device__ __forceinline__ void to_lds(float *lds, int left, int N) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int t = lane / S + j * (64 / S), n = 4 * (lane % S);
            const Quad one = __builtin_bit_cast(Quad, q[j]);
            float4 f;
            f.x = to_float(one.v[0]); f.y = to_float(one.v[1]); f.z = to_float(one.v[2]); f.w = to_float(one.v[3]);
            if (left < Q || N < 4 * S) {
                f.x = (t < left && n < N) ? f.x : 0.f;
                f.y = (t < left && n + 1 < N) ? f.y : 0.f;
                f.z = (t < left && n + 2 < N) ? f.z : 0.f;
                f.w = (t < left && n + 3 < N) ? f.w : 0.f;
            }
            if (F >= 64 || lane < F) reinterpret_cast<float4 *>(lds)[lane + 64 * j] = f;
        }
    }
};

// What a step reads from LDS, fetched one step ahead: a read takes as long as two steps' arithmetic of the four states,
// and the compiler, left alone, waits for each right behind it.  ahead() keeps the fetches in front of what follows.
struct StepIn { float4 v, b, c; };
__device__ __forceinline__ void ahead() { __builtin_amdgcn_sched_barrier(0); }

// A wave of the passes whose waves are independent of each other; false where there is none.
__device__ __forceinline__ bool place_wave(Wave &w, const tgru_scan_args &a, const Plan &pl) {
    const unsigned id = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned rest = id / (unsigned)pl.tiles, flat = id - rest * (unsigned)pl.tiles;
    w.b = (int)(rest / (unsigned)pl.nchunks);
    if (w.b >= a.B) return false;
    w.chunk = (int)(rest - (unsigned)w.b * (unsigned)pl.nchunks);
    w.g = (int)(flat / (unsigned)pl.tpg);
    const int in_group = (int)flat - w.g * pl.tpg;
    w.d0 = w.g * pl.Dg + in_group * pl.CH;
    w.nch = min(pl.CH, pl.Dg - in_group * pl.CH);
    set_time(w, pl, a.T, a.lengths);
    return true;
}

// An infinite rate is taken as 3e38: the same decay to nothing for every dt > 0, and a step of dt = 0 leaves the state as it
// is (0 times infinity would not).
__device__ __forceinline__ float finite_rate(float v) { return __builtin_isinf(v) ? __builtin_copysignf(3.0e38f, v) : v; }

// This lane's four states: where they are in a row of carry or ckpt, and their rates to base 2 per unit of dt.  Steps behind
// a sequence's end are staged as dt = 0, which leaves a state as it is, exactly: exp2(0 a2) = 1 for every finite a2.
template <int S>
struct Lane {
    int c, s;                        // channel of the wave, part of the channel
    bool on;
    long at;
    float a2[4];
    __device__ __forceinline__ void init(const float *rates, int N, const Wave &w) {
        c = (threadIdx.x & 63) / S;
        s = (threadIdx.x & 63) % S;
        on = c < w.nch;
        at = (long)(w.d0 + (on ? c : 0)) * (4 * S) + 4 * s;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a2[k] = has(k, N) ? finite_rate(rates[(long)(w.d0 + c) * N + 4 * s + k] * kLog2e) : 0.f;
        }
    }
    __device__ __forceinline__ bool has(int k, int N) const { return on && 4 * s + k < N; }
    // from / to a (B, D, N) tensor
    __device__ __forceinline__ void load(const float *t, const Wave &w, int D, int N, float (&v)[4]) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = has(k, N) ? t[((long)w.b * D + w.d0 + c) * N + 4 * s + k] : 0.f;
    }
    __device__ __forceinline__ void store(float *t, const Wave &w, int D, int N, const float (&v)[4]) const {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (has(k, N)) t[((long)w.b * D + w.d0 + c) * N + 4 * s + k] = v[k];
    }
};

__device__ __forceinline__ void unpack(const float4 &f, float (&v)[4]) { v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w; }

// MODE 0: the outputs.  MODE 1: a chunk's end state from a zero start and its sum of dt, for the joining kernel.
// 28 instructions a wave and step (21 in MODE 1), of which 20 (17) are the four states' arithmetic.  Measured, 16 states: one
// sequence of 16384 steps, 2048 channels, bf16, in 32 chunks: 140 us, MODE 1 100 us and the joining 6, which is 68 and 49 ns a
// wave and step of a SIMD with four waves where that arithmetic alone takes 37 and 35.  The other instructions are some 15 and 8 ns
// at their rates; the rest is waiting, though not for the maps: a copy that read one row of them for all steps was no faster,
// one without any of a step's LDS reads by 3 %, one without the exponentials by 22 % (MODE 1 by 35 %).  64 windows of 256
// steps, 1024 channels, fp32: 88 us, 86 ns a wave and step, 3.8 TB/s, so memory counts there as well.
template <typename X, int S, int MODE>
__global__ __launch_bounds__(64 * kWaves) void scan_fwd_kernel(tgru_scan_args a, Plan pl, float *carry, float *sdt) {
    constexpr int CH = 64 / S, NP = 4 * S, E = Q * CH / 64, M = MODE == 0 ? 2 : 1;
    __shared__ float2 s_steps[kWaves][Q][CH];                           // dt, dt * u
    __shared__ __align__(16) float s_maps[kWaves][M][Q][NP];            // b, c
    __shared__ __align__(16) float s_ys[MODE == 0 ? kWaves : 1][Q][64]; // the lanes' shares of c . h
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto &s_step = s_steps[wv];
    auto &s_map = s_maps[wv];
    auto &s_y = s_ys[MODE == 0 ? wv : 0];
    Wave w;
    if (!place_wave(w, a, pl)) return;
    if (MODE == 1 && w.chunk == pl.nchunks - 1) return;                 // nobody goes on from it
    Lane<S> me;
    me.init(a.a, a.N, w);
    const int ec = lane % CH, ed = w.d0 + min(ec, w.nch - 1);           // this lane's channel when it works per channel
    const bool e_on = ec < w.nch;
    const float bias = a.delta_bias ? a.delta_bias[ed] : 0.f, skip = (MODE == 0 && a.skip) ? a.skip[ed] : 0.f;
    float h[4] = {0.f, 0.f, 0.f, 0.f}, dts = 0.f;
    float4 *state = reinterpret_cast<float4 *>(carry + ((long)w.b * pl.nchunks + w.chunk) * a.D * NP + me.at);
    if (MODE == 0) {
        if (pl.nchunks > 1) { if (me.on) unpack(*state, h); }
        else if (a.initial_state) me.load(a.initial_state, w, a.D, a.N, h);
    }
    float *ckpt = (MODE == 0 && a.reserve) ? a.reserve + (long)w.b * pl.nblk * a.D * NP + me.at : nullptr;
    Rows<X, S> pu, pd, pz, py;
    Maps<X, S> mb, mc;
    pu.init(a.u, a.u_stride, w.b, w.d0, w.nch);
    pd.init(a.delta, a.delta_stride, w.b, w.d0, w.nch);
    mb.init(a.b, a.b_stride, w.b, w.g, a.N);
    if (MODE == 0) {
        py.init(a.y, a.y_stride, w.b, w.d0, w.nch);
        mc.init(a.c, a.c_stride, w.b, w.g, a.N);
        if (a.z) pz.init(a.z, a.z_stride, w.b, w.d0, w.nch);
    }
    X ru[E], rd[E], rz[E];
    auto request = [&](int t0) {
        const int left = w.tv - t0;
        pu.load(ru, t0, left);
        pd.load(rd, t0, left);
        mb.load(t0, left, a.N, pl.quads);
        if (MODE == 0) {
            mc.load(t0, left, a.N, pl.quads);
            if (a.z) pz.load(rz, t0, left);
        }
    };
    if (w.t_lo < w.tv) request(w.t_lo);
    for (int t0 = w.t_lo; t0 < w.tv; t0 += Q) {
        float u[E], z[E];
        const int left = w.tv - t0;
        wave_sync();
        // (a block that is there in full, in a wave whose channels all exist, needs no selection)
        auto stage = [&](auto full) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int et = lane / CH + j * S;
                const bool on = full.value || (e_on && et < left);
                u[j] = on ? to_float(ru[j]) : 0.f;
                z[j] = (MODE == 0 && a.z) ? to_float(rz[j]) : 0.f;
                const float raw = to_float(rd[j]) + bias;
                const float dt = on ? (a.softplus ? softplus(raw) : raw) : 0.f;
                s_step[et][ec] = make_float2(dt, dt * u[j]);
            }
        };
        const bool full = left >= Q && w.nch == CH;
        if (full) stage(std::true_type{});
        else stage(std::false_type{});
        mb.to_lds(&s_map[0][0][0], left, a.N);
        if (MODE == 0) mc.to_lds(&s_map[M - 1][0][0], left, a.N);
        if (left > Q) request(t0 + Q);
        wave_sync();
        if (ckpt && me.on) *reinterpret_cast<float4 *>(ckpt + (long)(t0 / Q) * a.D * NP) = make_float4(h[0], h[1], h[2], h[3]);
        auto fetch = [&](int i) {
            StepIn in;
            const float2 v = s_step[i][me.c];
            in.v = make_float4(v.x, v.y, 0.f, 0.f);
            in.b = *reinterpret_cast<const float4 *>(&s_map[0][i][4 * me.s]);
            if (MODE == 0) in.c = *reinterpret_cast<const float4 *>(&s_map[M - 1][i][4 * me.s]);
            return in;
        };
        auto step = [&](int i, const StepIn &in) {
            float bb[4];
            unpack(in.b, bb);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                h[k] = __builtin_fmaf(__builtin_amdgcn_exp2f(in.v.x * me.a2[k]), h[k], in.v.y * bb[k]);
            if (MODE == 1) dts += in.v.x;
            else s_y[i][lane] = __builtin_fmaf(in.c.x, h[0], __builtin_fmaf(in.c.y, h[1], __builtin_fmaf(in.c.z, h[2], in.c.w * h[3])));
        };
        auto steps = [&](auto count) {
            StepIn next = fetch(0);
#pragma unroll
            for (int i = 0; i < count.value; ++i) {
                const StepIn in = next;
                if (i + 1 < count.value) next = fetch(i + 1);
                ahead();
                step(i, in);
            }
        };
        if (left > Q / 2) steps(std::integral_constant<int, Q>{});
        else for (int i = 0; i < left; ++i) step(i, fetch(i));
        if (MODE == 0) {
            wave_sync();
            auto finish = [&](auto full) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const int et = lane / CH + j * S;
                    if (!full.value && (!e_on || et >= left)) continue;
                    float y = skip * u[j];
#pragma unroll
                    for (int q = 0; q < S; ++q) y += s_y[et][ec * S + q];
                    if (a.z) y *= z[j] * sigmoid(z[j]);
                    py.template store<decltype(full)::value>(t0, j, y);
                }
            };
            if (full) finish(std::true_type{});
            else finish(std::false_type{});
        }
    }
    if (MODE == 1) {
        if (!me.on) return;
        *state = make_float4(h[0], h[1], h[2], h[3]);
        if (me.s == 0) sdt[((long)w.b * pl.nchunks + w.chunk) * a.D + w.d0 + me.c] = dts;
        return;
    }
    for (int t = max(w.t_lo, w.tv) + lane / CH; t < w.t_hi; t += S)
        if (e_on) static_cast<X *>(a.y)[w.b * a.y_stride[0] + t * a.y_stride[1] + ed] = from_float<X>(0.f);
    if (a.final_state && w.chunk == pl.nchunks - 1) me.store(a.final_state, w, a.D, a.N, h);
}

// The gradient that a chunk hands to the one before it, from zero behind its end, and its sum of dt: MODE 1 above from the
// other end, with c dy in the place of b dt u.  54 us for 4 sequences of 2048 steps, 2048 channels, bf16.
template <typename X, int S>
__global__ __launch_bounds__(64 * kWaves) void scan_back_kernel(tgru_scan_args a, Plan pl, float *carry, float *sdt) {
    constexpr int CH = 64 / S, NP = 4 * S, E = Q * CH / 64;
    __shared__ float2 s_steps[kWaves][Q][CH];                           // dt, dy
    __shared__ __align__(16) float s_maps[kWaves][Q][NP];               // c
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto &s_step = s_steps[wv];
    auto &s_map = s_maps[wv];
    Wave w;
    if (!place_wave(w, a, pl) || w.chunk == 0) return;
    Lane<S> me;
    me.init(a.a, a.N, w);
    const int ec = lane % CH;
    const bool e_on = ec < w.nch;
    const float bias = a.delta_bias ? a.delta_bias[w.d0 + min(ec, w.nch - 1)] : 0.f;
    float g[4] = {0.f, 0.f, 0.f, 0.f}, dts = 0.f;
    Rows<X, S> pd, pz, pg;
    Maps<X, S> mc;
    pd.init(a.delta, a.delta_stride, w.b, w.d0, w.nch);
    mc.init(a.c, a.c_stride, w.b, w.g, a.N);
    if (a.dy) pg.init(a.dy, a.dy_stride, w.b, w.d0, w.nch);
    if (a.z) pz.init(a.z, a.z_stride, w.b, w.d0, w.nch);
    X rd[E], rz[E], rg[E];
    auto request = [&](int t0) {
        const int left = w.tv - t0;
        pd.load(rd, t0, left);
        if (a.dy) pg.load(rg, t0, left);
        if (a.z) pz.load(rz, t0, left);
        mc.load(t0, left, a.N, pl.quads);
    };
    const int last = w.tv > w.t_lo ? w.t_lo + (w.tv - 1 - w.t_lo) / Q * Q : w.t_lo - Q;
    if (last >= w.t_lo) request(last);
    for (int t0 = last; t0 >= w.t_lo; t0 -= Q) {
        const int left = w.tv - t0;
        wave_sync();
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int et = lane / CH + j * S;
            const bool on = e_on && et < left;
            const float raw = to_float(rd[j]) + bias;
            float dy = a.dy ? to_float(rg[j]) : 0.f;
            if (a.z) { const float z = to_float(rz[j]); dy *= z * sigmoid(z); }
            s_step[et][ec] = make_float2(on ? (a.softplus ? softplus(raw) : raw) : 0.f, on ? dy : 0.f);
        }
        mc.to_lds(&s_map[0][0], left, a.N);
        if (t0 > w.t_lo) request(t0 - Q);
        wave_sync();
        auto fetch = [&](int i) {
            StepIn in;
            const float2 v = s_step[i][me.c];
            in.v = make_float4(v.x, v.y, 0.f, 0.f);
            in.c = *reinterpret_cast<const float4 *>(&s_map[i][4 * me.s]);
            return in;
        };
        auto step = [&](const StepIn &in) {
            float cc[4];
            unpack(in.c, cc);
#pragma unroll
            for (int k = 0; k < 4; ++k) g[k] = __builtin_amdgcn_exp2f(in.v.x * me.a2[k]) * __builtin_fmaf(in.v.y, cc[k], g[k]);
            dts += in.v.x;
        };
        StepIn next = fetch(Q - 1);
#pragma unroll
        for (int i = Q - 1; i >= 0; --i) {
            const StepIn in = next;
            if (i > 0) next = fetch(i - 1);
            ahead();
            step(in);
        }
    }
    if (!me.on) return;
    *reinterpret_cast<float4 *>(carry + ((long)w.b * pl.nchunks + w.chunk) * a.D * NP + me.at) = make_float4(g[0], g[1], g[2], g[3]);
    if (me.s == 0) sdt[((long)w.b * pl.nchunks + w.chunk) * a.D + w.d0 + me.c] = dts;
}

// 2^x h + v.  The growth of a whole chunk may be beyond float (negative steps, positive rates: 32 steps of half a unit at a
// rate of 16 are 2^185) where what it makes of a small state, or of none, is not, so the whole part of x goes into the exponent
// of h: 0 stays 0, and the rest is a factor in [1, 2).  (Beyond 4000 every float but 0 has left the range; a NaN that this
// loses is in v as well.)
__device__ __forceinline__ float add_grown(float h, float x, float v) {
    const float in = fminf(fmaxf(x, -4000.f), 4000.f), whole = floorf(in);
    return __builtin_fmaf(__builtin_amdgcn_ldexpf(h, (int)whole), __builtin_amdgcn_exp2f(in - whole), v);
}

// Joins the chunks: carry[chunk] becomes what enters the chunk.  (What the last one in the order of the pass would hand on
// was not computed: its slot is read, and what comes of it is not used.)  `edge`: (B, D, N) entering the first chunk in the
// order of the pass (the initial state forward, the final state's gradient backward), or null.  One thread per state.
__global__ __launch_bounds__(64) void scan_join_kernel(const float *a, const float *edge, Plan pl, int B, int D, int N, int backward,
                                                       float *carry, const float *sdt) {
    const long id = (long)blockIdx.x * 64 + threadIdx.x, per = (long)D * pl.NP;
    const int b = (int)(id / per);
    if (b >= B) return;
    const int e = (int)(id - b * per), d = e / pl.NP, n = e - d * pl.NP;
    const float a2 = n < N ? a[(long)d * N + n] * kLog2e : 0.f;
    float h = (edge && n < N) ? edge[((long)b * D + d) * N + n] : 0.f;
    float *state = carry + (long)b * pl.nchunks * per + e;
    const float *sums = sdt + (long)b * pl.nchunks * D + d;
    constexpr int U = 8;                 // chunks requested together
    for (int i0 = 0; i0 < pl.nchunks; i0 += U) {
        float v[U], dt[U];
#pragma unroll
        for (int r = 0; r < U; ++r) {
            const int i = min(i0 + r, pl.nchunks - 1), at = backward ? pl.nchunks - 1 - i : i;
            v[r] = state[at * per];
            dt[r] = sums[(long)at * D];
        }
#pragma unroll
        for (int r = 0; r < U; ++r) {
            if (i0 + r >= pl.nchunks) break;
            state[(backward ? pl.nchunks - 1 - (i0 + r) : i0 + r) * per] = h;
            // a chunk without steps passes the state on as it is, also where A is infinite
            h = add_grown(h, dt[r] == 0.f ? 0.f : dt[r] * a2, v[r]);
        }
    }
}

// Backward.  With g_t the gradient of h_t:  g_t = c_t dy_t + exp(dt_{t+1} A) g_{t+1},
//     dc_t = sum over channels dy_t h_t            db_t = sum over channels g_t dt_t u_t
//     du_t = dt_t (g_t . b_t) + skip dy_t          w_t = g_t exp(dt_t A) h_{t-1}
//     d(dt_t) = u_t (g_t . b_t) + A . w_t          dA = sum over steps dt_t w_t
// where dy is the gradient in front of the gate.  The four waves of a workgroup are neighbouring waves of one group, one
// sequence and one chunk: their sums over channels are joined in LDS and one row per workgroup goes to memory.
//
// 101 instructions a wave and step, of which 83 are the four states' arithmetic and its sums, with two waves a SIMD (the
// states and decays of R steps are 64 registers; with bounds for three waves it spills and is half as slow again).  Measured: 64
// windows of 256 steps, 1024 channels, 16 states, fp32, 260 us; 4 sequences of 2048 steps, 2048 channels, bf16, 240 us: 254 and
// 234 ns a wave and step where that arithmetic alone takes 155 with two waves.  Some 35 ns are the other instructions at their rates,
// the rest is waiting that two waves do not cover (a step's sums are chains of seven instructions).  Of 275 us that an earlier
// run took, copies without one part each (wrong results) saved: the sums over channels 45 us, the exponentials 27, stores and
// their arithmetic 28, the first half's second run 20, the sums over states and softplus 12 each, the joining of the four waves 7;
// R = 4 took 289, sums over channels exchanged through LDS 318.  With N <= 8 (S = 2) a lane has twice the work per channel and the
// compiler spills 31 to 39 registers outside the loops over steps: such a call takes about as long as one with 16 states.
template <typename X, int S>
__global__ __launch_bounds__(64 * kWaves, 2) void scan_bwd_kernel(tgru_scan_args a, Plan pl, const float *carry, float *map_part,
                                                              float *par_part) {
    constexpr int CH = 64 / S, NP = 4 * S, E = Q * CH / 64;
    __shared__ float4 s_step[kWaves][Q][CH];         // dt, dt * u, dy; then the step's sums g . b, A . w, c . h
    // rows b, c; then the wave's db, dc, which the workgroup joins while the next block fills the other buffer
    __shared__ __align__(16) float s_maps[2][kWaves][2][Q][NP];
    int buf = 0;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Wave w;
    unsigned id = blockIdx.x;
    const int wg = (int)(id % (unsigned)pl.wpg);
    id /= (unsigned)pl.wpg;
    w.g = (int)(id % (unsigned)a.G);
    id /= (unsigned)a.G;
    w.chunk = (int)(id % (unsigned)pl.nchunks);
    w.b = (int)(id / (unsigned)pl.nchunks);
    const int in_group = wg * kWaves + wv;
    const bool wave_on = in_group < pl.tpg;          // the last workgroup of a group may have waves to spare:
    const int tile = wave_on ? in_group : pl.tpg - 1;     // they load a channel and use nothing of it
    w.d0 = w.g * pl.Dg + tile * CH;
    w.nch = wave_on ? min(CH, pl.Dg - tile * CH) : 0;
    set_time(w, pl, a.T, a.lengths);
    const int load_ch = wave_on ? w.nch : 1;
    Lane<S> me;
    me.init(a.a, a.N, w);
    const int c = me.c, s = me.s, ec = lane % CH;
    const bool e_on = ec < w.nch;
    const int ed = w.d0 + min(ec, load_ch - 1);
    const float bias = a.delta_bias ? a.delta_bias[ed] : 0.f, skip = a.skip ? a.skip[ed] : 0.f;
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    if (pl.nchunks > 1) {
        if (me.on) unpack(*reinterpret_cast<const float4 *>(carry + ((long)w.b * pl.nchunks + w.chunk) * a.D * NP + me.at), g);
    } else if (a.dfinal) {
        me.load(a.dfinal, w, a.D, a.N, g);
    }
    Rows<X, S> pu, pd, pz, pg, pdu, pdd, pdz;
    Maps<X, S> mb, mc;
    mb.init(a.b, a.b_stride, w.b, w.g, a.N);
    mc.init(a.c, a.c_stride, w.b, w.g, a.N);
    pu.init(a.u, a.u_stride, w.b, w.d0, load_ch);
    pd.init(a.delta, a.delta_stride, w.b, w.d0, load_ch);
    if (a.dy) pg.init(a.dy, a.dy_stride, w.b, w.d0, load_ch);
    if (a.z) pz.init(a.z, a.z_stride, w.b, w.d0, load_ch);
    if (a.du) pdu.init(a.du, a.du_stride, w.b, w.d0, load_ch);
    if (a.ddelta) pdd.init(a.ddelta, a.ddelta_stride, w.b, w.d0, load_ch);
    if (a.dz) pdz.init(a.dz, a.dz_stride, w.b, w.d0, load_ch);
    const float *ckpt = a.reserve + (long)w.b * pl.nblk * a.D * NP + me.at;
    X ru[E], rd[E], rz[E], rg[E];
    float4 rh;
    auto request = [&](int t0) {
        const int left = w.tv - t0;
        pd.load(rd, t0, left);
        pu.load(ru, t0, left);
        if (a.dy) pg.load(rg, t0, left);
        if (a.z) pz.load(rz, t0, left);
        mb.load(t0, left, a.N, pl.quads);
        mc.load(t0, left, a.N, pl.quads);
        rh = *reinterpret_cast<const float4 *>(ckpt + (long)(t0 / Q) * a.D * NP);
    };
    // sums over all steps: dA by state, dskip and ddelta_bias by channel
    float dA[4] = {0.f, 0.f, 0.f, 0.f}, dskip = 0.f, dbias = 0.f;
    const int last = w.tv > w.t_lo ? w.t_lo + (w.tv - 1 - w.t_lo) / Q * Q : w.t_lo - Q;
    if (last >= w.t_lo) request(last);
    for (int t0 = last; t0 >= w.t_lo; t0 -= Q) {
        float u[E], z[E], out[E], dt[E], dy[E], slope[E], gate[E];
        const int left = w.tv - t0;                  // steps of this block that exist (Q or more: all)
        auto &s_map = s_maps[buf][wv];
        wave_sync();
        // (a block that is there in full, in a wave whose channels all exist, needs no selection)
        const bool full = left >= Q && w.nch == CH;
        auto stage = [&](auto full) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const int et = lane / CH + j * S;
                const bool on = full.value || (e_on && et < left);
                u[j] = on ? to_float(ru[j]) : 0.f;
                out[j] = (a.dy && on) ? to_float(rg[j]) : 0.f;
                const float raw = to_float(rd[j]) + bias;
                dt[j] = raw;
                slope[j] = 1.f;
                if (a.softplus) softplus_slope(raw, dt[j], slope[j]);
                if (!full.value) dt[j] = on ? dt[j] : 0.f;
                dy[j] = out[j];
                if (a.z) {
                    z[j] = to_float(rz[j]);
                    gate[j] = sigmoid(z[j]);
                    dy[j] *= z[j] * gate[j];
                    if (!full.value) dy[j] = on ? dy[j] : 0.f;
                }
                s_step[wv][et][ec] = make_float4(dt[j], dt[j] * u[j], dy[j], 0.f);
            }
        };
        if (full) stage(std::true_type{});
        else stage(std::false_type{});
        mb.to_lds(&s_map[0][0][0], left, a.N);
        mc.to_lds(&s_map[1][0][0], left, a.N);
        const float h0[4] = {me.on ? rh.x : 0.f, me.on ? rh.y : 0.f, me.on ? rh.z : 0.f, me.on ? rh.w : 0.f};
        if (t0 > w.t_lo) request(t0 - Q);
        wave_sync();
        float blkA[4] = {0.f, 0.f, 0.f, 0.f};
        auto fetch = [&](int i, bool reverse) {
            StepIn in;
            in.v = s_step[wv][i][c];
            in.b = *reinterpret_cast<const float4 *>(&s_map[0][i][4 * s]);
            if (reverse) in.c = *reinterpret_cast<const float4 *>(&s_map[1][i][4 * s]);
            return in;
        };
        auto advance = [&](const StepIn &in, const float (&from)[4], float (&to)[4], float (&decay)[4]) {
            const float bb[4] = {in.b.x, in.b.y, in.b.z, in.b.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                decay[k] = __builtin_amdgcn_exp2f(in.v.x * me.a2[k]);
                to[k] = __builtin_fmaf(decay[k], from[k], in.v.y * bb[k]);
            }
        };
        // steps first .. first + R - 1 of the block, from state h0 in front of them; `next` is step `first`
        auto part = [&](auto first_, const float (&h0)[4], StepIn next) {
            constexpr int first = first_.value;
            float decay[R][4], h[R][4];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const StepIn in = next;
                next = i + 1 < R ? fetch(first + i + 1, false) : fetch(first + R - 1, true);
                ahead();
                advance(in, i ? h[i ? i - 1 : 0] : h0, h[i], decay[i]);
            }
            // from the last step to the first
#pragma unroll
            for (int i = R - 1; i >= 0; --i) {
                const StepIn in = next;
                if (i > 0) next = fetch(first + i - 1, true);
                ahead();
                float bb[4], cc[4], db[4], dc[4], gb = 0.f, aw = 0.f, ch = 0.f;
                unpack(in.b, bb);
                unpack(in.c, cc);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float gt = __builtin_fmaf(in.v.z, cc[k], g[k]);
                    dc[k] = in.v.z * h[i][k];
                    db[k] = in.v.y * gt;
                    gb = __builtin_fmaf(gt, bb[k], gb);
                    ch = __builtin_fmaf(cc[k], h[i][k], ch);
                    g[k] = gt * decay[i][k];
                    const float wk = g[k] * (i ? h[i ? i - 1 : 0][k] : h0[k]);
                    aw = __builtin_fmaf(wk, me.a2[k], aw);
                    blkA[k] = __builtin_fmaf(wk, in.v.x, blkA[k]);
                }
                // (all lanes that hold a sum write it, the same value to the same place: no selection, no branch)
                s_step[wv][first + i][c] = make_float4(sum_parts<S>(gb), sum_parts<S>(aw), sum_parts<S>(ch), 0.f);
                // quarter q of the wave has, in part s of each of its channels, the sums of state 4 s + value of q
                const int n = 4 * s + 2 * ((lane >> 4) & 1) + (lane >> 5);
                s_map[0][first + i][n] = sum_channels<S>(db);
                s_map[1][first + i][n] = sum_channels<S>(dc);
            }
        };
        // The states of R steps are kept in registers: the second half of the block first, from a state that is carried
        // through the first half and forgotten again.
        if (left > R) {
            float hm[4] = {h0[0], h0[1], h0[2], h0[3]}, decay[4];
            StepIn next = fetch(0, false);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const StepIn in = next;
                next = fetch(i + 1, false);
                ahead();
                advance(in, hm, hm, decay);
            }
            part(std::integral_constant<int, R>{}, hm, next);
        }
        part(std::integral_constant<int, 0>{}, h0, fetch(0, false));
#pragma unroll
        for (int k = 0; k < 4; ++k) dA[k] += blkA[k];
        wave_sync();
        float bs = 0.f, bb = 0.f;
        float4 sums[E];
#pragma unroll
        for (int j = 0; j < E; ++j) sums[j] = s_step[wv][lane / CH + j * S][ec];
        auto finish = [&](auto full) {
            auto each = [&](auto f) {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (full.value || (e_on && lane / CH + j * S < left)) f(j);
            };
            each([&](int j) {
                const float du = __builtin_fmaf(sums[j].x, dt[j], skip * dy[j]);
                bs = __builtin_fmaf(dy[j], u[j], bs);
                if (a.du) pdu.template store<decltype(full)::value>(t0, j, du);
            });
            each([&](int j) {
                const float dd = __builtin_fmaf(sums[j].x, u[j], kLn2 * sums[j].y) * slope[j];
                bb += dd;
                if (a.ddelta) pdd.template store<decltype(full)::value>(t0, j, dd);
            });
            if (a.dz)
                each([&](int j) {
                    pdz.template store<decltype(full)::value>(t0, j, out[j] * __builtin_fmaf(skip, u[j], sums[j].z) * gate[j] * __builtin_fmaf(z[j], 1.f - gate[j], 1.f));
                });
        };
        if (full) finish(std::true_type{});
        else finish(std::false_type{});
        dskip += bs;
        dbias += bb;
        if (map_part) {
            // the four waves' sums of this block, joined: map_part[b][g][workgroup][db, dc][t][NP]
            lds_barrier();
            const long row = (((long)w.b * a.G + w.g) * pl.wpg + wg) * 2;
            const int n = min(left, Q) * NP;
            for (int m = 0; m < 2; ++m) {
                float *to = map_part + ((row + m) * a.T + t0) * NP;
                for (int e = threadIdx.x; e < n; e += 64 * kWaves) {
                    float v = 0.f;
#pragma unroll
                    for (int q = 0; q < kWaves; ++q) v += (&s_maps[buf][q][m][0][0])[e];
                    to[e] = v;
                }
            }
            buf ^= 1;
        }
    }
    // rows behind the end
    for (int t = max(w.t_lo, w.tv) + lane / CH; t < w.t_hi; t += S) {
        if (!e_on) break;
        const X zero = from_float<X>(0.f);
        if (a.du) static_cast<X *>(a.du)[w.b * a.du_stride[0] + t * a.du_stride[1] + ed] = zero;
        if (a.ddelta) static_cast<X *>(a.ddelta)[w.b * a.ddelta_stride[0] + t * a.ddelta_stride[1] + ed] = zero;
        if (a.dz) static_cast<X *>(a.dz)[w.b * a.dz_stride[0] + t * a.dz_stride[1] + ed] = zero;
    }
    if (a.dinitial && w.chunk == 0) me.store(a.dinitial, w, a.D, a.N, g);
    if (!par_part) return;
    // par_part[b, chunk][dA (D, N) | dskip (D) | ddelta_bias (D)]
    float *to = par_part + ((long)w.b * pl.nchunks + w.chunk) * a.D * (a.N + 2);
    if (c < w.nch) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (4 * s + k < a.N) to[(long)(w.d0 + c) * a.N + 4 * s + k] = dA[k];
    }
#pragma unroll
    for (int m = CH; m < 64; m <<= 1) {
        dskip += __shfl_xor(dskip, m);
        dbias += __shfl_xor(dbias, m);
    }
    if (lane < CH && e_on) {
        to[(long)a.D * a.N + ed] = dskip;
        to[(long)a.D * (a.N + 1) + ed] = dbias;
    }
}

// The gradients that several workgroups of scan_bwd_kernel have a share of; everything is added in a fixed order.
//   workgroups [0, map_blocks): db, dc (B, T, G, N) from map_part[b][g][workgroup][db, dc][t][NP]; zeros behind the end
//   the others: da, dskip, ddelta_bias from the rows of par_part[rows][D (N + 2)], 32 columns x 8 groups of rows each
template <typename X>
__global__ __launch_bounds__(256) void scan_grads_kernel(tgru_scan_args a, Plan pl, const float *__restrict__ map_part, unsigned map_blocks,
                                                         const float *__restrict__ par_part) {
    if (blockIdx.x < map_blocks) {
        // four states a thread; (b, g, db | dc, t, quad of states)
        const int quads = pl.NP / 4, shift = __builtin_ctz(quads);
        const long per = (long)a.T * quads, all = (long)a.B * a.G * 2 * per, stride = (long)map_blocks * 256;
        struct alignas(sizeof(X)) Four { X v[4]; };
        for (long id = (long)blockIdx.x * 256 + threadIdx.x; id < all; id += stride) {
            const long part = all < 4294967296L ? (long)((unsigned)id / (unsigned)per) : id / per, bg = part >> 1;
            const int e = (int)(id - part * per), t = e >> shift, n = (e & (quads - 1)) * 4;
            if (n >= a.N) continue;
            const int b = a.G == 1 ? (int)bg : (int)(bg / a.G), g = (int)(bg - (long)b * a.G);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t < clamped_length(a.lengths, b, a.T)) {
                const float4 *p = reinterpret_cast<const float4 *>(map_part) + (bg * pl.wpg * 2 + (part & 1)) * per + e;
#pragma unroll 8
                for (int q = 0; q < pl.wpg; ++q) {
                    const float4 f = p[q * 2 * per];
                    v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
                }
            }
            X *to = static_cast<X *>((part & 1) ? a.dc : a.db);
            if (!to) continue;
            to += (((long)b * a.T + t) * a.G + g) * a.N + n;
            const Four four = {{from_float<X>(v.x), from_float<X>(v.y), from_float<X>(v.z), from_float<X>(v.w)}};
            if (n + 4 <= a.N) {
                *reinterpret_cast<Four *>(to) = four;
            } else {
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    if (n + k < a.N) to[k] = four.v[k];
            }
        }
        return;
    }
    __shared__ float red[8][32];
    const int c = threadIdx.x & 31, grp = threadIdx.x >> 5, rows = a.B * pl.nchunks;
    const int each = (rows + 7) / 8, r0 = grp * each, r1 = min(rows, r0 + each);
    const long cols = (long)a.D * (a.N + 2), dn = (long)a.D * a.N;
    for (long col0 = (long)(blockIdx.x - map_blocks) * 32; col0 < cols; col0 += (long)(gridDim.x - map_blocks) * 32) {
        const long col = col0 + c;
        const float s = col < cols ? sum_rows(par_part + col, cols, r0, r1) : 0.f;
        __syncthreads();
        red[grp][c] = s;
        __syncthreads();
        if (grp != 0 || col >= cols) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += red[q][c];
        if (col < dn) { if (a.da) a.da[col] = v; }
        else if (col < dn + a.D) { if (a.dskip) a.dskip[col - dn] = v; }
        else if (a.ddelta_bias) a.ddelta_bias[col - dn - a.D] = v;
    }
}

// One token: a wave takes CH channels of one row.  Bound by the states, read and written once: four of them a lane, in one
// load where N is a multiple of 4 (256 rows of 4096 channels with 16 states: 38 us, 3.8 TB/s; one row of 1024: 3.2 us, a
// chain of three loads).  Rows with one slot are taken in order by the first one's wave.  A wave lives for little
// more than its chain of dependent loads, so everything whose address does not depend on the slot is requested behind the
// slot's own load, and the states before the search for an earlier row with this slot.
// (QUADS is a template argument because the compiler joins the two ways of loading into one, by single values, else.)
template <typename X, int S, bool QUADS>
__global__ __launch_bounds__(64 * kWaves) void scan_step_kernel(tgru_scan_step_args a, int tpg, int tiles) {
    constexpr int CH = 64 / S;
    const int lane = threadIdx.x & 63, c = lane / S, s = lane % S;
    const unsigned id = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row0 = (int)(id / (unsigned)tiles), flat = (int)(id - (unsigned)row0 * (unsigned)tiles);
    if (row0 >= a.B) return;
    const int grp = flat / tpg, Dg = a.D / a.G, first = (flat - grp * tpg) * CH;
    const bool on = c < Dg - first;
    const int d = grp * Dg + first + (on ? c : 0);
    const int my_slot = a.slots ? a.slots[row0] : row0;
    __builtin_amdgcn_sched_barrier(0);
    const int n0 = min(4 * s, QUADS ? a.N - 4 : a.N - 1);               // parts without states read the last ones
    // four values of a row of N (zeros beyond it once they are unpacked)
    auto four = [&](const auto *p) {
        using E = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
        struct alignas(4 * sizeof(E)) Pack4 { E v[4]; } q;
        if constexpr (QUADS) {
            q = *reinterpret_cast<const Pack4 *>(p + n0);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) q.v[k] = p[min(4 * s + k, a.N - 1)];
        }
        return q;
    };
    auto spread = [&](const auto &q, float (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = 4 * s + k < a.N ? to_float(q.v[k]) : 0.f;
    };
    auto inputs = [&](int row) {
        struct { decltype(four((const X *)nullptr)) b, m; X u, delta, z; } in;
        in.u = static_cast<const X *>(a.u)[row * a.u_stride + d];
        in.delta = static_cast<const X *>(a.delta)[row * a.delta_stride + d];
        in.z = a.z ? static_cast<const X *>(a.z)[row * a.z_stride + d] : from_float<X>(0.f);
        in.b = four(static_cast<const X *>(a.b) + row * a.b_stride[0] + grp * a.b_stride[1]);
        in.m = four(static_cast<const X *>(a.c) + row * a.c_stride[0] + grp * a.c_stride[1]);
        return in;
    };
    const auto rates = four(a.a + (long)d * a.N);
    const float bias = a.delta_bias ? a.delta_bias[d] : 0.f, skip = a.skip ? a.skip[d] : 0.f;
    auto in = inputs(row0);
    __builtin_amdgcn_sched_barrier(0);
    const int slot = __builtin_amdgcn_readfirstlane(my_slot);
    if (slot < 0 || slot >= a.P) {
        if (on && s == 0) static_cast<X *>(a.y)[row0 * a.y_stride + d] = from_float<X>(0.f);
        return;
    }
    const long so = ((long)slot * a.D + d) * a.N;
    const auto state = four(a.state + so);
    __builtin_amdgcn_sched_barrier(0);       // on its way while the search waits for its own loads
    if (a.slots && find_slot(a.slots, 0, row0, slot) < row0) return;
    float h[4], a2[4];
    spread(state, h);
    spread(rates, a2);
#pragma unroll
    for (int k = 0; k < 4; ++k) a2[k] = finite_rate(a2[k]);
    for (int row = row0;;) {
        float b[4], m[4];
        spread(in.b, b);
        spread(in.m, m);
        const float u = to_float(in.u), raw = to_float(in.delta) + bias, z = to_float(in.z);
        const float dt = a.softplus ? softplus(raw) : raw, t = dt * kLog2e;
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = __builtin_fmaf(__builtin_amdgcn_exp2f(t * a2[k]), h[k], dt * u * b[k]);
            y = __builtin_fmaf(m[k], h[k], y);
        }
        y = __builtin_fmaf(skip, u, sum_parts<S>(y));
        if (a.z) y *= z * sigmoid(z);
        if (on && s == 0) static_cast<X *>(a.y)[row * a.y_stride + d] = from_float<X>(y);
        if (!a.slots) break;
        row = find_slot(a.slots, row + 1, a.B, slot);
        if (row >= a.B) break;
        in = inputs(row);
    }
    if (!on || 4 * s >= a.N) return;
    float *to = a.state_out + so + 4 * s;
    if constexpr (QUADS) {
        *reinterpret_cast<float4 *>(to) = make_float4(h[0], h[1], h[2], h[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (4 * s + k < a.N) to[k] = h[k];
    }
}

// States with padding: a power of two, 8 at least (with four a lane of scan_bwd_kernel would have too much of the work
// that is per channel in its registers).
int padded_states(int N) {
    int n = 8;
    while (n < N) n <<= 1;
    return n;
}

// What a pass of `waves` waves over `steps` steps takes, in us: cost[k - 1] is one step's time with k waves on each of the
// chip's 1024 SIMDs, of which it holds `most` -- so whole rounds of them and what is left over.
double pass_time(long waves, long steps, const double *cost, int most) {
    const long round = 1024L * most, rest = waves % round;
    return steps * (waves / round * cost[most - 1] + (rest ? cost[(rest + 1023) / 1024 - 1] : 0.));
}

// Chunks of time: the number that the times measured below give the shortest pass for.  A chunk more costs the main pass
// nothing but blocks cut short; the pass in front does more of its work again (all chunks but one), and with the joining
// costs two launches.  Measured with 16 states and sequences of full length (us a step), and used for all: fewer states a channel
// spill in the backward pass, and sequences of unequal length end before the time that is planned for.  One sequence more or less than a round matters most -- 14 and 16
// sequences (1792 and 2048 waves) of the backward pass take the same 503 us for 1024 steps, 20 take 708.
Plan make_plan(int B, int T, int D, int N, int G, bool backward) {
    Plan p;
    p.NP = padded_states(N);
    p.CH = 256 / p.NP;
    p.Dg = D / G;
    p.tpg = (p.Dg + p.CH - 1) / p.CH;
    p.tiles = p.tpg * G;
    p.wpg = (p.tpg + kWaves - 1) / kWaves;
    p.nblk = (T + Q - 1) / Q;
    p.quads = 0;
    static const double fwd[] = {.133, .165, .21, .30}, fwd_front[] = {.09, .124, .165, .225}, bwd[] = {.36, .503},
                        bwd_front[] = {.10, .135, .185, .26};
    const long waves = (long)B * p.tiles;
    double best = 0.;
    p.nchunks = 1;
    p.chunk = p.nblk * Q;
    for (int n = 1; n <= 128 && n <= p.nblk; n += n < 8 ? 1 : n / 4) {
        const int chunk = (p.nblk + n - 1) / n * Q, real = (T + chunk - 1) / chunk;
        double time = backward ? pass_time(waves * real, chunk, bwd, 2) : pass_time(waves * real, chunk, fwd, 4);
        if (real > 1) time += 10. + pass_time(waves * (real - 1), chunk, backward ? bwd_front : fwd_front, 4);
        if (n > 1 && time >= best) continue;
        best = time;
        p.nchunks = real;
        p.chunk = chunk;
    }
    return p;
}

int scan_dims(int B, int T, int D, int N, int G) {
    if (B <= 0 || T <= 0 || D <= 0 || N <= 0 || G <= 0 || N > TGRU_SCAN_MAX_STATES || D % G) return TGRU_E_DIMS;
    if (T > (1 << 30) || D >= kMaxRowStride) return TGRU_E_DIMS;
    // a launch holds less than 2^32 threads, and offsets within one sequence's maps or state are 32-bit numbers
    for (bool backward : {false, true}) {
        const Plan p = make_plan(B, T, D, N, G, backward);
        if ((double)B * p.nchunks * G * p.wpg * 64 * kWaves >= 4294967296.0 || (double)T * p.NP >= 2147483648.0 ||
            (double)D * p.NP >= 2147483648.0 || (p.nchunks > 1 && (double)B * D * p.NP >= 4294967232.0))
            return TGRU_E_DIMS;
    }
    return TGRU_OK;
}

size_t ckpt_floats(const Plan &p, int B, int D) { return (size_t)B * p.nblk * D * p.NP; }

struct Workspace { size_t carry, sdt, map, par, total; };       // offsets in floats, each a multiple of 4
Workspace workspace_of(const Plan &p, int B, int T, int D, int N, int G, bool backward) {
    Workspace w;
    size_t off = 0;
    auto take = [&](size_t n) { const size_t at = off; off += (n + 3) & ~(size_t)3; return at; };
    w.carry = take(p.nchunks > 1 ? (size_t)B * p.nchunks * D * p.NP : 0);
    w.sdt = take(p.nchunks > 1 ? (size_t)B * p.nchunks * D : 0);
    w.map = take(backward ? (size_t)B * G * p.wpg * T * 2 * p.NP : 0);
    w.par = take(backward ? (size_t)B * p.nchunks * D * (N + 2) : 0);
    w.total = off;
    return w;
}

#define TGRU_DONE() do { if (hipGetLastError() != hipSuccess) return TGRU_E_LAUNCH; } while (0)

template <typename X, int S>
int run_scan(const tgru_scan_args &a, bool backward, hipStream_t s) {
    Plan pl = make_plan(a.B, a.T, a.D, a.N, a.G, backward);
    auto quads = [&](const void *p, const int64_t *st) {
        return (uintptr_t)p % (4 * sizeof(X)) == 0 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
    };
    pl.quads = a.N % 4 == 0 && quads(a.b, a.b_stride) && quads(a.c, a.c_stride);
    const Workspace ws = workspace_of(pl, a.B, a.T, a.D, a.N, a.G, backward);
    float *carry = a.workspace + ws.carry, *sdt = a.workspace + ws.sdt;
    const dim3 run((unsigned)(((long)a.B * pl.nchunks * pl.tiles + kWaves - 1) / kWaves)), block(64 * kWaves);
    const dim3 join((unsigned)(((long)a.B * a.D * pl.NP + 63) / 64));
    if (!backward) {
        if (pl.nchunks > 1) {
            TGRU_LAUNCH((scan_fwd_kernel<X, S, 1>), run, block, 0, s, a, pl, carry, sdt);
            TGRU_DONE();
            TGRU_LAUNCH(scan_join_kernel, join, dim3(64), 0, s, a.a, a.initial_state, pl, a.B, a.D, a.N, 0, carry, sdt);
            TGRU_DONE();
        }
        TGRU_LAUNCH((scan_fwd_kernel<X, S, 0>), run, block, 0, s, a, pl, carry, sdt);
        TGRU_DONE();
        return TGRU_OK;
    }
    const dim3 grid((unsigned)((long)a.B * pl.nchunks * a.G * pl.wpg));
    float *map = (a.db || a.dc) ? a.workspace + ws.map : nullptr;
    float *par = (a.da || a.dskip || a.ddelta_bias) ? a.workspace + ws.par : nullptr;
    if (pl.nchunks > 1) {
        TGRU_LAUNCH((scan_back_kernel<X, S>), run, block, 0, s, a, pl, carry, sdt);
        TGRU_DONE();
        TGRU_LAUNCH(scan_join_kernel, join, dim3(64), 0, s, a.a, a.dfinal, pl, a.B, a.D, a.N, 1, carry, sdt);
        TGRU_DONE();
    }
    TGRU_LAUNCH((scan_bwd_kernel<X, S>), grid, block, 0, s, a, pl, carry, map, par);
    TGRU_DONE();
    if (map || par) {
        // (workgroups beyond these numbers take turns)
        const unsigned maps = map ? (unsigned)std::min<long>(((long)a.B * a.G * a.T * pl.NP / 2 + 255) / 256, 1 << 18) : 0;
        const unsigned pars = par ? (unsigned)std::min<long>(((long)a.D * (a.N + 2) + 31) / 32, 1 << 17) : 0;
        TGRU_LAUNCH((scan_grads_kernel<X>), dim3(maps + pars), dim3(256), 0, s, a, pl, map, maps, par);
        TGRU_DONE();
    }
    return TGRU_OK;
}

template <typename X>
int run_scan_states(const tgru_scan_args &a, bool backward, hipStream_t s) {
    switch (padded_states(a.N)) {
    case 8: return run_scan<X, 2>(a, backward, s);
    case 16: return run_scan<X, 4>(a, backward, s);
    case 32: return run_scan<X, 8>(a, backward, s);
    default: return run_scan<X, 16>(a, backward, s);
    }
}

int scan_call(const tgru_scan_args *a, bool backward, hipStream_t s) {
    if (!a) return TGRU_E_NULL;
    if (int rc = scan_dims(a->B, a->T, a->D, a->N, a->G)) return rc;
    if (!known_dtype(a->dtype)) return TGRU_E_DTYPE;
    if (!a->u || !a->delta || !a->b || !a->c || !a->a) return TGRU_E_NULL;
    if (backward ? !a->reserve || (a->dz && !a->z) : !a->y) return TGRU_E_NULL;
    if (!a->workspace && tgru_scan_workspace_bytes(a->B, a->T, a->D, a->N, a->G, backward)) return TGRU_E_NULL;
    auto wide = [](const void *p, const int64_t *stride) { return p && (stride[1] < 0 || stride[1] >= kMaxRowStride); };
    if (wide(a->u, a->u_stride) || wide(a->delta, a->delta_stride) || wide(a->z, a->z_stride) || wide(a->b, a->b_stride) ||
        wide(a->c, a->c_stride) || wide(a->y, a->y_stride) || wide(a->dy, a->dy_stride) || wide(a->du, a->du_stride) ||
        wide(a->ddelta, a->ddelta_stride) || wide(a->dz, a->dz_stride))
        return TGRU_E_DIMS;
    if (((uintptr_t)a->reserve & 15) || ((uintptr_t)a->workspace & 15)) return TGRU_E_ALIGN;
    if (int rc = check_device()) return rc;
    if (a->dtype == TGRU_DTYPE_F32) return run_scan_states<float>(*a, backward, s);
    if (a->dtype == TGRU_DTYPE_BF16) return run_scan_states<__bf16>(*a, backward, s);
    return run_scan_states<_Float16>(*a, backward, s);
}

// Waves a group of the one-token form, of CH channels each.
int step_tiles(int D, int G, int CH) { return (D / G - 1) / CH + 1; }

template <typename X, int S>
int run_scan_step(const tgru_scan_step_args &a, hipStream_t s) {
    const int tpg = step_tiles(a.D, a.G, 64 / S), tiles = tpg * a.G;
    auto ok = [](const void *p, size_t align) { return (uintptr_t)p % align == 0; };
    const bool quads = a.N % 4 == 0 && ok(a.state, 16) && ok(a.state_out, 16) && ok(a.a, 16) && ok(a.b, 4 * sizeof(X)) &&
                      ok(a.c, 4 * sizeof(X)) && a.b_stride[0] % 4 == 0 && a.b_stride[1] % 4 == 0 && a.c_stride[0] % 4 == 0 &&
                      a.c_stride[1] % 4 == 0;
    const dim3 grid((unsigned)(((long)a.B * tiles + kWaves - 1) / kWaves)), block(64 * kWaves);
    if (quads) TGRU_LAUNCH((scan_step_kernel<X, S, true>), grid, block, 0, s, a, tpg, tiles);
    else TGRU_LAUNCH((scan_step_kernel<X, S, false>), grid, block, 0, s, a, tpg, tiles);
    TGRU_DONE();
    return TGRU_OK;
}

template <typename X>
int run_scan_step_lanes(const tgru_scan_step_args &a, hipStream_t s) {
    int S = 1;
    while (4 * S < a.N) S <<= 1;
    switch (S) {
    case 1: return run_scan_step<X, 1>(a, s);
    case 2: return run_scan_step<X, 2>(a, s);
    case 4: return run_scan_step<X, 4>(a, s);
    case 8: return run_scan_step<X, 8>(a, s);
    default: return run_scan_step<X, 16>(a, s);
    }
}

}  // namespace ssm
}  // namespace tgru

using namespace tgru::ssm;

extern "C" {

size_t tgru_scan_reserve_bytes(int B, int T, int D, int N, int G) {
    if (scan_dims(B, T, D, N, G) != TGRU_OK) return 0;
    return ckpt_floats(make_plan(B, T, D, N, G, false), B, D) * sizeof(float);
}

size_t tgru_scan_workspace_bytes(int B, int T, int D, int N, int G, int backward) {
    if (scan_dims(B, T, D, N, G) != TGRU_OK) return 0;
    return workspace_of(make_plan(B, T, D, N, G, backward != 0), B, T, D, N, G, backward != 0).total * sizeof(float);
}

int tgru_scan_forward(const tgru_scan_args *a, tgru_stream_t stream) { return scan_call(a, false, (hipStream_t)stream); }
int tgru_scan_backward(const tgru_scan_args *a, tgru_stream_t stream) { return scan_call(a, true, (hipStream_t)stream); }

int tgru_scan_step(const tgru_scan_step_args *a, tgru_stream_t stream) {
    if (!a) return TGRU_E_NULL;
    if (a->B <= 0 || a->P <= 0 || a->D <= 0 || a->N <= 0 || a->G <= 0 || a->N > TGRU_SCAN_MAX_STATES || a->D % a->G) return TGRU_E_DIMS;
    if (!a->slots && a->P < a->B) return TGRU_E_DIMS;
    // less than 2^32 threads
    const int tpg = step_tiles(a->D, a->G, 256 / (a->N <= 4 ? 4 : padded_states(a->N)));
    if ((double)a->B * tpg * a->G >= 67108860.0 || search_too_long(a->slots, a->B, (long)tpg * a->G)) return TGRU_E_DIMS;
    if (!known_dtype(a->dtype)) return TGRU_E_DTYPE;
    if (!a->u || !a->delta || !a->b || !a->c || !a->a || !a->state || !a->state_out || !a->y) return TGRU_E_NULL;
    if (int rc = tgru::check_device()) return rc;
    if (a->dtype == TGRU_DTYPE_F32) return run_scan_step_lanes<float>(*a, (hipStream_t)stream);
    if (a->dtype == TGRU_DTYPE_BF16) return run_scan_step_lanes<__bf16>(*a, (hipStream_t)stream);
    return run_scan_step_lanes<_Float16>(*a, (hipStream_t)stream);
}

}  // extern "C"
