// selective.hip — selective state space scan along each sequence (ray), forward, backward and one row at a time, for gfx950.
//
//   step = softplus(delta + bias),  h[t] = exp(step A) h[t-1] + step B[t] u[t],  y[t] = C[t] . h[t] + D u[t],  out = y silu(gate)
//
// What bounds it: per (row, channel, state) one exponential (a quarter-rate instruction) and four full-rate ones, against 2-4 bytes per
// (row, channel) and tensor: with 16 states the vector units need two to three times as long as memory.  So a lane keeps as many of a
// channel's states as registers allow (up to 16, P lanes per channel beyond that), everything per (row, channel) — softplus, gate,
// loads — is shared by them, B[t] and C[t] come from LDS as broadcasts, and the loads of the next eight rows are in flight meanwhile.
//
// A wave owns 64 / P channels of one sequence and walks its rows: no hand-off, no atomics.  Where the sequences are too few for the
// chip, they are cut into chunks: a first pass leaves what each chunk adds to the state and the sum of its steps (its decay is
// exp(A sum)), a short pass chains the chunks, and the main pass starts every chunk from its state.
//
// Backward: h is formed again from states the forward pass left every eight rows (any place of a row grid holds the start of at most
// one such eighth, because sequences do not overlap: slot = row / 8 needs no table).  With G = dL/dh,  G[t] = C[t] dy[t] +
// exp(step[t+1] A) G[t+1]:
//   dC = sum_d dy h,  dB = sum_d G step u,  du = step sum_s G B + D dy,  dstep = sum_s G (A a h[t-1] + B u),  dA = sum_t G step a h[t-1].
// The sums over channels are exchanged across lanes (halving the values at every step, as long as there are two: 16 values over 32 lanes
// take 8 + 4 + 2 + 1 + 1 exchanges); the sums over rows stay in registers over all rows of a wave; both are joined in a fixed order.
//
// On one MI355X, kernels alone, 16 states: 2^18 rows of 64 channels in 4096 ragged rays, bf16: forward 126 us with the kept states (144
// vector instructions per row and wave, 91 % of the CUs' busy cycles), backward 348 us (267 instructions, 84 %) + 18 + 9 to join; memory
// would take 49 us for all of it at 6.2 TB/s.  32768 rows of 1024 channels, one sequence, bf16: 287 us in all (124 + 37 + 156 profiled).  Two
// sequences of 8192 rows of 512 channels, fp32: forward 39 + 20 + 53 us, backward 47 + 14 + 167 + 14.  One row of 256 rays of 1024 channels:
// 8.3 us (35 MB, 4.3 TB/s).
#include "feature.hpp"

#include <algorithm>

namespace nfa {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 8;                // rows between kept states, and rows whose loads are in flight together
constexpr int64_t kMaxStride = 1 << 25; // elements: sixteen rows of four bytes are 2^31 bytes apart at most

struct ScanArgs {
    const void *u, *dt, *z, *B, *C, *gy;
    int64_t ld_u, ld_dt, ld_z, ld_B, ld_C, ld_gy;
    const float *A, *D, *bias, *init, *gfinal;
    const int64_t *info;
    const int32_t *ray, *pos, *order;
    void *y, *gu, *gdt, *gz;
    float *final_state, *kept, *ginit;
    float *ends, *sums;                 // chunks: [slots][states][channels], [slots][channels]
    float *part_bc;                     // backward: [groups of channel blocks][rows][2][padded states]
    float *part_w;                      // backward: [workers][channels * states + 2 * channels]
    int64_t rows, n_rays, length, chunk, chunks, slots, tasks, workers;
    int32_t channels, states, softplus, blocks, groups;
};
// Channel blocks that a wave of the backward pass takes one after the other, summing their dB and dC in memory.  A block's channels are
// 64 / P, so that partial sums of every block would be as large as all of h (34 GB at 32768 rows of 1024 channels of 256 states, whose
// states kept every eight rows take 4.3): so they are as large as the kept states, at most.  8192 rows of 512 channels of 128 states: 289 MiB
// of workspace and 1.79 ms, 1033 and 1.51 with partial sums of every block; up to 32 states every block has its own.
constexpr int blocks_of_wave(int p) { return p > 4 ? p / 4 : 1; }

// a task: a run of rows of one sequence
struct Task { int64_t ray, start, count, first, n, slot; bool live; };      // sequence rows [start, start + count), the task's [first, first + n) of it

__device__ __forceinline__ void sequence_rows(const ScanArgs &a, int64_t ray, int64_t &start, int64_t &count) {
    if (!a.info) { start = ray * a.length; count = a.length; return; }
    start = readfirstlane_i64(a.info[2 * ray]);
    count = readfirstlane_i64(a.info[2 * ray + 1]);
    if (start < 0) { count += start; start = 0; }
    if (start > a.rows) start = a.rows;
    if (count < 0) count = 0;
    if (count > a.rows - start) count = a.rows - start;
}
// chunk k >= 1 of a sequence begins `chunk` rows behind the one before it, so no two of them begin in the same block of `chunk` rows
__device__ __forceinline__ int64_t chunk_slot(const ScanArgs &a, int64_t ray, int64_t first, int64_t k) {       // first: start / chunk
    return k == 0 ? a.slots - a.n_rays + ray : first + k;
}

__device__ __forceinline__ Task find_task(const ScanArgs &a, int64_t id, int lane) {
    Task t;
    int64_t k = 0;
    t.live = true;
    if (a.chunk == 0) t.ray = a.order ? __builtin_amdgcn_readfirstlane(a.order[id]) : id;
    else if (!a.info) { t.ray = id / a.chunks; k = id - t.ray * a.chunks; }
    else if (id < a.n_rays) t.ray = id;
    else {                              // the chunk that begins inside block id - n_rays, if one does
        const int64_t base = (id - a.n_rays) * a.chunk;
        t.live = false;
        t.ray = 0;
        for (int64_t r = base; r < base + a.chunk && r < a.rows; r += kWave) {
            const int64_t row = r + lane;
            int32_t p = -1;
            if (row < base + a.chunk && row < a.rows) p = a.pos[row];
            const unsigned long long hit = __ballot(p > 0 && p % (int32_t)a.chunk == 0);
            if (hit) {
                const int src = __ffsll((long long)hit) - 1;
                k = __builtin_amdgcn_readlane(p, src) / (int32_t)a.chunk;
                t.ray = __builtin_amdgcn_readfirstlane(a.ray[r + src]);
                t.live = true;
                break;
            }
        }
        if (!t.live) { t.start = t.count = t.first = t.n = t.slot = 0; return t; }
    }
    sequence_rows(a, t.ray, t.start, t.count);
    t.first = k * a.chunk;
    t.n = t.count - t.first;
    if (a.chunk && t.n > a.chunk) t.n = a.chunk;
    if (t.n < 0) t.n = 0;
    t.slot = a.chunk ? chunk_slot(a, t.ray, t.start / a.chunk, k) : 0;
    if (k > 0 && t.n == 0) t.live = false;
    return t;
}

// exchanges the upper half (odd rows) of `a` with the lower half (even rows) of `b` in one instruction and adds: with a = b every lane
// gets its pair's sum, with two values lanes without the bit get a's sum and lanes with it b's
template <int BIT>
__device__ __forceinline__ float swap_add(float a, float b) {
    const unsigned i = __builtin_bit_cast(unsigned, a), j = __builtin_bit_cast(unsigned, b);
    unsigned x, y;                                          // (elements by value: a bit cast of an element takes the first one)
    if constexpr (BIT == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(i, j, false, false);
        x = r[0], y = r[1];
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(i, j, false, false);
        x = r[0], y = r[1];
    }
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}
// the value of the lane whose number differs in BIT
template <int BIT>
__device__ __forceinline__ float other_lane(float v) {
    if constexpr (BIT == 8) return dpp_f<0x128>(0.0f, v);                                    // row_ror:8
    else if constexpr (BIT == 4) return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x101f));   // xor 4
    else if constexpr (BIT == 2) return dpp_f<0x4e>(0.0f, v);                                // quad_perm [2, 3, 0, 1]
    else return dpp_f<0xb1>(0.0f, v);                                                        // quad_perm [1, 0, 3, 2]
}
template <int BIT>
__device__ __forceinline__ float add_other(float v) {
    if constexpr (BIT >= 16) return swap_add<BIT>(v, v);
    else return v + other_lane<BIT>(v);
}
// two values summed over the lane pair that differs in BIT: lanes without the bit get v0's sum, lanes with it v1's
template <int BIT>
__device__ __forceinline__ float halve(float v0, float v1, int lane) {
    if constexpr (BIT >= 16) {
        return swap_add<BIT>(v0, v1);
    } else {
        const bool up = lane & BIT;
        return (up ? v1 : v0) + other_lane<BIT>(up ? v0 : v1);
    }
}
// sums v[0 .. CNT) over the lanes that differ in the bits BIT, BIT / 2, ... 1; afterwards v[0 .. left) holds the values
// that number_of() names
template <int CNT, int BIT>
__device__ __forceinline__ void sum_over_lanes(float *v, int lane) {
    if constexpr (BIT > 0) {
        if constexpr (CNT > 1) {
#pragma unroll
            for (int i = 0; i < CNT / 2; ++i) v[i] = halve<BIT>(v[2 * i], v[2 * i + 1], lane);
            sum_over_lanes<CNT / 2, BIT / 2>(v, lane);
        } else {
            v[0] = add_other<BIT>(v[0]);
            sum_over_lanes<1, BIT / 2>(v, lane);
        }
    }
}
constexpr int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v / 2); }

// sum over the P lanes of a channel (lane = part * (64 / P) + channel)
template <int P>
__device__ __forceinline__ float sum_parts(float v) {
    if constexpr (P >= 2) v = add_other<32>(v);
    if constexpr (P >= 4) v = add_other<16>(v);
    if constexpr (P >= 8) v = add_other<8>(v);
    if constexpr (P >= 16) v = add_other<4>(v);
    if constexpr (P >= 32) v = add_other<2>(v);
    return v;
}

// column c of row `row` + r: one scalar base per tensor, a 32-bit offset from it (row strides are at most kMaxStride)
template <class T>
__device__ __forceinline__ T row_at(const void *base, int64_t row, int64_t ld, uint32_t r, uint32_t c) {
    return *reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + row * ld * (int64_t)sizeof(T) + (r * (uint32_t)ld + c) * (uint32_t)sizeof(T));
}

// What a wave has in hand: eight rows' numbers, each replaced by those of the row eight further on as soon as it is used, so that one set
// of registers keeps eight rows of loads in flight.  Rows and bases are the same in all lanes (scalar registers); lanes without a channel
// read the last one's, rows beyond the end the end's, so that no load has a branch.
template <class T, int NS, int P, bool HAS_U, bool HAS_C, bool HAS_Z, bool HAS_G>
struct Rows {
    static constexpr int SP = NS * P, kStates = (kTile * SP + kWave - 1) / kWave;
    T u[HAS_U ? kTile : 1], dt[kTile], z[HAS_Z ? kTile : 1], g[HAS_G ? kTile : 1];
    T b[kStates], c[HAS_C ? kStates : 1];

    // row base + r into place j
    __device__ __forceinline__ void load_row(const ScanArgs &a, int j, int64_t base, uint32_t r, uint32_t ch) {
        if (HAS_U) u[j] = row_at<T>(a.u, base, a.ld_u, r, ch);
        dt[j] = row_at<T>(a.dt, base, a.ld_dt, r, ch);
        if (HAS_G) g[j] = row_at<T>(a.gy, base, a.ld_gy, r, ch);
        if (HAS_Z && a.z) z[j] = row_at<T>(a.z, base, a.ld_z, r, ch);
    }
    // the n rows from `row` on: B and C
    __device__ __forceinline__ void load_states(const ScanArgs &a, int64_t row, int n, int lane) {
#pragma unroll
        for (int k = 0; k < kStates; ++k) {
            const int e = k * kWave + lane, s = e % SP;
            const uint32_t t = e / SP < n ? e / SP : n - 1, sc = s < a.states ? s : 0;
            b[k] = row_at<T>(a.B, row, a.ld_B, t, sc);
            if (HAS_C) c[k] = row_at<T>(a.C, row, a.ld_C, t, sc);
        }
    }
    // B and C into this wave's LDS: [2][kTile][SP]
    __device__ __forceinline__ void stage(const ScanArgs &a, float *lds, int lane) const {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < kStates; ++k) {
            const int e = k * kWave + lane;
            if (e < kTile * SP) {
                lds[e] = e % SP < a.states ? to_f(b[k]) : 0.0f;
                if (HAS_C) lds[kTile * SP + e] = e % SP < a.states ? to_f(c[k]) : 0.0f;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};

// Places behind the last state have A = B = C = 0 and stay 0 by themselves, unless their row holds an infinity (0 infinity is NaN, and would
// join the sums over states).  Forward such rows take a loop that keeps them 0 (`size` is finite where the row's numbers are): 12 states of
// 2^18 rows of 64 channels take 91 us, 106 with the test for every state in every row, 86 without any.  Backward the test is for every
// state: 362 us, 375 with two loops, 340 without any.
template <bool MASKED>
__device__ __forceinline__ float only_states(const ScanArgs &a, int s, float v) { return !MASKED || s < a.states ? v : 0.0f; }
template <bool PADDED, class F>
__device__ __forceinline__ void with_mask(float size, F &&f) {
    if (PADDED && __any(!(fabsf(size) < __builtin_inff()))) f(std::bool_constant<PADDED>{});
    else f(std::false_type{});
}

// y + D u; without D nothing: 0 u would be NaN for an infinite u
__device__ __forceinline__ float add_skip(const ScanArgs &a, float D, float u, float y) { return a.D ? fmaf(D, u, y) : y; }

// softplus and its derivative from one exponential
struct Step { float step, slope; };
__device__ __forceinline__ Step softplus_step(float raw) {
    const float e = fast_exp2(-fabsf(raw) * kLog2e), r = fast_rcp(1.0f + e);
    return {softplus_from(raw, e), raw >= 0.0f ? r : e * r};
}

template <int NS> __device__ __forceinline__ void read_states(const float *at, float (&v)[NS]) {
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = at[i];
}

// main pass (LOCAL = false): outputs, kept states, final state; first pass over chunks (LOCAL): what a chunk adds, and its steps' sum.
// The vector units bound both: 89 us over 2^18 rows of 64 channels (2.7e8 states, 3.0e12 of them a second), 39 us the first pass
// over 16384 rows of 512 channels.
template <class T, int NS, int P, bool PADDED, bool LOCAL>
__global__ __launch_bounds__(kWave) void scan_fwd_kernel(ScanArgs a) {
    constexpr int SP = NS * P, CH = kWave / P;
    __shared__ __attribute__((aligned(16))) float lds[2 * kTile * SP];
    const int lane = lane_id(), part = lane / CH;
    const int64_t id = blockIdx.x;
    const int64_t task = id / a.blocks;
    if (task >= a.tasks) return;
    const uint32_t ch = (uint32_t)(id - task * a.blocks) * CH + lane % CH, last = a.channels - 1, chc = ch < last ? ch : last;
    const bool on = ch <= last;
    const Task t = find_task(a, task, lane);
    if (!t.live) return;
    float A2[NS], h[NS];
    const float D = on && a.D ? a.D[ch] : 0.0f, bias = on && a.bias ? a.bias[ch] : 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = part * NS + i;
        const bool here = on && s < a.states;
        A2[i] = here ? a.A[ch * a.states + s] * kLog2e : 0.0f;
        h[i] = 0.0f;
        if (!LOCAL && here) {
            if (a.chunk) h[i] = a.ends[(t.slot * a.states + s) * a.channels + ch];
            else if (a.init) h[i] = a.init[(t.ray * a.channels + ch) * a.states + s];
        }
    }
    Rows<T, NS, P, true, !LOCAL, !LOCAL, false> rows;
    const int64_t row0 = t.start + t.first;
    const int total = (int)t.n;
    if (total > 0) {
#pragma unroll
        for (int j = 0; j < kTile; ++j) rows.load_row(a, j, row0, j < total ? j : total - 1, chc);
        rows.load_states(a, row0, total < kTile ? total : kTile, lane);
    }
    for (int k = 0; k < total; k += kTile) {
        rows.stage(a, lds, lane);
        const int n = total - k < kTile ? total - k : kTile, more = total - k - kTile;
        if (more > 0) rows.load_states(a, row0 + k + kTile, more < kTile ? more : kTile, lane);
        if (!LOCAL && a.kept && t.first + k > 0) {
            float *to = a.kept + ((row0 + k) / kTile) * a.states * a.channels;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int s = part * NS + i;
                if (on && s < a.states) to[(int64_t)s * a.channels + ch] = h[i];
            }
        }
#pragma unroll
        for (int j = 0; j < kTile; ++j) {
            if (j >= n) break;
            const float u = to_f(rows.u[j]);
            float step = to_f(rows.dt[j]) + bias;
            if (a.softplus) step = softplus_f(step);
            const float in = step * u;
            float B[NS], C[NS], y = 0.0f;
            read_states<NS>(lds + j * SP + part * NS, B);
            if (!LOCAL) read_states<NS>(lds + (kTile + j) * SP + part * NS, C);
            sum += step;
            with_mask<PADDED>(in, [&](auto masked) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    h[i] = only_states<masked()>(a, part * NS + i, fmaf(fast_exp2(step * A2[i]), h[i], in * B[i]));
                    if (!LOCAL) y = fmaf(C[i], h[i], y);
                }
            });
            if (!LOCAL) {
                y = add_skip(a, D, u, sum_parts<P>(y));
                if (a.z) {
                    const float z = to_f(rows.z[j]);
                    y *= z * sigmoid_f(z);
                }
                if (on && part == 0) (reinterpret_cast<T *>(a.y) + (row0 + k + j) * a.channels)[ch] = from_f<T>(y);
            }
            if (more > 0) rows.load_row(a, j, row0 + k, kTile + (j < more ? j : more - 1), chc);
        }
    }
    if (LOCAL) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int s = part * NS + i;
            if (on && s < a.states) a.ends[(t.slot * a.states + s) * a.channels + ch] = h[i];
        }
        if (on && part == 0) a.sums[t.slot * a.channels + ch] = sum;
    } else if (a.final_state && t.first + t.n == t.count) {
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int s = part * NS + i;
            if (on && s < a.states) a.final_state[(t.ray * a.channels + ch) * a.states + s] = h[i];
        }
    }
}

// chunk by chunk, a lane per (channel, state): ends[slot] becomes the state that the chunk starts from (REV: the gradient that
// reaches its last row from behind), from what each chunk adds on its own.  One dependent product-sum after the other, 32 chunks' loads
// in flight: latency bounds it, about 0.1 us a chunk (512 chunks of 1024 channels 37 us).
template <bool REV>
__global__ __launch_bounds__(kBlock) void scan_chain_kernel(ScanArgs a) {
    const int64_t per = (int64_t)a.channels * a.states;
    const int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x, ray = blockIdx.y;
    if (e >= per) return;
    const int64_t s = e / a.channels, ch = e - s * a.channels;
    int64_t start, count;
    sequence_rows(a, ray, start, count);
    const float A2 = a.A[ch * a.states + s] * kLog2e;
    const float *from = REV ? a.gfinal : a.init;
    float h = from ? from[(ray * a.channels + ch) * a.states + s] : 0.0f;
    const int64_t chunks = count > 0 ? (count + a.chunk - 1) / a.chunk : 1, first = start / a.chunk;
    constexpr int kAhead = 32;                              // chunks in flight: the chain itself is one fma each
    for (int64_t k0 = 0; k0 < chunks; k0 += kAhead) {
        // A chunk's decay may be beyond 32 bits where no row's is (growing states), and what it meets may be 0 or tiny: it is applied as two
        // powers of two, the second 1 for all that fit one, and never to 0.
        float add[kAhead], decay[kAhead], more[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int64_t k = k0 + i < chunks ? k0 + i : chunks - 1, slot = chunk_slot(a, ray, first, REV ? chunks - 1 - k : k);
            add[i] = a.ends[(slot * a.states + s) * a.channels + ch];
            const float e = a.sums[slot * a.channels + ch] * A2, one = fminf(fmaxf(e, -126.0f), 126.0f);
            decay[i] = fast_exp2(one);
            more[i] = fast_exp2(e - one);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (k0 + i >= chunks) break;
            const int64_t k = k0 + i, slot = chunk_slot(a, ray, first, REV ? chunks - 1 - k : k);
            a.ends[(slot * a.states + s) * a.channels + ch] = h;
            h = h == 0.0f ? add[i] : fmaf(decay[i], h * more[i], add[i]);
        }
    }
}

// the gradient that a chunk adds at its first row, and its steps' sum: 47 us for 16384 rows of 512 channels, the vector units' time
template <class T, int NS, int P, bool PADDED>
__global__ __launch_bounds__(kWave) void scan_bwd_local_kernel(ScanArgs a) {
    constexpr int SP = NS * P, CH = kWave / P;
    __shared__ __attribute__((aligned(16))) float lds[2 * kTile * SP];
    const int lane = lane_id(), part = lane / CH;
    const int64_t id = blockIdx.x;
    const int64_t task = id / a.blocks;
    if (task >= a.tasks) return;
    const uint32_t ch = (uint32_t)(id - task * a.blocks) * CH + lane % CH, last = a.channels - 1, chc = ch < last ? ch : last;
    const bool on = ch <= last;
    const Task t = find_task(a, task, lane);
    if (!t.live) return;
    float A2[NS], G[NS], sum = 0.0f;
    const float bias = on && a.bias ? a.bias[ch] : 0.0f;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = part * NS + i;
        A2[i] = on && s < a.states ? a.A[ch * a.states + s] * kLog2e : 0.0f;
        G[i] = 0.0f;
    }
    const int64_t row0 = t.start + t.first, tiles = (t.n + kTile - 1) / kTile;
    Rows<T, NS, P, false, true, true, true> rows;
    auto rows_in = [&](int64_t k) { const int64_t r = t.n - k * kTile; return (int)(r < kTile ? r : kTile); };
    if (tiles > 0) {
        const int64_t row = row0 + (tiles - 1) * kTile;
        const int n = rows_in(tiles - 1);
#pragma unroll
        for (int j = 0; j < kTile; ++j) rows.load_row(a, j, row, j < n ? j : n - 1, chc);
        rows.load_states(a, row, n, lane);
    }
    for (int64_t k = tiles - 1; k >= 0; --k) {
        const int n = rows_in(k);
        const int64_t before = row0 + (k - 1) * kTile;
        rows.stage(a, lds, lane);
        if (k > 0) rows.load_states(a, before, kTile, lane);
#pragma unroll
        for (int j = kTile - 1; j >= 0; --j) {
            float step = to_f(rows.dt[j]) + bias, dy = to_f(rows.g[j]), z = 0.0f;
            if (a.z) z = to_f(rows.z[j]);
            if (k > 0) rows.load_row(a, j, before, j, chc);
            if (j >= n) continue;
            if (a.softplus) step = softplus_f(step);
            if (a.z) dy *= z * sigmoid_f(z);
            float C[NS];
            read_states<NS>(lds + (kTile + j) * SP + part * NS, C);
            sum += step;
            with_mask<PADDED>(fabsf(step) + fabsf(dy), [&](auto masked) {
#pragma unroll
                for (int i = 0; i < NS; ++i) G[i] = only_states<masked()>(a, part * NS + i, fmaf(C[i], dy, G[i]) * fast_exp2(step * A2[i]));
            });
        }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int s = part * NS + i;
        if (on && s < a.states) a.ends[(t.slot * a.states + s) * a.channels + ch] = G[i];
    }
    if (on && part == 0) a.sums[t.slot * a.channels + ch] = sum;
}

// The backward main pass.  A tile of eight rows at a time, from the last to the first: the lanes of a channel share the rows' own
// numbers (step and its slope, dy, ...: each lane forms them for 8 / P rows) through LDS, which also keeps h before each row; so a lane's
// registers hold one row, the loops stay loops (the body is several hundred instructions), and LDS (20 KiB a wave with sixteen states:
// eight waves on a CU) sets how many waves a CU holds.  The vector units bound it: 348 us for 2^18 rows of 64 channels, 267 instructions
// per row and wave.
template <class T, int NS, int P, bool PADDED>
__global__ __launch_bounds__(kWave) void scan_bwd_kernel(ScanArgs a) {
    constexpr int SP = NS * P, CH = kWave / P, PR = P < kTile ? kTile / P : 1, kStates = (kTile * SP + kWave - 1) / kWave;
    __shared__ f32x4 hist[kTile - 1][NS / 4][kWave];        // h after row j; before row 0 it stays in registers
    __shared__ __attribute__((aligned(16))) float bc[2][kTile * SP];
    __shared__ float own_rows[5][kTile][CH];                // step, u, slope, dy, dL/dy of the gate; later du, dstep, dgate
    enum { kStep, kU, kSlope, kDy, kGate };
    constexpr int EACH = blocks_of_wave(P);
    const int lane = lane_id(), part = lane / CH, col = lane % CH;
    const int64_t id = blockIdx.x;
    const int64_t worker = id / a.groups;
    if (worker >= a.workers) return;
    const int group = (int)(id - worker * a.groups);
    // after the exchange over channels: this lane's values, their places, and whether it is the one that stores them
    constexpr int kBits = log2_of(CH), kHalvings = kBits < log2_of(2 * NS) ? kBits : log2_of(2 * NS), kLeft = 2 * NS >> kHalvings;
    int number = 0;
#pragma unroll
    for (int i = 0; i < kHalvings; ++i) number |= ((lane >> (kBits - 1 - i)) & 1) << i;
    const bool stores = (lane & ((1 << (kBits - kHalvings)) - 1)) == 0;

    for (int block = group * EACH; block < (group + 1) * EACH && block < a.blocks; ++block) {
        const bool first_block = block == group * EACH;
        const uint32_t ch = (uint32_t)block * CH + col, last = a.channels - 1, chc = ch < last ? ch : last;
        const bool on = ch <= last;
        float A2[NS], dA[NS], dD = 0.0f, dbias = 0.0f;          // A2 = A log2(e): dstep is summed with it and scaled once
        const float D = on && a.D ? a.D[ch] : 0.0f, bias = on && a.bias ? a.bias[ch] : 0.0f;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int s = part * NS + i;
            A2[i] = on && s < a.states ? a.A[ch * a.states + s] * kLog2e : 0.0f;
            dA[i] = 0.0f;
        }
        int64_t place = worker;                                 // of this worker's sums; its ray's where it has one ray: the dealing order leaves no trace
        for (int64_t task = worker; task < a.tasks; task += a.workers) {
            const Task t = find_task(a, task, lane);
            if (!t.live) continue;
            if (a.order) place = t.ray;
            float G[NS];                                        // dL/dh of the row behind, times its decay
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                const int s = part * NS + i;
                const bool here = on && s < a.states;
                G[i] = 0.0f;
                if (here && a.chunk) G[i] = a.ends[(t.slot * a.states + s) * a.channels + ch];
                else if (here && a.gfinal) G[i] = a.gfinal[(t.ray * a.channels + ch) * a.states + s];
            }
            const int64_t row0 = t.start + t.first, tiles = (t.n + kTile - 1) / kTile;
            auto rows_in = [&](int64_t k) { const int64_t r = t.n - k * kTile; return (int)(r < kTile ? r : kTile); };

            // what the next tile needs from memory
            T nu[PR], ndt[PR], nz[PR], ng[PR], nb[kStates], nc[kStates];
            float nh[NS];
            auto load = [&](int64_t k) {
                const int64_t row = row0 + k * kTile;
                const int n = rows_in(k);
#pragma unroll
                for (int r = 0; r < PR; ++r) {
                    const int j = part * PR + r;
                    const uint32_t at = j < n ? j : n - 1;
                    nu[r] = row_at<T>(a.u, row, a.ld_u, at, chc);
                    ndt[r] = row_at<T>(a.dt, row, a.ld_dt, at, chc);
                    ng[r] = row_at<T>(a.gy, row, a.ld_gy, at, chc);
                    nz[r] = a.z ? row_at<T>(a.z, row, a.ld_z, at, chc) : T(0.0f);
                }
#pragma unroll
                for (int q = 0; q < kStates; ++q) {
                    const int e = q * kWave + lane, s = e % SP;
                    const uint32_t at = e / SP < n ? e / SP : n - 1, sc = s < a.states ? s : 0;
                    nb[q] = row_at<T>(a.B, row, a.ld_B, at, sc);
                    nc[q] = row_at<T>(a.C, row, a.ld_C, at, sc);
                    if (s >= a.states) nb[q] = nc[q] = T(0.0f);
                }
                const bool inside = t.first + k > 0;
                const float *from = inside ? a.kept + (row / kTile) * a.states * a.channels : a.init;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int s = part * NS + i;
                    nh[i] = 0.0f;
                    if (from && on && s < a.states) nh[i] = from[inside ? (uint32_t)s * a.channels + ch : (t.ray * a.channels + ch) * a.states + s];
                }
            };
            if (tiles > 0) load(tiles - 1);
            for (int64_t k = tiles - 1; k >= 0; --k) {
                const int64_t row = row0 + k * kTile;
                const int n = rows_in(k);
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int r = 0; r < PR; ++r) {
                    const int j = part * PR + r;
                    // lanes without a channel: no input and no gradient, so that they add nothing to dB and dC
                    const float raw = to_f(ndt[r]) + bias, u = on ? to_f(nu[r]) : 0.0f, gy = on ? to_f(ng[r]) : 0.0f;
                    Step st = {raw, 1.0f};
                    if (a.softplus) st = softplus_step(raw);
                    float dy = gy, gate = 0.0f;
                    if (a.z) {
                        const float z = on ? to_f(nz[r]) : 0.0f, sig = sigmoid_f(z);
                        dy = gy * (z * sig);
                        gate = gy * (sig * fmaf(z, 1.0f - sig, 1.0f));
                    }
                    if (P <= kTile || j < kTile) {
                        own_rows[kStep][j][col] = on ? st.step : 0.0f;
                        own_rows[kU][j][col] = u;
                        own_rows[kSlope][j][col] = st.slope;
                        own_rows[kDy][j][col] = dy;
                        own_rows[kGate][j][col] = gate;
                    }
                }
#pragma unroll
                for (int q = 0; q < kStates; ++q) {
                    const int e = q * kWave + lane;
                    if (e < kTile * SP) {
                        bc[0][e] = to_f(nb[q]);
                        bc[1][e] = to_f(nc[q]);
                    }
                }
                float h[NS], h0[NS];
#pragma unroll
                for (int i = 0; i < NS; ++i) h[i] = h0[i] = nh[i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (k > 0) load(k - 1);

                auto states_at = [&](int which, int j, float (&v)[NS]) { read_states<NS>(&bc[which][j * SP + part * NS], v); };
#pragma unroll 2
                for (int j = 0; j < n; ++j) {
                    const float step = own_rows[kStep][j][col], in = step * own_rows[kU][j][col];
                    float B[NS];
                    states_at(0, j, B);
#pragma unroll
                    for (int i = 0; i < NS; ++i) h[i] = only_states<PADDED>(a, part * NS + i, fmaf(fast_exp2(step * A2[i]), h[i], in * B[i]));
                    if (j + 1 < n)
#pragma unroll
                        for (int i = 0; i < NS; i += 4) hist[j][i / 4][lane] = f32x4{h[i], h[i + 1], h[i + 2], h[i + 3]};
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                for (int j = n - 1; j >= 0; --j) {
                    const float step = own_rows[kStep][j][col], u = own_rows[kU][j][col], slope = own_rows[kSlope][j][col], dy = own_rows[kDy][j][col],
                                gate = own_rows[kGate][j][col], in = step * u;
                    float B[NS], C[NS], before[NS], v[2 * NS], y = 0.0f, sB = 0.0f, sA = 0.0f;
                    states_at(0, j, B);
                    states_at(1, j, C);
                    float *to = a.part_bc + ((int64_t)group * a.rows + row + j) * (2 * SP), before_sum[kLeft];
                    if (EACH > 1 && !first_block)               // what the blocks before this one left, read early
#pragma unroll
                        for (int i = 0; i < kLeft; ++i) {
                            const uint32_t q = i * (1 << kHalvings) + number;
                            before_sum[i] = to[(q / NS) * SP + part * NS + q % NS];
                        }
#pragma unroll
                    for (int i = 0; i < NS; i += 4) {
                        f32x4 q = {h0[i], h0[i + 1], h0[i + 2], h0[i + 3]};
                        if (j > 0) q = hist[j - 1][i / 4][lane];
#pragma unroll
                        for (int r = 0; r < 4; ++r) before[i + r] = q[r];
                    }
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        const float g = only_states<PADDED>(a, part * NS + i, fmaf(C[i], dy, G[i]));
                        y = fmaf(C[i], h[i], y);
                        v[i] = g * in;
                        v[NS + i] = dy * h[i];
                        sB = fmaf(g, B[i], sB);
                        G[i] = only_states<PADDED>(a, part * NS + i, g * fast_exp2(step * A2[i]));
                        const float w = G[i] * before[i];
                        sA = fmaf(w, A2[i], sA);
                        dA[i] = fmaf(w, step, dA[i]);
                        h[i] = before[i];
                    }
                    sB = sum_parts<P>(sB);
                    sA = sum_parts<P>(sA);
                    const float dstep = fmaf(u, sB, sA * kLn2) * slope;
                    if (a.z) y = add_skip(a, D, u, sum_parts<P>(y));
                    if (part == 0) {
                        own_rows[kU][j][col] = add_skip(a, D, dy, step * sB);
                        own_rows[kSlope][j][col] = dstep;
                        own_rows[kGate][j][col] = gate * y;
                    }
                    dD = fmaf(dy, u, dD);
                    dbias += dstep;
                    sum_over_lanes<2 * NS, CH / 2>(v, lane);
                    if (stores) {
#pragma unroll
                        for (int i = 0; i < kLeft; ++i) {
                            const uint32_t q = i * (1 << kHalvings) + number;
                            to[(q / NS) * SP + part * NS + q % NS] = EACH > 1 && !first_block ? before_sum[i] + v[i] : v[i];
                        }
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int r = 0; r < PR; ++r) {
                    const int j = part * PR + r;
                    if (!on || j >= n) continue;
                    const int64_t at = row * a.channels;
                    const uint32_t to = (uint32_t)j * a.channels + ch;
                    (reinterpret_cast<T *>(a.gu) + at)[to] = from_f<T>(own_rows[kU][j][col]);
                    (reinterpret_cast<T *>(a.gdt) + at)[to] = from_f<T>(own_rows[kSlope][j][col]);
                    if (a.z) (reinterpret_cast<T *>(a.gz) + at)[to] = from_f<T>(own_rows[kGate][j][col]);
                }
            }
            if (a.ginit && t.first == 0) {
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int s = part * NS + i;
                    if (on && s < a.states) a.ginit[(t.ray * a.channels + ch) * a.states + s] = G[i];
                }
            }
        }
        if (!on) continue;
        float *to = a.part_w + place * ((int64_t)a.channels * (a.states + 2));
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int s = part * NS + i;
            if (s < a.states) to[ch * a.states + s] = dA[i];
        }
        if (part == 0) {
            to[(int64_t)a.channels * a.states + ch] = dD;
            to[(int64_t)a.channels * (a.states + 1) + ch] = dbias;
        }
    }
}

// dB and dC of a row: the groups' sums in order; zeros for rows of no sequence.  A thread: four neighbouring states.  Memory: 2^18
// rows of two blocks and 16 states, 67 MB in and 17 out, 18 us (4.7 TB/s).
template <class T>
__global__ __launch_bounds__(kBlock) void scan_join_bc_kernel(ScanArgs a, int log_sp, T *gB, T *gC) {
    const int64_t n = a.rows << (log_sp - 1);               // 2 sp / 4 groups in a row
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < n; e += (int64_t)gridDim.x * kBlock) {
        const int64_t row = e >> (log_sp - 1);
        const int q = (int)(e & ((1 << (log_sp - 1)) - 1)) * 4, which = q >> log_sp, s = q & ((1 << log_sp) - 1);
        if (s >= a.states) continue;
        f32x4 v = {0, 0, 0, 0};
        if (!a.info || a.pos[row] >= 0)
            for (int b = 0; b < a.groups; ++b) {
                const f32x4 w = *reinterpret_cast<const f32x4 *>(a.part_bc + (((int64_t)b * a.rows + row) << (log_sp + 1)) + q);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += w[i];
            }
        T *to = (which ? gC : gB) + row * a.states + s;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (s + i < a.states) to[i] = from_f<T>(v[i]);
    }
}

// rows of no sequence; where there are none it reads the map of 2^18 rows in 2.2 us
template <class T>
__global__ __launch_bounds__(kBlock) void zero_rows_kernel(const int32_t *__restrict__ pos, int64_t rows, int32_t cols, T *p, T *q, T *r) {
    const int lane = lane_id();
    for (int64_t base = ((int64_t)blockIdx.x * kWavesPerBlock + wave_in_block()) * kWave; base < rows;
         base += (int64_t)gridDim.x * kBlock) {
        unsigned long long none = __ballot(base + lane < rows && pos[base + lane < rows ? base + lane : base] < 0);
        while (none) {
            const int64_t row = base + __ffsll((long long)none) - 1;
            none &= none - 1;
            for (int c = lane; c < cols; c += kWave) {
                p[row * cols + c] = T(0.0f);
                if (q) q[row * cols + c] = T(0.0f);
                if (r) r[row * cols + c] = T(0.0f);
            }
        }
    }
}

// a state's gradient without rows: that of the final state (nullptr: zeros)
__global__ __launch_bounds__(kBlock) void copy_state_kernel(const float *from, float *to, int64_t n) {
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < n; e += (int64_t)gridDim.x * kBlock) to[e] = from ? from[e] : 0.0f;
}

// One row per sequence: reading and writing the state bounds it (8 bytes per state).  L lanes share a channel, each with four
// neighbouring states (one 16-byte access); L = 0: a lane per channel and states one by one, for numbers of states that do not divide.
// 256 x 1024 x 16, bf16: 8.2 us (4.3 TB/s), 39.5 with states one by one.
template <class T, int L>
__global__ __launch_bounds__(kBlock) void scan_step_kernel(ScanArgs a, const float *state, float *next) {
    constexpr int LL = L ? L : 1;
    const uint32_t e = blockIdx.x * kBlock + threadIdx.x, ch = e / LL, s0 = e % LL * 4;
    if (ch >= (uint32_t)a.channels) return;                 // (whole groups of lanes: LL divides the wave)
    const float bias = a.bias ? a.bias[ch] : 0.0f, D = a.D ? a.D[ch] : 0.0f;
    f32x4 A = {0, 0, 0, 0};
    if (L) A = *reinterpret_cast<const f32x4 *>(a.A + ch * a.states + s0);
    for (int64_t ray = blockIdx.y; ray < a.n_rays; ray += gridDim.y) {
        const int64_t at = (ray * a.channels + ch) * a.states + s0;
        const float u = to_f((reinterpret_cast<const T *>(a.u) + ray * a.ld_u)[ch]);
        float step = to_f((reinterpret_cast<const T *>(a.dt) + ray * a.ld_dt)[ch]) + bias, y = 0.0f;
        const T *B = reinterpret_cast<const T *>(a.B) + ray * a.ld_B, *C = reinterpret_cast<const T *>(a.C) + ray * a.ld_C;
        f32x4 h = {0, 0, 0, 0};
        if (L) h = *reinterpret_cast<const f32x4 *>(state + at);
        float z = 0.0f;
        if (a.z) z = to_f((reinterpret_cast<const T *>(a.z) + ray * a.ld_z)[ch]);
        if (a.softplus) step = softplus_f(step);
        const float in = step * u, d2 = step * kLog2e;
        if (L) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = fmaf(fast_exp2(d2 * A[i]), h[i], in * to_f(B[s0 + i]));
                y = fmaf(to_f(C[s0 + i]), h[i], y);
            }
            *reinterpret_cast<f32x4 *>(next + at) = h;
            if constexpr (L >= 2) y = add_other<1>(y);
            if constexpr (L >= 4) y = add_other<2>(y);
            if constexpr (L >= 8) y = add_other<4>(y);
            if constexpr (L >= 16) y = add_other<8>(y);
        } else {
            for (int s = 0; s < a.states; ++s) {
                const float v = fmaf(fast_exp2(d2 * a.A[ch * a.states + s]), state[at + s], in * to_f(B[s]));
                next[at + s] = v;
                y = fmaf(to_f(C[s]), v, y);
            }
        }
        y = add_skip(a, D, u, y);
        if (a.z) y *= z * sigmoid_f(z);
        if (s0 == 0) (reinterpret_cast<T *>(a.y) + ray * a.channels)[ch] = from_f<T>(y);
    }
}

// lanes per channel and states per lane: up to 16 in a lane forward (2^18 rows of 64 channels of 16: 95 us, 106 by eights), 8 backward,
// where a wave's history in LDS decides how many waves there are (349 us, 473 by sixteens)
struct Shape { int ns, p; };
Shape shape_of(int states, int most) {
    Shape s{4, 1};
    while (s.ns < most && s.ns < states) s.ns *= 2;
    while (s.ns * s.p < states) s.p *= 2;
    return s;
}
constexpr int kFwdStates = 16, kBwdStates = 8;

// calls g(T{}, integral NS, integral P, integral whether there are more places than states)
template <int MOST, class F>
void with_shape(int32_t dtype, Shape sh, int states, F &&g) {
    auto f = [&](auto t, auto ns, auto p) {
        if (states == ns() * p()) g(t, ns, p, std::false_type{});
        else g(t, ns, p, std::true_type{});
    };
    with_dtype(dtype, [&](auto t) {
        if constexpr (MOST >= 16) {
            if (sh.ns == 16) {
                auto ns = std::integral_constant<int, 16>{};
                if (sh.p == 1) f(t, ns, std::integral_constant<int, 1>{});
                else if (sh.p == 2) f(t, ns, std::integral_constant<int, 2>{});
                else if (sh.p == 4) f(t, ns, std::integral_constant<int, 4>{});
                else if (sh.p == 8) f(t, ns, std::integral_constant<int, 8>{});
                else f(t, ns, std::integral_constant<int, 16>{});
                return;
            }
        }
        if (sh.ns == 4) {
            f(t, std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
            return;
        }
        auto ns = std::integral_constant<int, 8>{};
        if constexpr (MOST >= 16) {
            f(t, ns, std::integral_constant<int, 1>{});
        } else {
            if (sh.p == 1) f(t, ns, std::integral_constant<int, 1>{});
            else if (sh.p == 2) f(t, ns, std::integral_constant<int, 2>{});
            else if (sh.p == 4) f(t, ns, std::integral_constant<int, 4>{});
            else if (sh.p == 8) f(t, ns, std::integral_constant<int, 8>{});
            else if (sh.p == 16) f(t, ns, std::integral_constant<int, 16>{});
            else f(t, ns, std::integral_constant<int, 32>{});
        }
    });
}

// How a call is cut.  Cutting costs a second pass over the exponentials, so whole sequences where they give every SIMD a wave (256
// sequences of 256 rows, 256 channels: 151 us, 215 in chunks) or would be cut in less than four (512 of 64 rows, 64 channels: 42 us, 66 in
// chunks of 32; 256 of 128 rows: 74 us, 58 in chunks); packed ones, of which a few may be much longer than the mean, in less than two.
// (The mean decides: one ray that holds most rows of a thousand others is walked by one wave for each block of its channels.)
// Otherwise chunks of at least 32 rows, for two waves per SIMD; in the forward pass
// four (32768 rows of 1024 channels 331 -> 297 us, 64 sequences of 512 rows, 512 channels 200 -> 165), unless that makes them shorter than
// 64 rows (two sequences of 8192 rows, 512 channels: 106 us, 116 with four) or a chain longer than 512 (131072 rows of 64 channels: 298
// and 497).  The backward pass holds two waves per SIMD at most (its LDS).
struct ScanPlan { Shape sh; int blocks, groups; int64_t chunk, chunks, slots, tasks, workers; };
ScanPlan scan_plan(int64_t n_rays, int64_t rows, int channels, int states, bool packed, bool backward) {
    ScanPlan p{};
    p.sh = shape_of(states, backward ? kBwdStates : kFwdStates);
    p.blocks = (int)ceil_div(channels, kWave / p.sh.p);
    p.groups = backward ? (int)ceil_div(p.blocks, blocks_of_wave(p.sh.p)) : p.blocks;      // waves side by side
    const int64_t waves = n_rays * p.groups, want = (int64_t)kNumCU * 8;
    p.tasks = n_rays;
    if (n_rays > 0 && waves < kNumCU * 4 && rows / n_rays >= 64) {
        const int64_t length = rows / n_rays;
        auto chunk_for = [&](int64_t waves) { return ceil_div(ceil_div(rows * p.groups, waves), kTile) * kTile; };
        int64_t chunk = chunk_for(want);
        if (!backward && chunk_for(2 * want) >= 64 && length / chunk_for(2 * want) <= 512) chunk = chunk_for(2 * want);
        if (chunk < 32) chunk = 32;
        if (packed ? chunk < length : 4 * chunk <= length) {
            p.chunk = chunk;
            p.chunks = ceil_div(length, chunk);
            p.slots = rows / chunk + 1 + n_rays;
            p.tasks = packed ? n_rays + ceil_div(rows, chunk) : n_rays * p.chunks;
        }
    }
    p.workers = p.tasks;
    // partial sums of the backward pass: one per sequence, so that the long ones can be dealt out first, up to 32768 waves (16384 ragged
    // sequences, 64 channels: 1.32 ms, 1.60 with half as many waves; 65536: 1.51 with a quarter, 1.57 with all of them)
    const int64_t most = ceil_div(32768, p.blocks);
    if (backward && p.workers > most) p.workers = most;
    return p;
}
int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }
struct ScanSpace { int64_t ends, sums, bc, w, total; };
ScanSpace scan_space(const ScanPlan &p, int64_t rows, int channels, int states, bool backward) {
    ScanSpace s{};
    s.ends = align256(p.slots * states * channels * 4);
    s.sums = align256(p.slots * channels * 4);
    if (backward) {
        s.bc = align256((int64_t)p.groups * rows * 2 * p.sh.ns * p.sh.p * 4);
        s.w = align256(p.workers * channels * (states + 2) * 4);
    }
    s.total = s.ends + s.sums + s.bc + s.w;
    return s;
}

int check_scan(const nfa_selective_scan_args *a, const char *who, bool step) {
    NFA_REQUIRE(a, "%s: NULL arguments", who);
    NFA_REQUIRE(a->n_rays >= 0 && a->rows >= 0 && a->channels >= 1, "%s: bad size", who);
    NFA_REQUIRE(a->states >= 1 && a->states <= NFA_SCAN_MAX_STATES, "%s: states must be 1 .. %d, got %d", who, NFA_SCAN_MAX_STATES, a->states);
    NFA_REQUIRE(dtype_ok(a->dtype), "%s: bad dtype %d", who, a->dtype);
    NFA_REQUIRE(a->rows < (1ll << 31) && a->n_rays < (1ll << 31) && a->channels <= (1 << 23), "%s: too many rows, rays or channels", who);
    const int64_t rows = step ? a->n_rays : a->rows;
    NFA_REQUIRE(a->A, "%s: NULL pointer", who);
    NFA_REQUIRE(rows == 0 || (a->inputs && a->delta && a->B && a->C), "%s: NULL pointer", who);
    NFA_REQUIRE(rows <= 1 || (a->inputs_stride >= a->channels && a->delta_stride >= a->channels && (!a->gate || a->gate_stride >= a->channels) &&
                              a->B_stride >= a->states && a->C_stride >= a->states), "%s: a row stride is shorter than its row", who);
    if (step) return NFA_OK;
    for (int64_t ld : {a->inputs_stride, a->delta_stride, a->gate_stride, a->B_stride, a->C_stride, a->grad_outputs_stride})
        NFA_REQUIRE(ld <= kMaxStride, "%s: a row stride is over 2^25", who);
    NFA_REQUIRE(a->packed_info || a->n_rays == 0 || a->rows % a->n_rays == 0, "%s: rows do not divide into equal sequences", who);
    NFA_REQUIRE(a->n_rays > 0 || a->packed_info || a->rows == 0, "%s: rows without sequences", who);
    NFA_REQUIRE(!a->packed_info || a->rows == 0 || (a->row_ray && a->row_pos), "%s: packed sequences need their row map", who);
    return NFA_OK;
}

ScanArgs scan_args(const nfa_selective_scan_args *a) {
    ScanArgs d{};
    d.u = a->inputs; d.ld_u = a->inputs_stride;
    d.dt = a->delta; d.ld_dt = a->delta_stride;
    d.z = a->gate; d.ld_z = a->gate_stride;
    d.B = a->B; d.ld_B = a->B_stride;
    d.C = a->C; d.ld_C = a->C_stride;
    d.gy = a->grad_outputs; d.ld_gy = a->grad_outputs_stride;
    d.A = a->A; d.D = a->D; d.bias = a->delta_bias; d.init = a->initial_state; d.gfinal = a->grad_final_state;
    d.info = a->packed_info; d.ray = a->row_ray; d.pos = a->row_pos;
    d.order = a->packed_info ? a->ray_order : nullptr;
    d.rows = a->rows; d.n_rays = a->n_rays;
    d.length = a->n_rays > 0 ? a->rows / a->n_rays : 0;
    d.channels = a->channels; d.states = a->states; d.softplus = a->delta_softplus != 0;
    return d;
}
void use_plan(ScanArgs &d, const ScanPlan &p, const ScanSpace &sp, void *workspace) {
    d.chunk = p.chunk; d.chunks = p.chunks; d.slots = p.slots; d.tasks = p.tasks; d.workers = p.workers; d.blocks = p.blocks; d.groups = p.groups;
    char *w = (char *)workspace;
    d.ends = (float *)w;
    d.sums = (float *)(w + sp.ends);
    d.part_bc = (float *)(w + sp.ends + sp.sums);
    d.part_w = (float *)(w + sp.ends + sp.sums + sp.bc);
}

template <bool REV>
void launch_chain(const ScanArgs &d, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div((int64_t)d.channels * d.states, kBlock), (unsigned)d.n_rays);
    hipLaunchKernelGGL((scan_chain_kernel<REV>), grid, dim3(kBlock), 0, s, d);
}
void launch_zero_rows(const ScanArgs &d, int32_t dtype, void *p, void *q, void *r, hipStream_t s) {
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((zero_rows_kernel<T>), dim3(blocks_for(d.rows)), dim3(kBlock), 0, s, d.pos, d.rows, d.channels, (T *)p, (T *)q, (T *)r);
    });
}

}  // namespace
}  // namespace nfa

using namespace nfa;

NFA_EXPORT int64_t nfa_selective_scan_checkpoint_bytes(int64_t rows, int32_t channels, int32_t states) {
    if (rows <= 0 || channels <= 0 || states <= 0) return 0;
    return ceil_div(rows, kTile) * channels * states * 4;
}

NFA_EXPORT int64_t nfa_selective_scan_workspace_bytes(int64_t n_rays, int64_t rows, int32_t channels, int32_t states, int32_t backward) {
    if (n_rays <= 0 || rows <= 0 || channels <= 0 || states <= 0 || states > NFA_SCAN_MAX_STATES) return 0;
    const ScanPlan p = scan_plan(n_rays, rows, channels, states, true, backward != 0), q = scan_plan(n_rays, rows, channels, states, false, backward != 0);
    const int64_t x = scan_space(p, rows, channels, states, backward != 0).total, y = scan_space(q, rows, channels, states, backward != 0).total;
    return x > y ? x : y;
}

NFA_EXPORT int nfa_selective_scan_fwd(const nfa_selective_scan_args *a, void *outputs, float *final_state, float *checkpoints,
                                      void *workspace, void *stream) {
    if (int rc = check_scan(a, "selective_scan_fwd", false)) return rc;
    NFA_REQUIRE(outputs || a->rows == 0, "selective_scan_fwd: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    ScanArgs d = scan_args(a);
    const ScanPlan p = scan_plan(a->n_rays, a->rows, a->channels, a->states, a->packed_info != nullptr, false);
    const ScanSpace sp = scan_space(p, a->rows, a->channels, a->states, false);
    NFA_REQUIRE(workspace || sp.total == 0, "selective_scan_fwd: NULL workspace");
    use_plan(d, p, sp, workspace);
    d.y = outputs; d.final_state = final_state; d.kept = checkpoints;
    if (a->packed_info && a->rows > 0) launch_zero_rows(d, a->dtype, outputs, nullptr, nullptr, s);
    if (p.tasks > 0) {
        const int64_t grid = p.tasks * p.blocks;
        NFA_REQUIRE(grid < kMaxThreads / kWave && a->n_rays * (int64_t)(p.chunk ? 1 : 0) < 65536, "selective_scan_fwd: too large for one launch");
        with_shape<kFwdStates>(a->dtype, p.sh, a->states, [&](auto t, auto ns, auto pp, auto padded) {
            using T = decltype(t);
            if (p.chunk) {
                hipLaunchKernelGGL((scan_fwd_kernel<T, ns(), pp(), padded(), true>), dim3((unsigned)grid), dim3(kWave), 0, s, d);
                launch_chain<false>(d, s);
            }
            hipLaunchKernelGGL((scan_fwd_kernel<T, ns(), pp(), padded(), false>), dim3((unsigned)grid), dim3(kWave), 0, s, d);
        });
    }
    return check_launch("scan_fwd_kernel");
}

NFA_EXPORT int nfa_selective_scan_bwd(const nfa_selective_scan_args *a, const float *checkpoints, const nfa_selective_scan_grads *g,
                                      void *workspace, void *stream) {
    if (int rc = check_scan(a, "selective_scan_bwd", false)) return rc;
    NFA_REQUIRE(g && g->A && (a->rows == 0 || (g->inputs && g->delta && g->B && g->C && (!a->gate || g->gate))), "selective_scan_bwd: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    if (a->rows == 0 || a->n_rays == 0) {                   // no row of a sequence: zeros, and the final state's gradient as it came
        for (void *p : {g->inputs, g->delta, g->gate}) launch_zero(p, a->rows * a->channels, a->dtype, s);
        for (void *p : {g->B, g->C}) launch_zero(p, a->rows * a->states, a->dtype, s);
        launch_zero(g->A, (int64_t)a->channels * a->states, NFA_DTYPE_F32, s);
        for (float *p : {g->D, g->delta_bias}) launch_zero(p, a->channels, NFA_DTYPE_F32, s);
        const int64_t n = a->n_rays * a->channels * a->states;
        if (g->initial_state && n > 0)
            hipLaunchKernelGGL(copy_state_kernel, dim3(blocks_for(n)), dim3(kBlock), 0, s, a->grad_final_state, g->initial_state, n);
        return check_launch("copy_state_kernel");
    }
    NFA_REQUIRE(a->grad_outputs && checkpoints && workspace, "selective_scan_bwd: NULL pointer");
    NFA_REQUIRE(a->grad_outputs_stride >= a->channels || a->rows <= 1, "selective_scan_bwd: grad_outputs_stride < channels");
    ScanArgs d = scan_args(a);
    const ScanPlan p = scan_plan(a->n_rays, a->rows, a->channels, a->states, a->packed_info != nullptr, true);
    const ScanSpace sp = scan_space(p, a->rows, a->channels, a->states, true);
    use_plan(d, p, sp, workspace);
    if (p.workers != a->n_rays || p.chunk) d.order = nullptr;
    d.kept = (float *)checkpoints;
    d.gu = g->inputs; d.gdt = g->delta; d.gz = a->gate ? g->gate : nullptr; d.ginit = g->initial_state;
    const int64_t grid = p.tasks * p.blocks, main_grid = p.workers * p.groups;
    NFA_REQUIRE(grid < kMaxThreads / kWave && a->n_rays * (int64_t)(p.chunk ? 1 : 0) < 65536, "selective_scan_bwd: too large for one launch");
    if (a->packed_info) launch_zero_rows(d, a->dtype, d.gu, d.gdt, d.gz, s);
    with_shape<kBwdStates>(a->dtype, p.sh, a->states, [&](auto t, auto ns, auto pp, auto padded) {
        using T = decltype(t);
        if (p.chunk) {
            hipLaunchKernelGGL((scan_bwd_local_kernel<T, ns(), pp(), padded()>), dim3((unsigned)grid), dim3(kWave), 0, s, d);
            launch_chain<true>(d, s);
        }
        hipLaunchKernelGGL((scan_bwd_kernel<T, ns(), pp(), padded()>), dim3((unsigned)main_grid), dim3(kWave), 0, s, d);
        hipLaunchKernelGGL((scan_join_bc_kernel<T>), dim3(blocks_for(a->rows * ns() * pp() / 2)), dim3(kBlock), 0, s, d, log2_of(ns() * pp()), (T *)g->B,
                           (T *)g->C);
    });
    launch_reduce_rows(d.part_w, p.workers, {{g->A, (int64_t)a->channels * a->states}, {g->D, a->channels}, {g->delta_bias, a->channels}}, NFA_DTYPE_F32, s);
    return check_launch("scan_bwd_kernel");
}

NFA_EXPORT int nfa_selective_scan_step(const nfa_selective_scan_args *a, const float *state, void *outputs, float *out_state, void *stream) {
    if (int rc = check_scan(a, "selective_scan_step", true)) return rc;
    if (a->n_rays == 0) return NFA_OK;
    NFA_REQUIRE(state && outputs && out_state, "selective_scan_step: NULL pointer");
    ScanArgs d = scan_args(a);
    d.y = outputs;
    const bool whole = ((uintptr_t)state | (uintptr_t)out_state | (uintptr_t)a->A) % 16 == 0;
    int lanes = 0;
    for (int l : {1, 2, 4, 8, 16})
        if (whole && a->states == 4 * l) lanes = l;
    const int64_t per = (int64_t)a->channels * (lanes ? lanes : 1);
    const dim3 grid((unsigned)ceil_div(per, kBlock), (unsigned)std::min<int64_t>(a->n_rays, 32768));
    with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        const auto kernel = lanes == 1 ? scan_step_kernel<T, 1> : lanes == 2 ? scan_step_kernel<T, 2> : lanes == 4 ? scan_step_kernel<T, 4>
                          : lanes == 8 ? scan_step_kernel<T, 8> : lanes == 16 ? scan_step_kernel<T, 16> : scan_step_kernel<T, 0>;
        hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, (hipStream_t)stream, d, state, out_state);
    });
    return check_launch("scan_step_kernel");
}
