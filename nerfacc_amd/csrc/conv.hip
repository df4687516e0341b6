// conv.hip — short causal convolution along each sequence (ray), channel by channel, for gfx950.
//
//   z[t] = b + sum_{j < W} w[j] x[t - W + 1 + j]     (rows before the sequence: its state, or zeros),   y = act(z)
//   g = dy act'(z),  dx[t] = sum_{i < W} w[W - 1 - i] g[t + i] (+ the final state's gradient),  dw[j] = sum_t g[t] x[t - W + 1 + j]
//
// Bound by memory: one read of x and one write of y (backward: x and dy in, dx out).  A thread owns up to sixteen bytes of channels
// and walks a piece of consecutive rows with the last W - 1 inputs in registers, so each input is fetched once per piece (+ W - 1
// rows in front of it, which the caches hold).  The backward walk runs forward too: it forms z again from x, and dx[t] is finished
// W - 1 rows later, when its last g is known.  Weight gradients stay in registers over all of a thread's pieces, are joined in LDS
// and then in order over the workgroups: no atomics.
//
// On one MI355X (copies reach 5.1 TB/s, tuned ones 6.2): 2^18 rows of 128 channels, bf16, 4096 rays: forward 33 us (134 MB: 4.1 TB/s), backward 67 us (201
// MB: 3.0 TB/s) + 6 to join; 32768 x 2048 fp16: forward 58-63 us (268 MB: 4.3-4.6 TB/s); one row of 256 rays of 2048 channels 5 us.
#include "feature.hpp"

#include <algorithm>

namespace nfa {
namespace {

struct ConvArgs {
    const void *x, *w, *bias, *init, *gy, *gfinal;
    void *y, *gx;
    float *partial;                     // backward: [workgroups][channels * W + channels]
    const int64_t *info;
    const int32_t *ray, *pos;
    int64_t rows, n_rays, length;       // length: of every sequence where info is NULL
    int64_t ld_x, ld_gy;
    int32_t channels, piece, lanes, act;
    int64_t pieces;
};

// where a row lies: its sequence and its position there (-1: in none)
struct Place { int32_t ray, pos; };
__device__ __forceinline__ Place place_of(const ConvArgs &a, int64_t row) {
    if (a.info) return {a.ray[row], a.pos[row]};
    const int64_t r = row / a.length;
    return {(int32_t)r, (int32_t)(row - r * a.length)};
}
__device__ __forceinline__ Place place_after(const ConvArgs &a, Place p, int64_t row) {     // of `row`, from that of row - 1
    if (a.info) return {a.ray[row], a.pos[row]};
    return p.pos + 1 == a.length ? Place{p.ray + 1, 0} : Place{p.ray, p.pos + 1};
}

template <class T, int VC> struct alignas(VC * sizeof(T)) Vec { T v[VC]; };
template <class T, int VC>
__device__ __forceinline__ void load_row(const void *base, int64_t at, float (&out)[VC]) {
    const Vec<T, VC> v = *reinterpret_cast<const Vec<T, VC> *>(reinterpret_cast<const T *>(base) + at);
#pragma unroll
    for (int c = 0; c < VC; ++c) out[c] = to_f(v.v[c]);
}
template <class T, int VC>
__device__ __forceinline__ void store_row(void *base, int64_t at, const float (&in)[VC]) {
    Vec<T, VC> v;
#pragma unroll
    for (int c = 0; c < VC; ++c) v.v[c] = from_f<T>(in[c]);
    *reinterpret_cast<Vec<T, VC> *>(reinterpret_cast<T *>(base) + at) = v;
}

// the input `back` rows before position p of its sequence: a row of x, of the state, or zeros
template <class T, int W, int VC>
__device__ __forceinline__ void load_before(const ConvArgs &a, int64_t row, Place p, int back, int64_t c, float (&out)[VC]) {
    if (p.pos >= back) {
        load_row<T, VC>(a.x, (row - back) * a.ld_x + c, out);
    } else if (a.init && p.pos >= 0) {
        load_row<T, VC>(a.init, ((int64_t)p.ray * (W - 1) + (W - 1 - back + p.pos)) * a.channels + c, out);
    } else {
#pragma unroll
        for (int i = 0; i < VC; ++i) out[i] = 0.0f;
    }
}

constexpr int kAhead = 4;               // rows whose loads are in flight together

// Three waves on a SIMD: a fourth would take the registers of the window and the rows in flight (it spilled); memory bounds it at 4.1 TB/s.
template <class T, int W, int VC>
__global__ __launch_bounds__(kBlock, 3) void conv_fwd_kernel(ConvArgs a) {
    const int lane = threadIdx.x % a.lanes;
    const int64_t c = ((int64_t)blockIdx.y * a.lanes + lane) * VC;
    const int64_t piece = (int64_t)blockIdx.x * (kBlock / a.lanes) + threadIdx.x / a.lanes;
    if (c >= a.channels || piece >= a.pieces) return;
    const int64_t begin = piece * a.piece, end = begin + a.piece < a.rows ? begin + a.piece : a.rows;
    float w[W][VC], b[VC], win[W][VC];                      // win[j]: the input W - 1 - j rows back
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        b[i] = a.bias ? to_f(reinterpret_cast<const T *>(a.bias)[c + i]) : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = to_f(reinterpret_cast<const T *>(a.w)[(c + i) * W + j]);
    }
    Place p = place_of(a, begin);
#pragma unroll
    for (int j = 1; j < W; ++j) load_before<T, W, VC>(a, begin, p, W - j, c, win[j]);
    // the next rows' loads are in flight while these are computed; rows behind the piece read its last row again
    Vec<T, VC> next[kAhead];
    Place after[kAhead];
    auto load = [&](int64_t row, Place before) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int64_t r = row + k < end ? row + k : end - 1;
            after[k] = r == begin ? p : place_after(a, k ? after[k - 1] : before, r);
            next[k] = *reinterpret_cast<const Vec<T, VC> *>(reinterpret_cast<const T *>(a.x) + r * a.ld_x + c);
        }
    };
    load(begin, p);
    for (int64_t row = begin; row < end; row += kAhead) {
        Vec<T, VC> now[kAhead];
        Place at[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            now[k] = next[k];
            at[k] = after[k];
        }
        if (row + kAhead < end) load(row + kAhead, at[kAhead - 1]);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (row + k >= end) continue;
            if (at[k].pos == 0 && row + k != begin) {       // a new sequence: its state comes before it
#pragma unroll
                for (int j = 1; j < W; ++j) load_before<T, W, VC>(a, row + k, at[k], W - j, c, win[j]);
            }
#pragma unroll
            for (int j = 0; j + 1 < W; ++j)
#pragma unroll
                for (int i = 0; i < VC; ++i) win[j][i] = win[j + 1][i];
            float y[VC];
#pragma unroll
            for (int i = 0; i < VC; ++i) {
                win[W - 1][i] = to_f(now[k].v[i]);
                float z = b[i];
#pragma unroll
                for (int j = 0; j < W; ++j) z = fmaf(w[j][i], win[j][i], z);
                y[i] = z;
            }
            if (a.act == NFA_ACT_SILU)
#pragma unroll
                for (int i = 0; i < VC; ++i) y[i] *= sigmoid_f(y[i]);
            if (at[k].pos < 0)
#pragma unroll
                for (int i = 0; i < VC; ++i) y[i] = 0.0f;
            store_row<T, VC>(a.y, (row + k) * a.channels + c, y);
        }
    }
}

// x and dy in, dx out in one walk.  3.0 TB/s: z, the activation's slope and two windows of W rows keep the vector units busy for 85 % of the
// CUs' cycles (2^18 x 128 bf16), and the W - 1 rows in front of a piece are walked twice.
template <class T, int W, int VC>
__global__ __launch_bounds__(kBlock, 3) void conv_bwd_kernel(ConvArgs a) {
    extern __shared__ float joined[];
    const int lane = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes, groups = kBlock / a.lanes;
    const int64_t c = ((int64_t)blockIdx.y * a.lanes + lane) * VC;
    const bool on = c < a.channels;
    float w[W][VC], b[VC], dw[W][VC], db[VC];
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        b[i] = on && a.bias ? to_f(reinterpret_cast<const T *>(a.bias)[c + i]) : 0.0f;
        db[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            w[j][i] = on ? to_f(reinterpret_cast<const T *>(a.w)[(c + i) * W + j]) : 0.0f;
            dw[j][i] = 0.0f;
        }
    }
    for (int64_t piece = (int64_t)blockIdx.x * groups + group; on && piece < a.pieces; piece += (int64_t)gridDim.x * groups) {
        const int64_t begin = piece * a.piece, end = begin + a.piece < a.rows ? begin + a.piece : a.rows;
        const int64_t stop = end + W - 1 < a.rows ? end + W - 1 : a.rows;      // g of the rows behind reaches back into the piece
        float win[W][VC], acc[W][VC];                                          // acc[i]: dx of the row i rows back, so far
        Place p = place_of(a, begin);
#pragma unroll
        for (int j = 1; j < W; ++j) load_before<T, W, VC>(a, begin, p, W - j, c, win[j]);
#pragma unroll
        for (int j = 0; j < W; ++j)
#pragma unroll
            for (int i = 0; i < VC; ++i) acc[j][i] = 0.0f;
        auto finish = [&](int64_t row, const float (&v)[VC]) {                 // dx of a row of this piece is complete
            if (row < begin || row >= end || !a.gx) return;
            float out[VC];
#pragma unroll
            for (int i = 0; i < VC; ++i) out[i] = v[i];
            if (a.gfinal) {
                const Place q = place_of(a, row);
                if (q.pos >= 0) {
                    int64_t count = a.length;
                    if (a.info) {                                              // (the rows that exist: cut at the array's end)
                        const int64_t start = row - q.pos, n = a.info[2 * q.ray + 1] + (a.info[2 * q.ray] < 0 ? a.info[2 * q.ray] : 0);
                        count = n < a.rows - start ? n : a.rows - start;
                    }
                    const int64_t rest = count - 1 - q.pos;
                    if (rest >= 0 && rest < W - 1) {                          // (rays that overlap leave rows behind their ray's end)
                        float f[VC];
                        load_row<T, VC>(a.gfinal, ((int64_t)q.ray * (W - 1) + (W - 2 - rest)) * a.channels + c, f);
#pragma unroll
                        for (int i = 0; i < VC; ++i) out[i] += f[i];
                    }
                }
            }
            store_row<T, VC>(a.gx, row * a.channels + c, out);
        };
        for (int64_t row = begin; row < stop; row += kAhead) {
            Vec<T, VC> nx[kAhead], ng[kAhead];
            Place at[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int64_t r = row + k < stop ? row + k : stop - 1;
                at[k] = r == begin ? p : place_after(a, k ? at[k - 1] : p, r);
                nx[k] = *reinterpret_cast<const Vec<T, VC> *>(reinterpret_cast<const T *>(a.x) + r * a.ld_x + c);
                ng[k] = *reinterpret_cast<const Vec<T, VC> *>(reinterpret_cast<const T *>(a.gy) + r * a.ld_gy + c);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (row + k >= stop) continue;
                if (at[k].pos == 0 && row + k != begin) {
#pragma unroll
                    for (int j = 1; j < W; ++j) load_before<T, W, VC>(a, row + k, at[k], W - j, c, win[j]);
                }
#pragma unroll
                for (int j = 0; j + 1 < W; ++j)
#pragma unroll
                    for (int i = 0; i < VC; ++i) win[j][i] = win[j + 1][i];
#pragma unroll
                for (int j = W - 1; j > 0; --j)
#pragma unroll
                    for (int i = 0; i < VC; ++i) acc[j][i] = acc[j - 1][i];
                const bool in = at[k].pos >= 0, mine = row + k < end;
#pragma unroll
                for (int i = 0; i < VC; ++i) {
                    win[W - 1][i] = to_f(nx[k].v[i]);
                    float g = to_f(ng[k].v[i]);
                    if (a.act == NFA_ACT_SILU) {
                        float z = b[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) z = fmaf(w[j][i], win[j][i], z);
                        g *= act_slope<NFA_ACT_SILU>(z);
                    }
                    acc[0][i] = 0.0f;
                    if (in) {
#pragma unroll
                        for (int j = 0; j < W; ++j)                            // dx[row - j] of the same sequence
                            if (at[k].pos >= j) acc[j][i] = fmaf(w[W - 1 - j][i], g, acc[j][i]);
                        if (mine) {
                            db[i] += g;
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[j][i] = fmaf(g, win[j][i], dw[j][i]);
                        }
                    }
                }
                finish(row + k - (W - 1), acc[W - 1]);
                p = at[k];
            }
        }
        // the array ended before the last rows' sums were W rows old
#pragma unroll
        for (int j = W - 2; j >= 0; --j) finish(stop - 1 - j, acc[j]);
    }
    if (!a.partial) return;
    // groups of the workgroup join in order
    constexpr int kEach = (W + 1) * VC;
#pragma unroll
    for (int i = 0; i < VC; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) joined[(threadIdx.x * kEach) + i * W + j] = dw[j][i];
        joined[threadIdx.x * kEach + VC * W + i] = db[i];
    }
    __syncthreads();
    float *part = a.partial + (int64_t)blockIdx.x * a.channels * (W + 1);
    for (int e = threadIdx.x; e < a.lanes * kEach; e += kBlock) {
        const int l = e / kEach, k = e % kEach;
        const int64_t ch = ((int64_t)blockIdx.y * a.lanes + l) * VC;
        if (ch >= a.channels) continue;
        float v = 0.0f;
        for (int g = 0; g < groups; ++g) v += joined[(g * a.lanes + l) * kEach + k];
        if (k < VC * W) part[ch * W + k] = v;
        else part[(int64_t)a.channels * W + ch + k - VC * W] = v;
    }
}

// the rows [start, start + count) of a sequence that lie in the array
__device__ __forceinline__ void rows_of(const int64_t *info, int64_t ray, int64_t rows, int64_t length, int64_t &start, int64_t &count) {
    if (!info) { start = ray * length; count = length; return; }
    start = info[2 * ray];
    count = info[2 * ray + 1];
    if (start < 0) { count += start; start = 0; }
    if (start > rows) start = rows;
    if (count < 0) count = 0;
    if (count > rows - start) count = rows - start;
}

// final_state[ray][i]: row count - (W - 1) + i of the sequence, or the initial state's row behind that place
template <class T, int W>
__global__ __launch_bounds__(kBlock) void conv_final_kernel(ConvArgs a, T *final_state) {
    const int64_t n = a.n_rays * (W - 1) * a.channels;
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < n; e += (int64_t)gridDim.x * kBlock) {
        const int64_t c = e % a.channels, i = e / a.channels % (W - 1), ray = e / a.channels / (W - 1);
        int64_t start, count;
        rows_of(a.info, ray, a.rows, a.length, start, count);
        const int64_t at = count - (W - 1) + i;
        T v = T(0.0f);
        if (at >= 0) v = reinterpret_cast<const T *>(a.x)[(start + at) * a.ld_x + c];
        else if (a.init) v = reinterpret_cast<const T *>(a.init)[(ray * (W - 1) + count + i) * a.channels + c];
        final_state[e] = v;
    }
}

// grad_initial_state[ray][i] = sum_{p <= i} w[i - p] g[start + p], and the final state's gradient where the sequence is shorter than it
template <class T, int W>
__global__ __launch_bounds__(kBlock) void conv_init_grad_kernel(ConvArgs a, T *grad_init) {
    const int64_t n = a.n_rays * a.channels;
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < n; e += (int64_t)gridDim.x * kBlock) {
        const int64_t c = e % a.channels, ray = e / a.channels;
        int64_t start, count;
        rows_of(a.info, ray, a.rows, a.length, start, count);
        float w[W], g[W - 1], line[2 * (W - 1)];            // the state's rows and the first of the sequence
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = to_f(reinterpret_cast<const T *>(a.w)[c * W + j]);
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            line[i] = to_f(reinterpret_cast<const T *>(a.init)[(ray * (W - 1) + i) * a.channels + c]);
            line[W - 1 + i] = i < count ? to_f(reinterpret_cast<const T *>(a.x)[(start + i) * a.ld_x + c]) : 0.0f;
        }
        const float b = a.bias ? to_f(reinterpret_cast<const T *>(a.bias)[c]) : 0.0f;
#pragma unroll
        for (int p = 0; p < W - 1; ++p) {
            float z = b;
#pragma unroll
            for (int j = 0; j < W; ++j) z = fmaf(w[j], line[p + j], z);
            g[p] = 0.0f;
            if (p < count) {
                g[p] = to_f(reinterpret_cast<const T *>(a.gy)[(start + p) * a.ld_gy + c]);
                if (a.act == NFA_ACT_SILU) g[p] *= act_slope<NFA_ACT_SILU>(z);
            }
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            float v = 0.0f;
#pragma unroll
            for (int p = 0; p <= i; ++p) v = fmaf(w[i - p], g[p], v);
            if (a.gfinal && i - count >= 0) v += to_f(reinterpret_cast<const T *>(a.gfinal)[(ray * (W - 1) + i - count) * a.channels + c]);
            grad_init[(ray * (W - 1) + i) * a.channels + c] = from_f<T>(v);
        }
    }
}

// one row of every sequence: the launch bounds it (256 x 2048 bf16, 8 MB: 5.0 us)
template <class T, int W, int VC>
__global__ __launch_bounds__(kBlock) void conv_step_kernel(ConvArgs a, const T *state, T *y, T *next) {
    const int64_t c = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * VC;
    if (c >= a.channels) return;
    float w[W][VC], b[VC];
#pragma unroll
    for (int i = 0; i < VC; ++i) {
        b[i] = a.bias ? to_f(reinterpret_cast<const T *>(a.bias)[c + i]) : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = to_f(reinterpret_cast<const T *>(a.w)[(c + i) * W + j]);
    }
    for (int64_t ray = blockIdx.y; ray < a.n_rays; ray += gridDim.y) {
        using V = Vec<T, VC>;
        V line[W], out;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) line[j] = *reinterpret_cast<const V *>(state + (ray * (W - 1) + j) * a.channels + c);
        line[W - 1] = *reinterpret_cast<const V *>(reinterpret_cast<const T *>(a.x) + ray * a.ld_x + c);
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            float z = b[i];
#pragma unroll
            for (int j = 0; j < W; ++j) z = fmaf(w[j][i], to_f(line[j].v[i]), z);
            if (a.act == NFA_ACT_SILU) z = z * sigmoid_f(z);
            out.v[i] = from_f<T>(z);
        }
        *reinterpret_cast<V *>(y + ray * a.channels + c) = out;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) *reinterpret_cast<V *>(next + (ray * (W - 1) + j) * a.channels + c) = line[j + 1];
    }
}

__global__ __launch_bounds__(kBlock) void fill_map_kernel(int32_t *ray, int32_t *pos, int64_t rows) {
    for (int64_t r = (int64_t)blockIdx.x * kBlock + threadIdx.x; r < rows; r += (int64_t)gridDim.x * kBlock) ray[r] = pos[r] = -1;
}
// sixteen lanes per sequence; 2^18 rows of 4096 sequences 3 us, the fill before it 2.3
__global__ __launch_bounds__(kBlock) void row_map_kernel(const int64_t *__restrict__ info, int64_t n_rays, int64_t rows,
                                                         int32_t *__restrict__ row_ray, int32_t *__restrict__ row_pos) {
    const int64_t groups = (int64_t)gridDim.x * (kBlock / 16);
    for (int64_t ray = ((int64_t)blockIdx.x * kBlock + threadIdx.x) / 16; ray < n_rays; ray += groups) {
        int64_t start, count;
        rows_of(info, ray, rows, 0, start, count);
        for (int64_t k = threadIdx.x & 15; k < count; k += 16) {
            row_ray[start + k] = (int32_t)ray;
            row_pos[start + k] = (int32_t)k;
        }
    }
}

// One workgroup: the longest length, the sequences in each of 32 classes of length, and a place for every sequence behind the longer
// classes.  (Within a class the order is the LDS atomics'; nothing depends on it.)  4096 sequences take 9.6 us, latency, and spare a scan of
// them 65 us forward and 145 us backward (ragged, 2^18 rows of 64 channels).
constexpr int kClasses = 32;
__global__ __launch_bounds__(1024) void ray_order_kernel(const int64_t *__restrict__ info, int64_t n_rays, int64_t rows, int32_t *__restrict__ order) {
    __shared__ int longest, place[kClasses];
    const int tid = threadIdx.x;
    auto length = [&](int64_t r) {
        int64_t start, count;
        rows_of(info, r, rows, 0, start, count);
        return (int)count;
    };
    if (tid == 0) longest = 0;
    if (tid < kClasses) place[tid] = 0;
    __syncthreads();
    int most = 0;
#pragma unroll 4
    for (int64_t r = tid; r < n_rays; r += 1024) {
        const int n = length(r);
        most = n > most ? n : most;
    }
    atomicMax(&longest, most);
    __syncthreads();
    const float scale = (float)kClasses / (float)(longest + 1.0f);
    auto class_of = [&](int64_t r) {
        const int c = (int)((float)length(r) * scale);
        return c < kClasses ? kClasses - 1 - c : 0;
    };
#pragma unroll 4
    for (int64_t r = tid; r < n_rays; r += 1024) atomicAdd(&place[class_of(r)], 1);
    __syncthreads();
    if (tid == 0) {
        int sum = 0;
        for (int c = 0; c < kClasses; ++c) {
            const int n = place[c];
            place[c] = sum;
            sum += n;
        }
    }
    __syncthreads();
#pragma unroll 4
    for (int64_t r = tid; r < n_rays; r += 1024) order[atomicAdd(&place[class_of(r)], 1)] = (int32_t)r;
}

bool fits(const void *p, int64_t ld, int64_t bytes, int64_t vec) { return !p || ((uintptr_t)p % (vec * bytes) == 0 && ld % vec == 0); }

// calls f(T{}, integral W, integral VC)
template <class F>
void with_conv(int32_t dtype, int width, int vec, F &&f) {
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int full = 16 / (int)sizeof(T);
        auto by_width = [&](auto vc) {
            if (width == 2) f(t, std::integral_constant<int, 2>{}, vc);
            else if (width == 3) f(t, std::integral_constant<int, 3>{}, vc);
            else f(t, std::integral_constant<int, 4>{}, vc);
        };
        if (vec == full) by_width(std::integral_constant<int, full>{});
        else if (vec == 4) by_width(std::integral_constant<int, 4>{});
        else by_width(std::integral_constant<int, 1>{});
    });
}

constexpr int64_t kBwdGroups = 3 * kNumCU;      // workgroups (and partial sums) of a backward pass, at most: all resident

struct ConvPlan { int vec, lanes, piece; int64_t pieces, blocks_x, blocks_y; };
ConvPlan conv_plan(int64_t rows, int64_t channels, int vec, bool backward) {
    ConvPlan p;
    p.vec = vec;
    const int64_t vecs = ceil_div(channels, vec);
    p.lanes = 1;
    while (p.lanes < vecs && p.lanes < 64) p.lanes *= 2;
    p.blocks_y = ceil_div(vecs, p.lanes);
    // as many rows per wave as fill the chip's 3 x 1024 wave places once, at most 64 (then twice, ...): long pieces read their halo rows
    // rarely, and a launch of one and a third rounds takes two (43 rows against 32 at 32768 x 2048: 64 against 75 us)
    const int64_t each = ceil_div(ceil_div(rows * p.lanes * p.blocks_y, kWave), 3 * 4 * kNumCU);
    p.piece = (int)ceil_div(each, ceil_div(each, 64));
    if (p.piece < 4) p.piece = 4;
    p.pieces = ceil_div(rows, p.piece);
    p.blocks_x = ceil_div(p.pieces, kBlock / p.lanes);
    if (backward && p.blocks_x > ceil_div(kBwdGroups, p.blocks_y)) p.blocks_x = ceil_div(kBwdGroups, p.blocks_y);
    return p;
}

}  // namespace
}  // namespace nfa

using namespace nfa;

NFA_EXPORT int nfa_row_map(const int64_t *packed_info, int64_t n_rays, int64_t rows, int32_t *row_ray, int32_t *row_pos, void *stream) {
    NFA_REQUIRE(n_rays >= 0 && rows >= 0, "row_map: negative size");
    NFA_REQUIRE(n_rays < (1ll << 31) && rows < (1ll << 31), "row_map: more than 2^31 - 1 rays or rows");
    if (rows == 0) return NFA_OK;
    NFA_REQUIRE(row_ray && row_pos && (packed_info || n_rays == 0), "row_map: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(fill_map_kernel, dim3(blocks_for(rows)), dim3(kBlock), 0, s, row_ray, row_pos, rows);
    if (n_rays > 0) hipLaunchKernelGGL(row_map_kernel, dim3(blocks_for(n_rays * 16)), dim3(kBlock), 0, s, packed_info, n_rays, rows, row_ray, row_pos);
    return check_launch("row_map_kernel");
}

NFA_EXPORT int nfa_ray_order(const int64_t *packed_info, int64_t n_rays, int64_t rows, int32_t *order, void *stream) {
    NFA_REQUIRE(n_rays >= 0 && rows >= 0, "ray_order: negative size");
    NFA_REQUIRE(n_rays < (1ll << 31) && rows < (1ll << 31), "ray_order: more than 2^31 - 1 rays or rows");
    if (n_rays == 0) return NFA_OK;
    NFA_REQUIRE(packed_info && order, "ray_order: NULL pointer");
    hipLaunchKernelGGL(ray_order_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, packed_info, n_rays, rows, order);
    return check_launch("ray_order_kernel");
}

static int check_conv(const nfa_causal_conv_args *a, const char *who, bool step) {
    NFA_REQUIRE(a, "%s: NULL arguments", who);
    NFA_REQUIRE(a->n_rays >= 0 && a->rows >= 0 && a->channels >= 1 && a->channels <= (1 << 23), "%s: bad size", who);
    NFA_REQUIRE(a->width >= 2 && a->width <= 4, "%s: width must be 2, 3 or 4, got %d", who, a->width);
    NFA_REQUIRE(dtype_ok(a->dtype), "%s: bad dtype %d", who, a->dtype);
    NFA_REQUIRE(a->activation == NFA_ACT_NONE || a->activation == NFA_ACT_SILU, "%s: bad activation %d", who, a->activation);
    NFA_REQUIRE(a->rows < (1ll << 31) && a->n_rays < (1ll << 31), "%s: more than 2^31 - 1 rows or rays", who);
    if (step) return NFA_OK;
    NFA_REQUIRE(a->weight, "%s: NULL pointer", who);
    NFA_REQUIRE(a->packed_info || a->n_rays == 0 || a->rows % a->n_rays == 0, "%s: rows do not divide into equal sequences", who);
    NFA_REQUIRE(a->n_rays > 0 || a->packed_info || a->rows == 0, "%s: rows without sequences", who);
    NFA_REQUIRE(!a->packed_info || a->rows == 0 || (a->row_ray && a->row_pos), "%s: packed sequences need their row map", who);
    NFA_REQUIRE(a->rows == 0 || a->inputs, "%s: NULL pointer", who);
    NFA_REQUIRE(a->inputs_stride >= a->channels || a->rows <= 1, "%s: inputs_stride < channels", who);
    return NFA_OK;
}

static ConvArgs conv_args(const nfa_causal_conv_args *a) {
    ConvArgs d{};
    d.x = a->inputs; d.ld_x = a->inputs_stride;
    d.w = a->weight; d.bias = a->bias; d.init = a->initial_state;
    d.gy = a->grad_outputs; d.ld_gy = a->grad_outputs_stride; d.gfinal = a->grad_final_state;
    d.info = a->packed_info; d.ray = a->row_ray; d.pos = a->row_pos;
    d.rows = a->rows; d.n_rays = a->n_rays;
    d.length = a->n_rays > 0 ? a->rows / a->n_rays : 0;
    d.channels = a->channels; d.act = a->activation;
    return d;
}

NFA_EXPORT int nfa_causal_conv_fwd(const nfa_causal_conv_args *a, void *outputs, void *final_state, void *stream) {
    if (int rc = check_conv(a, "causal_conv_fwd", false)) return rc;
    NFA_REQUIRE(outputs || a->rows == 0, "causal_conv_fwd: NULL pointer");
    hipStream_t s = (hipStream_t)stream;
    ConvArgs d = conv_args(a);
    d.y = outputs;
    const int64_t bytes = dtype_bytes(a->dtype);
    // sixteen bytes to a thread where rows allow it (32768 x 2048 bf16 58 us, 66 with eight bytes; 2^18 x 128 fp32 48, 81 with four), else one
    // number
    int vec = (int)(16 / bytes);
    if (a->channels % vec || !fits(d.x, d.ld_x, bytes, vec) || !fits(outputs, 0, bytes, vec) || !fits(d.init, 0, bytes, vec)) vec = 1;
    if (a->rows > 0) {
        const ConvPlan p = conv_plan(a->rows, a->channels, vec, false);
        NFA_REQUIRE(p.blocks_x < kMaxThreads / kBlock && p.blocks_y < 65536, "causal_conv_fwd: too large for one launch");
        d.piece = p.piece; d.lanes = p.lanes; d.pieces = p.pieces;
        with_conv(a->dtype, a->width, vec, [&](auto t, auto w, auto vc) {
            using T = decltype(t);
            hipLaunchKernelGGL((conv_fwd_kernel<T, w(), vc()>), dim3((unsigned)p.blocks_x, (unsigned)p.blocks_y), dim3(kBlock), 0, s, d);
        });
        if (int rc = check_launch("conv_fwd_kernel")) return rc;
    }
    if (final_state && a->n_rays > 0) {
        with_conv(a->dtype, a->width, 1, [&](auto t, auto w, auto) {
            using T = decltype(t);
            const unsigned nb = blocks_for(a->n_rays * (a->width - 1) * a->channels);
            hipLaunchKernelGGL((conv_final_kernel<T, w()>), dim3(nb), dim3(kBlock), 0, s, d, (T *)final_state);
        });
        return check_launch("conv_final_kernel");
    }
    return NFA_OK;
}

NFA_EXPORT int64_t nfa_causal_conv_bwd_workspace_bytes(int64_t rows, int32_t channels, int32_t width, int32_t dtype) {
    if (rows <= 0 || channels <= 0) return 0;
    int64_t most = 1;                                        // of either vector width: which one runs depends on the pointers
    for (int vec : {1, 4}) {
        const ConvPlan p = conv_plan(rows, channels, vec, true);
        if (p.blocks_x > most) most = p.blocks_x;
    }
    return most * channels * (width + 1) * 4;
}

NFA_EXPORT int nfa_causal_conv_bwd(const nfa_causal_conv_args *a, void *grad_inputs, void *grad_weight, void *grad_bias,
                                   void *grad_initial_state, void *workspace, void *stream) {
    if (int rc = check_conv(a, "causal_conv_bwd", false)) return rc;
    NFA_REQUIRE(a->rows == 0 || a->grad_outputs, "causal_conv_bwd: NULL pointer");
    NFA_REQUIRE(a->grad_outputs_stride >= a->channels || a->rows <= 1, "causal_conv_bwd: grad_outputs_stride < channels");
    NFA_REQUIRE(!grad_initial_state || a->initial_state, "causal_conv_bwd: a gradient of no initial state");
    NFA_REQUIRE(workspace || a->rows == 0 || !(grad_weight || grad_bias), "causal_conv_bwd: NULL workspace");
    hipStream_t s = (hipStream_t)stream;
    ConvArgs d = conv_args(a);
    d.gx = grad_inputs;
    const int64_t bytes = dtype_bytes(a->dtype);
    // four channels to a thread: with eight, the windows, sums and weights of 16-bit channels do not fit the registers of three waves (2^18 x
    // 128 bf16 71 us, 433 with eight); one where rows are not aligned (fp32 111 us, 218 with one)
    int vec = 4;
    if (a->channels % vec || !fits(d.x, d.ld_x, bytes, vec) || !fits(d.gy, d.ld_gy, bytes, vec) || !fits(grad_inputs, 0, bytes, vec) ||
        !fits(d.init, 0, bytes, vec) || !fits(d.gfinal, 0, bytes, vec))
        vec = 1;
    if (a->rows == 0) {
        launch_zero(grad_weight, (int64_t)a->channels * a->width, a->dtype, s);
        launch_zero(grad_bias, a->channels, a->dtype, s);
        if (int rc = check_launch("zero_kernel")) return rc;
    }
    if (a->rows > 0 && (grad_inputs || grad_weight || grad_bias)) {
        const ConvPlan p = conv_plan(a->rows, a->channels, vec, true);
        NFA_REQUIRE(p.blocks_x < kMaxThreads / kBlock && p.blocks_y < 65536, "causal_conv_bwd: too large for one launch");
        d.piece = p.piece; d.lanes = p.lanes; d.pieces = p.pieces;
        d.partial = grad_weight || grad_bias ? (float *)workspace : nullptr;
        with_conv(a->dtype, a->width, vec, [&](auto t, auto w, auto vc) {
            using T = decltype(t);
            const size_t lds = (size_t)kBlock * (w() + 1) * vc() * 4;
            hipLaunchKernelGGL((conv_bwd_kernel<T, w(), vc()>), dim3((unsigned)p.blocks_x, (unsigned)p.blocks_y), dim3(kBlock), lds, s, d);
        });
        if (int rc = check_launch("conv_bwd_kernel")) return rc;
        if (grad_weight || grad_bias)
            launch_reduce_rows(d.partial, p.blocks_x, {{grad_weight, (int64_t)a->channels * a->width}, {grad_bias, a->channels}}, a->dtype, s);
        if (int rc = check_launch("reduce_rows_kernel")) return rc;
    }
    if (grad_initial_state && a->n_rays > 0) {
        with_conv(a->dtype, a->width, 1, [&](auto t, auto w, auto) {
            using T = decltype(t);
            hipLaunchKernelGGL((conv_init_grad_kernel<T, w()>), dim3(blocks_for(a->n_rays * a->channels)), dim3(kBlock), 0, s, d, (T *)grad_initial_state);
        });
        return check_launch("conv_init_grad_kernel");
    }
    return NFA_OK;
}

NFA_EXPORT int nfa_causal_conv_step(const nfa_causal_conv_args *a, const void *state, void *outputs, void *out_state, void *stream) {
    if (int rc = check_conv(a, "causal_conv_step", true)) return rc;
    if (a->n_rays == 0) return NFA_OK;
    NFA_REQUIRE(a->inputs && a->weight && state && outputs && out_state, "causal_conv_step: NULL pointer");
    NFA_REQUIRE(a->inputs_stride >= a->channels || a->n_rays <= 1, "causal_conv_step: inputs_stride < channels");
    ConvArgs d = conv_args(a);
    const int64_t bytes = dtype_bytes(a->dtype);
    int vec = (int)(16 / bytes);
    if (a->channels % vec || !fits(d.x, d.ld_x, bytes, vec) || !fits(state, 0, bytes, vec) || !fits(outputs, 0, bytes, vec) || !fits(out_state, 0, bytes, vec)) vec = 1;
    const dim3 grid((unsigned)ceil_div(ceil_div(a->channels, vec), kBlock), (unsigned)std::min<int64_t>(a->n_rays, 32768));
    with_conv(a->dtype, a->width, vec, [&](auto t, auto w, auto vc) {
        using T = decltype(t);
        hipLaunchKernelGGL((conv_step_kernel<T, w(), vc()>), grid, dim3(kBlock), 0, (hipStream_t)stream, d, (const T *)state, (T *)outputs, (T *)out_state);
    });
    return check_launch("conv_step_kernel");
}
