// dense.hip — a dense layer with its epilogue, and its backward pass, on the matrix units of gfx950.
//
//   y = act(x W^T + b) + r        x [M, K], W [N, K], b [N], r and y [M, N]
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz,  dr = dy
//
// One tile product serves the three.  out[p][q] = sum_c P(p, c) Q(q, c):
//   forward   p = m, q = n, c = k    P = x,  Q = W        both contiguous along c
//   dgrad     p = m, q = k, c = n    P = dz, Q = W        Q contiguous along q: read from LDS transposed
//   wgrad     p = n, q = k, c = m    P = dz, Q = x        both transposed; c is split over workgroups, partial sums joined in order
// dz is formed from dy and the saved number while a tile is staged: it never goes to memory.
//
// A field's layers are narrow (8 .. 256 features) and their batches long (2^18 samples): reading x and writing y bounds them, so a
// workgroup takes 128 rows of samples and the whole width where it can, x goes through the chip once, and everything elementwise
// rides on the tile in registers.
#include "feature.hpp"

namespace nfa {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kRowBytes = 128;                  // of the contraction axis in one staged tile: 64 16-bit or 32 32-bit numbers
template <class T> constexpr int kChunk = 16 / (int)sizeof(T);           // numbers in one 16-byte access
template <class T> constexpr int kStage = kRowBytes / (int)sizeof(T);    // contraction steps in one staged tile

struct DenseArgs {
    const void *p, *q, *saved, *bias, *residual;
    void *out, *saved_out;
    float *partial;                             // wgrad: [splits][P * Q + P]
    int64_t n_p, n_c;                           // rows of the output; length of the contraction
    int32_t n_q;
    int64_t ld_p, ld_q, ld_saved, ld_residual;  // in elements
    int64_t split;                              // wgrad: contraction steps of one workgroup
    int32_t act, vec_p, vec_q, vec_out, want_bias, tiles_q, tiles;
};

enum { kForward, kDgrad, kWgrad };

// sixteen bytes of a row, zero outside it; `vec`: every row starts on 16 bytes and holds whole chunks
template <class T>
__device__ __forceinline__ u32x4 load_chunk(const T *row, int64_t col, int64_t cols, bool inside, bool vec) {
    u32x4 v = {0, 0, 0, 0};
    if (vec) {
        if (inside && col < cols) v = *reinterpret_cast<const u32x4 *>(row + col);
    } else if (inside) {
        T e[kChunk<T>];
#pragma unroll
        for (int i = 0; i < kChunk<T>; ++i) e[i] = col + i < cols ? row[col + i] : T(0.0f);
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

// LDS layouts.  c-contiguous tiles: 128-byte rows, the 16-byte chunks of row r exchanged by r & 7.  Transposed tiles (rows along c,
// 64 or 128 columns): the 32-byte (16-bit types) or 64-byte units of a row exchanged so that the rows that one instruction reads
// lie in different banks.
template <class T, int COLS>
__device__ __forceinline__ int unit_swizzle(int row) {
    if (sizeof(T) == 4) return (row >> 2) & 3;
    if (COLS == 128) return (row & 3) | (((row >> 3) & 1) << 2);
    return ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
}
template <class T, bool TR, int ROWS>
__device__ __forceinline__ int stage_offset(int row, int chunk) {        // byte offset of a chunk in its tile
    if (!TR) return row * kRowBytes + ((chunk ^ (row & 7)) << 4);
    if (sizeof(T) == 4) return row * ROWS * 4 + (((chunk >> 2) ^ unit_swizzle<T, ROWS>(row)) << 6) + ((chunk & 3) << 4);
    return row * ROWS * 2 + (((chunk >> 1) ^ unit_swizzle<T, ROWS>(row)) << 5) + ((chunk & 1) << 4);
}

template <class T> struct Frag { T v[kChunk<T>]; };

// the sixteen bytes that lane l feeds to the matrix units for rows (or columns) c0 .. c0 + 15 and half `ks` of the tile
template <class T, bool TR, int ROWS>
__device__ __forceinline__ u32x4 read_frag(const char *tile, int c0, int ks, int lane) {
    const int i = lane & 15, g = lane >> 4;
    u32x4 v;
    if (!TR) {
        v = *reinterpret_cast<const u32x4 *>(tile + stage_offset<T, false, ROWS>(c0 + i, ks * 4 + g));
    } else if (sizeof(T) == 4) {
        float e[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int row = ks * 16 + g * 4 + s;
            e[s] = *reinterpret_cast<const float *>(tile + row * ROWS * 4 + (((c0 >> 4) ^ unit_swizzle<T, ROWS>(row)) << 6) + (i << 2));
        }
        __builtin_memcpy(&v, e, 16);
    } else {
        // ds_read_b64_tr_b16: sixteen lanes read four rows of sixteen columns, lane i gets column i of the four
        s16x4 h[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int row = ks * 32 + g * 8 + s * 4 + (i >> 2);
            const char *at = tile + row * ROWS * 2 + (((c0 >> 4) ^ unit_swizzle<T, ROWS>(row)) << 5) + ((i & 3) << 3);
            h[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
        }
        s16x8 w = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
        __builtin_memcpy(&v, &w, 16);
    }
    return v;
}

// acc[q][p] += Q P over the lane's chunk.  32-bit numbers go in four steps: the contraction may run in any order as long as both
// sides agree, so lane group g feeds chunk g and each step takes one number of it.
template <class T>
__device__ __forceinline__ f32x4 multiply(u32x4 q, u32x4 p, f32x4 acc) {
    if constexpr (std::is_same_v<T, bf16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), acc, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, f16>) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q), __builtin_bit_cast(f16x8, p), acc, 0, 0, 0);
    } else {
        const f32x4 a = __builtin_bit_cast(f32x4, q), b = __builtin_bit_cast(f32x4, p);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], acc, 0, 0, 0);
        return acc;
    }
}

template <class T, int MODE, int BP, int BQ>
__global__ __launch_bounds__(kBlock) void dense_kernel(DenseArgs a) {
    constexpr bool PT = MODE == kWgrad, QT = MODE != kForward, FUSE = MODE != kForward;
    constexpr int CE = kChunk<T>, ST = kStage<T>;
    constexpr int NP = BP / 32, NQ = BQ / 32;               // chunks a thread stages per tile = 16-wide fragments per wave
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int wp = wave >> 1, wq = wave & 1;

    // tile of this workgroup: eight runs of tiles, one per XCD (workgroups are dealt to them in turn), so that the column tiles of
    // a row tile share an L2
    int tile = blockIdx.x;
    const int per = (a.tiles + kNumXCD - 1) / kNumXCD;
    tile = (tile % kNumXCD) * per + tile / kNumXCD;
    if (tile >= a.tiles) return;
    const int64_t p0 = (int64_t)(tile / a.tiles_q) * BP;
    const int q0 = (tile % a.tiles_q) * BQ;
    const int64_t c_begin = MODE == kWgrad ? (int64_t)blockIdx.y * a.split : 0;
    const int64_t c_end = MODE == kWgrad ? (c_begin + a.split < a.n_c ? c_begin + a.split : a.n_c) : a.n_c;

    const T *P = reinterpret_cast<const T *>(a.p), *Q = reinterpret_cast<const T *>(a.q), *S = reinterpret_cast<const T *>(a.saved);
    u32x4 rp[NP], rs[NP], rq[NQ];
    f32x4 acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    float db[FUSE ? CE : 1];
#pragma unroll
    for (int i = 0; i < (FUSE ? CE : 1); ++i) db[i] = 0.0f;

    // which row and chunk of a tile this thread stages in its k-th turn
    auto place = [&](bool tr, int rows, int k, int &row, int &chunk) {
        const int per_row = tr ? rows / CE : 8;
        chunk = tid % per_row;
        row = tid / per_row + k * (kBlock / per_row);
    };
    auto load = [&](int64_t c) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            int row, chunk;
            place(PT, BP, k, row, chunk);
            const int64_t r = PT ? c + row : p0 + row, col = PT ? p0 + chunk * CE : c + chunk * CE;
            const int64_t rows = PT ? c_end : a.n_p, cols = PT ? a.n_p : a.n_c;
            rp[k] = load_chunk<T>(P + r * a.ld_p, col, cols, r < rows, a.vec_p);
            if (FUSE && a.act != NFA_ACT_NONE) rs[k] = load_chunk<T>(S + r * a.ld_saved, col, cols, r < rows, a.vec_p);
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
            int row, chunk;
            place(QT, BQ, k, row, chunk);
            const int64_t r = QT ? c + row : q0 + row, col = QT ? q0 + chunk * CE : c + chunk * CE;
            const int64_t rows = QT ? c_end : a.n_q, cols = QT ? a.n_q : a.n_c;
            rq[k] = load_chunk<T>(Q + r * a.ld_q, col, cols, r < rows, a.vec_q);
        }
    };
    auto store = [&](char *buf) {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            int row, chunk;
            place(PT, BP, k, row, chunk);
            if (FUSE) {
                Frag<T> g = __builtin_bit_cast(Frag<T>, rp[k]);
                if (a.act != NFA_ACT_NONE) {
                    const Frag<T> s = __builtin_bit_cast(Frag<T>, rs[k]);
#pragma unroll
                    for (int i = 0; i < CE; ++i) {
                        const float dz = to_f(g.v[i]) * act_slope(a.act, to_f(s.v[i]));
                        if (MODE == kWgrad) db[i] += dz;
                        g.v[i] = from_f<T>(dz);             // rounded: the matrix units take T
                    }
                    rp[k] = __builtin_bit_cast(u32x4, g);
                } else if (MODE == kWgrad) {
#pragma unroll
                    for (int i = 0; i < CE; ++i) db[i] += to_f(g.v[i]);
                }
            }
            *reinterpret_cast<u32x4 *>(buf + stage_offset<T, PT, BP>(row, chunk)) = rp[k];
        }
#pragma unroll
        for (int k = 0; k < NQ; ++k) {
            int row, chunk;
            place(QT, BQ, k, row, chunk);
            *reinterpret_cast<u32x4 *>(buf + BP * kRowBytes + stage_offset<T, QT, BQ>(row, chunk)) = rq[k];
        }
    };
    auto compute = [&](const char *buf, int64_t c) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (c + ks * (ST / 2) >= c_end) break;          // a half that holds only zeros
            u32x4 fp[NP], fq[NQ];
#pragma unroll
            for (int i = 0; i < NP; ++i) fp[i] = read_frag<T, PT, BP>(buf, wp * (BP / 2) + i * 16, ks, lane);
#pragma unroll
            for (int j = 0; j < NQ; ++j) fq[j] = read_frag<T, QT, BQ>(buf + BP * kRowBytes, wq * (BQ / 2) + j * 16, ks, lane);
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < NQ; ++j) acc[i][j] = multiply<T>(fq[j], fp[i], acc[i][j]);
        }
    };

    constexpr int kBuf = (BP + BQ) * kRowBytes;
    load(c_begin);
    store(lds);
    __syncthreads();
    int cur = 0;
    for (int64_t c = c_begin; c < c_end; c += ST) {
        const bool more = c + ST < c_end;
        if (more) load(c + ST);
        compute(lds + cur * kBuf, c);
        if (more) store(lds + (cur ^ 1) * kBuf);
        __syncthreads();
        cur ^= 1;
    }

    // lane l holds row p = l % 16 of each fragment and four neighbouring columns q
    const int i = lane & 15, g = lane >> 4;
    if (MODE == kWgrad) {
        float *part = a.partial + (int64_t)blockIdx.y * (a.n_p * a.n_q + a.n_p);
#pragma unroll
        for (int pi = 0; pi < NP; ++pi)
#pragma unroll
            for (int qi = 0; qi < NQ; ++qi) {
                const int64_t p = p0 + wp * (BP / 2) + pi * 16 + i;
                const int q = q0 + wq * (BQ / 2) + qi * 16 + g * 4;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (p < a.n_p && q + r < a.n_q) part[p * a.n_q + q + r] = acc[pi][qi][r];
            }
        if (q0 == 0 && a.want_bias) {                       // db: the threads that staged the same columns, in order
            constexpr int per_row = BP / CE, n = kBlock / per_row;
            float *sum = reinterpret_cast<float *>(lds);
#pragma unroll
            for (int e = 0; e < CE; ++e) sum[(tid / per_row) * BP + (tid % per_row) * CE + e] = db[e];
            __syncthreads();
            if (tid < BP && p0 + tid < a.n_p) {
                float v = 0.0f;
                for (int k = 0; k < n; ++k) v += sum[k * BP + tid];
                part[a.n_p * a.n_q + p0 + tid] = v;
            }
        }
        return;
    }
    T *out = reinterpret_cast<T *>(a.out), *kept = reinterpret_cast<T *>(a.saved_out);
    const T *bias = reinterpret_cast<const T *>(a.bias), *res = reinterpret_cast<const T *>(a.residual);
    struct alignas(4 * sizeof(T)) V4 { T v[4]; };
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
        const int q = q0 + wq * (BQ / 2) + qi * 16 + g * 4;
        float b[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = (MODE == kForward && bias && q + r < a.n_q) ? to_f(bias[q + r]) : 0.0f;
#pragma unroll
        for (int pi = 0; pi < NP; ++pi) {
            const int64_t p = p0 + wp * (BP / 2) + pi * 16 + i;
            if (p >= a.n_p || q >= a.n_q) continue;
            V4 y, k;
            if (MODE == kForward) {
                V4 add{};
                if (res) {
                    if (a.vec_out) add = *reinterpret_cast<const V4 *>(res + p * a.ld_residual + q);
                    else
#pragma unroll
                        for (int r = 0; r < 4; ++r) add.v[r] = q + r < a.n_q ? res[p * a.ld_residual + q + r] : T(0.0f);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float z = acc[pi][qi][r] + b[r], v = act_fwd(a.act, z);
                    k.v[r] = from_f<T>(a.want_bias ? v : z);        // (forward: want_bias = the saved number is act(z))
                    y.v[r] = from_f<T>(res ? v + to_f(add.v[r]) : v);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) y.v[r] = from_f<T>(acc[pi][qi][r]);
            }
            if (a.vec_out) {
                *reinterpret_cast<V4 *>(out + p * a.n_q + q) = y;
                if (MODE == kForward && kept) *reinterpret_cast<V4 *>(kept + p * a.n_q + q) = k;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (q + r < a.n_q) {
                        out[p * a.n_q + q + r] = y.v[r];
                        if (MODE == kForward && kept) kept[p * a.n_q + q + r] = k.v[r];
                    }
            }
        }
    }
}

// columns by lane, sixteen rows side by side; a column's sum is formed in the same order every time
template <class T>
__global__ __launch_bounds__(1024) void reduce_rows_kernel(const float *__restrict__ part, int64_t rows, int64_t cols, int64_t ld,
                                                           T *__restrict__ out) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float v = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t r = grp; r < rows; r += 16) v += part[r * ld + c];
    }
    sum[grp][lane] = v;
    __syncthreads();
    if (grp == 0 && c < cols) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += sum[k][lane];
        out[c] = from_f<T>(t);
    }
}

bool aligned(const void *p, int64_t ld, int64_t cols, int64_t bytes, int64_t to) {
    return (uintptr_t)p % to == 0 && ld * bytes % to == 0 && cols * bytes % to == 0;
}

template <class T, int MODE, int BP, int BQ>
int launch_tiles(DenseArgs a, int64_t splits, hipStream_t s) {
    const int64_t tiles_p = ceil_div(a.n_p, BP);
    a.tiles_q = (int32_t)ceil_div(a.n_q, BQ);
    NFA_REQUIRE(tiles_p * a.tiles_q < (1 << 30), "linear: too many rows for one launch");
    a.tiles = (int32_t)(tiles_p * a.tiles_q);
    const int64_t steps = MODE == kWgrad ? a.split : a.n_c;
    const size_t bytes = (size_t)(BP + BQ) * kRowBytes * (steps > kStage<T> ? 2 : 1);
    const dim3 grid((unsigned)(ceil_div(a.tiles, kNumXCD) * kNumXCD), (unsigned)splits);
    hipLaunchKernelGGL((dense_kernel<T, MODE, BP, BQ>), grid, dim3(kBlock), bytes, s, a);
    return check_launch("dense_kernel");
}

// rows of the long axis that one workgroup of the weight gradient sums: enough workgroups for every CU twice, and not so many that
// their partial sums (a whole weight each) outweigh the rows read
struct WgradPlan { int64_t split, splits, bp, bq; };
WgradPlan wgrad_plan(int64_t rows, int64_t n, int64_t k, int32_t dtype) {
    const int64_t stage = dtype == NFA_DTYPE_F32 ? 32 : 64;
    WgradPlan w;
    w.bp = n <= 64 ? 64 : 128;
    w.bq = k <= 64 ? 64 : 128;
    const int64_t tiles = ceil_div(n, w.bp) * ceil_div(k, w.bq);
    int64_t splits = ceil_div(2 * kNumCU, tiles);
    const int64_t most = ceil_div(rows, 4 * stage);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    w.split = ceil_div(ceil_div(rows, splits), stage) * stage;
    w.splits = ceil_div(rows, w.split);
    return w;
}

}  // namespace

void launch_reduce_rows(const float *part, int64_t rows, int64_t cols, int64_t ld, void *out, int32_t dtype, hipStream_t s) {
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((reduce_rows_kernel<T>), dim3((unsigned)ceil_div(cols, 64)), dim3(1024), 0, s, part, rows, cols, ld, (T *)out);
    });
}

}  // namespace nfa

using namespace nfa;

static int check_linear(const nfa_linear_args *a, const char *who) {
    NFA_REQUIRE(a, "%s: NULL arguments", who);
    NFA_REQUIRE(a->rows >= 0 && a->in_features >= 1 && a->out_features >= 1, "%s: bad size %lld x %d x %d", who, (long long)a->rows,
                a->in_features, a->out_features);
    NFA_REQUIRE(a->in_features <= (1 << 20) && a->out_features <= (1 << 20), "%s: more than 2^20 features", who);
    NFA_REQUIRE(dtype_ok(a->dtype), "%s: bad dtype %d", who, a->dtype);
    NFA_REQUIRE(act_ok(a->activation), "%s: bad activation %d", who, a->activation);
    if (a->rows == 0) return NFA_OK;
    NFA_REQUIRE(a->inputs && a->weight, "%s: NULL pointer", who);
    NFA_REQUIRE(a->inputs_stride >= a->in_features || a->rows == 1, "%s: inputs_stride %lld < in_features", who, (long long)a->inputs_stride);
    return NFA_OK;
}

NFA_EXPORT int64_t nfa_linear_saved_bytes(int64_t rows, int32_t out_features, int32_t dtype, int32_t activation, int32_t has_residual) {
    if (activation == NFA_ACT_NONE || (act_from_value(activation) && !has_residual)) return 0;
    return rows * out_features * dtype_bytes(dtype);
}

NFA_EXPORT int nfa_linear_fwd(const nfa_linear_args *a, void *outputs, void *saved, void *stream) {
    if (int rc = check_linear(a, "linear_fwd")) return rc;
    if (a->rows == 0) return NFA_OK;
    NFA_REQUIRE(outputs, "linear_fwd: NULL pointer");
    NFA_REQUIRE(!a->residual || a->residual_stride >= a->out_features || a->rows == 1, "linear_fwd: residual_stride < out_features");
    const int64_t bytes = dtype_bytes(a->dtype);
    DenseArgs d{};
    d.p = a->inputs; d.ld_p = a->inputs_stride;
    d.q = a->weight; d.ld_q = a->in_features;
    d.bias = a->bias; d.residual = a->residual; d.ld_residual = a->residual_stride;
    d.out = outputs; d.saved_out = saved;
    d.n_p = a->rows; d.n_q = a->out_features; d.n_c = a->in_features;
    d.act = a->activation;
    d.want_bias = act_from_value(a->activation);
    d.vec_p = aligned(d.p, d.ld_p, a->in_features, bytes, 16);
    d.vec_q = aligned(d.q, d.ld_q, a->in_features, bytes, 16);
    d.vec_out = aligned(outputs, d.n_q, d.n_q, bytes, 4 * bytes) && (!saved || aligned(saved, d.n_q, d.n_q, bytes, 4 * bytes)) &&
                (!a->residual || aligned(a->residual, a->residual_stride, d.n_q, bytes, 4 * bytes));
    int rc = NFA_OK;
    with_dtype(a->dtype, [&](auto t) {
        using T = decltype(t);
        rc = d.n_q <= 64 ? launch_tiles<T, kForward, 128, 64>(d, 1, (hipStream_t)stream)
                         : launch_tiles<T, kForward, 128, 128>(d, 1, (hipStream_t)stream);
    });
    return rc;
}

NFA_EXPORT int64_t nfa_linear_bwd_workspace_bytes(int64_t rows, int32_t in_features, int32_t out_features, int32_t dtype) {
    if (rows <= 0 || in_features <= 0 || out_features <= 0) return 0;
    const WgradPlan w = wgrad_plan(rows, out_features, in_features, dtype);
    return w.splits * ((int64_t)out_features * in_features + out_features) * 4;
}

NFA_EXPORT int nfa_linear_bwd(const nfa_linear_args *a, const void *saved, void *grad_inputs, void *grad_weight, void *grad_bias,
                              void *workspace, void *stream) {
    if (int rc = check_linear(a, "linear_bwd")) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (a->rows == 0) return NFA_OK;
    NFA_REQUIRE(a->grad_outputs, "linear_bwd: NULL pointer");
    NFA_REQUIRE(a->grad_outputs_stride >= a->out_features || a->rows == 1, "linear_bwd: grad_outputs_stride < out_features");
    NFA_REQUIRE(saved || a->activation == NFA_ACT_NONE, "linear_bwd: the activation needs what the forward call saved");
    NFA_REQUIRE(workspace || !(grad_weight || grad_bias), "linear_bwd: NULL workspace");
    const int64_t bytes = dtype_bytes(a->dtype), n = a->out_features, k = a->in_features;
    const bool vec_g = aligned(a->grad_outputs, a->grad_outputs_stride, n, bytes, 16) && (!saved || aligned(saved, n, n, bytes, 16));
    DenseArgs d{};
    d.p = a->grad_outputs; d.ld_p = a->grad_outputs_stride;
    d.saved = saved; d.ld_saved = n;
    d.act = a->activation;
    d.vec_p = vec_g;
    int rc = NFA_OK;
    if (grad_inputs) {
        DenseArgs e = d;
        e.q = a->weight; e.ld_q = k;
        e.vec_q = aligned(a->weight, k, k, bytes, 16);
        e.out = grad_inputs;
        e.vec_out = aligned(grad_inputs, k, k, bytes, 4 * bytes);
        e.n_p = a->rows; e.n_q = (int32_t)k; e.n_c = n;
        with_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            rc = k <= 64 ? launch_tiles<T, kDgrad, 128, 64>(e, 1, s) : launch_tiles<T, kDgrad, 128, 128>(e, 1, s);
        });
        if (rc) return rc;
    }
    if (grad_weight || grad_bias) {
        const WgradPlan w = wgrad_plan(a->rows, n, k, a->dtype);
        DenseArgs e = d;
        e.q = a->inputs; e.ld_q = a->inputs_stride;
        e.vec_q = aligned(a->inputs, a->inputs_stride, k, bytes, 16);
        e.partial = (float *)workspace;
        e.n_p = n; e.n_q = (int32_t)k; e.n_c = a->rows;
        e.split = w.split;
        e.want_bias = grad_bias != nullptr;
        with_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            if (w.bp == 64) rc = w.bq == 64 ? launch_tiles<T, kWgrad, 64, 64>(e, w.splits, s) : launch_tiles<T, kWgrad, 64, 128>(e, w.splits, s);
            else rc = w.bq == 64 ? launch_tiles<T, kWgrad, 128, 64>(e, w.splits, s) : launch_tiles<T, kWgrad, 128, 128>(e, w.splits, s);
        });
        if (rc) return rc;
        const int64_t ld = n * k + n;
        if (grad_weight) launch_reduce_rows(e.partial, w.splits, n * k, ld, grad_weight, a->dtype, s);
        if (grad_bias) launch_reduce_rows(e.partial + n * k, w.splits, n, ld, grad_bias, a->dtype, s);
        return check_launch("reduce_rows_kernel");
    }
    return NFA_OK;
}
