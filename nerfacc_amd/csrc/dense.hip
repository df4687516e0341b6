// dense.hip — a dense layer with its epilogue, and its backward pass, on the matrix units of gfx950.
//
//   y = act(x W^T + b) + r        x [M, K], W [N, K], b [N], r and y [M, N]
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_m dz,  dr = dy
//
// One tile product serves the three.  out[p][q] = sum_c P(p, c) Q(q, c):
//   forward   p = m, q = n, c = k    P = x,  Q = W        both contiguous along c
//   dgrad     p = m, q = k, c = n    P = dz, Q = W        Q contiguous along q: read from LDS transposed
//   wgrad     p = n, q = k, c = m    P = dz, Q = x        both transposed; c is split over workgroups, partial sums joined in order
// dz is formed from dy and act' (or relu's bit) while a tile is staged: it never goes to memory.  In 16-bit types a smooth activation's dz
// is multiplied in two parts.
//
// A field's layers are narrow (8 .. 256 features) and their batches long (2^18 samples): reading x and writing y bounds them.  For
// a contraction of up to 256 the forward pass and dgrad keep the weight in LDS for the life of a workgroup and every wave takes rows
// straight from memory into the registers that feed the matrix units: no barrier after the first, x read once, everything elementwise
// in registers (resident_kernel).  Longer contractions and wgrad go tile by tile through LDS (tile_kernel); few rows, and few outputs of
// a long contraction, go through neither (stream_kernel); the weight gradient of a narrow layer in 32 bits is summed straight from
// memory (narrow_wgrad_kernel).
//
// On one MI355X (copies reach 5.1 TB/s, tuned ones 6.2; large library products 1335 TF bf16, 153 TF fp32), kernels alone:
//   2^18 x 256 -> 256 bf16, relu + residual: forward 100 us (410 MB: 4.1 TB/s), dgrad 93 us (276 MB), wgrad 90 us + 8 to join
//   2^18 x 8 -> 32 fp32, relu: 15, 15 and 13 us + 4;   100003 x 63 -> 65 fp16, softplus, no row aligned: 29, 27 and 27 us + 4
//   2^18 x 256 -> 256 silu, training: fp16 131 + 155 + 184 us, bf16 108 + 148 + 182 (relu 77 + 85 + 92: one product, a bit a number)
//   65536 x 1024 -> 1024 bf16, silu: 186 us, 740 TF;   1 x 256 -> 256 bf16: 4.6 us a call
#include "feature.hpp"

#include <algorithm>

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
    int64_t ld_p, ld_q, ld_saved, ld_residual;  // in elements (ld_saved of bits: in bytes)
    int64_t split;                              // wgrad: contraction steps of one workgroup
    int32_t act, mask, vec, want_bias, tiles_q, tiles, block_q, splits;
};

enum { kForward, kDgrad, kWgrad };

// Sixteen bytes of row `row`.  VEC: every row starts on 16 bytes and holds whole chunks; the load is then made in any case, from a place
// that exists, so that a tile's loads are one block without branches, and only_inside() clears what lies outside the array where the
// value is used: a select right behind the load would wait for it.  Otherwise sixteen bytes at the alignment of a number (global memory
// takes that), with zeros behind the row's end; number by number only at the end of the array.
template <class T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const T *base, int64_t row, int64_t rows, int64_t ld, int64_t col, int64_t cols) {
    if constexpr (VEC) {
        return *reinterpret_cast<const u32x4 *>(base + (row < rows ? row : rows - 1) * ld + (col < cols ? col : 0));
    } else {
        u32x4 v = {0, 0, 0, 0};
        if (row < rows && col < cols) {
            T e[kChunk<T>];
            base += row * ld + col;
            if ((row - rows + 1) * ld + col + kChunk<T> <= cols) {          // the array holds sixteen bytes from here on
                __builtin_memcpy(&v, base, 16);
                if (col + kChunk<T> > cols) {
                    __builtin_memcpy(e, &v, 16);
#pragma unroll
                    for (int i = 0; i < kChunk<T>; ++i) e[i] = col + i < cols ? e[i] : T(0.0f);
                    __builtin_memcpy(&v, e, 16);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kChunk<T>; ++i) e[i] = col + i < cols ? base[i] : T(0.0f);
                __builtin_memcpy(&v, e, 16);
            }
        }
        return v;
    }
}
template <bool VEC>
__device__ __forceinline__ u32x4 only_inside(u32x4 v, bool inside) {
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = inside ? v[i] : 0;
    }
    return v;
}
// of what is kept for one chunk of a smooth activation: 16-byte chunks (fp16: eight slopes in 32 bits)
template <class T> constexpr int kKept = std::is_same_v<T, f16> ? 2 : 1;
template <class T, bool SPLIT> constexpr int kSaved = SPLIT ? kKept<T> : 1;
// what dz is formed from beside dy: kept numbers, or a byte of relu's bits
template <class T, bool SPLIT, bool VEC>
__device__ __forceinline__ void load_saved(const DenseArgs &a, int64_t row, int64_t rows, int64_t col, int64_t cols, u32x4 *v) {
    v[0] = u32x4{0, 0, 0, 0};
    if constexpr (kSaved<T, SPLIT> == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = load_chunk<float, VEC>(reinterpret_cast<const float *>(a.saved), row, rows, a.ld_saved, col + 4 * i, cols);
    } else if (a.mask) {
        const bool inside = row < rows && col < cols;
        v[0][0] = reinterpret_cast<const uint8_t *>(a.saved)[inside ? row * a.ld_saved + col / kChunk<T> : 0];
    } else if (a.act != NFA_ACT_NONE) {
        v[0] = load_chunk<T, VEC>(reinterpret_cast<const T *>(a.saved), row, rows, a.ld_saved, col, cols);
    }
}

template <class T> struct Frag { T v[kChunk<T>]; };

// Smooth activations of 16-bit types: the product is taken of dz in two parts, so that a gradient carries the rounding of its own result and,
// in bf16, of act' only.  The parts are bf16 for fp16 too, whose own range dz leaves at both ends: the gradient of a mean over 2^18 rows
// is below fp16's smallest step, exp' under a loss scale above its largest number.  dz = high + low to 2^-17.  The other side is exact in
// bf16's one part, and in fp16's two (11 bits in 8 + 8); of its four products the one of both second parts, 2^-18 of the term, is left out.
constexpr float kLargest = 0x1.fep127f;         // of bf16
template <class T, bool SPLIT> constexpr bool kSplitBoth = SPLIT && std::is_same_v<T, f16>;
template <class T, bool SPLIT> using Fed = std::conditional_t<SPLIT, bf16, T>;      // what the matrix units multiply

// a chunk of fp16 in two parts; infinity is 1 + infinity, whose products with dz's parts are infinities of one sign
__device__ __forceinline__ void split_chunk(u32x4 v, u32x4 &high, u32x4 &low) {
    const Frag<f16> x = __builtin_bit_cast(Frag<f16>, v);
    Frag<bf16> h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = to_f(x.v[i]);
        const bool inf = fabsf(f) > 65504.0f;
        h.v[i] = from_f<bf16>(inf ? copysignf(1.0f, f) : f);
        l.v[i] = from_f<bf16>(inf ? f : f - to_f(h.v[i]));
    }
    high = __builtin_bit_cast(u32x4, h);
    low = __builtin_bit_cast(u32x4, l);
}

// dz = dy act'(.) of N chunks, rounded to what is multiplied.  SPLIT: what the rounding lost goes into `rest`.  relu's dz is dy or 0:
// nothing is lost there.  What rounds to infinity becomes bf16's largest number and a rest, which is infinite where dz is (infinity minus
// infinity would be NaN).  each(chunk, dz of one number in 32 bits, place in the chunk)
template <class T, bool SPLIT, int N, class F>
__device__ __forceinline__ void form_dz(const DenseArgs &a, u32x4 (&g)[N], const u32x4 (&s)[N * kSaved<T, SPLIT>], u32x4 (&rest)[SPLIT ? N : 1], F &&each) {
    auto with = [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const Frag<T> v = __builtin_bit_cast(Frag<T>, g[k]);
            Frag<Fed<T, SPLIT>> hi, lo;
            float w[kChunk<T>];
#pragma unroll
            for (int i = 0; i < kChunk<T>; ++i) {
                if constexpr (kSaved<T, SPLIT> == 2) w[i] = __builtin_bit_cast(Frag<float>, s[2 * k + i / 4]).v[i % 4];
                else w[i] = to_f(__builtin_bit_cast(Frag<T>, s[k]).v[i]);
            }
#pragma unroll
            for (int i = 0; i < kChunk<T>; ++i) {
                float dz = to_f(v.v[i]);
                if constexpr (SPLIT) dz *= ACT == NFA_ACT_SOFTPLUS ? -expm1f(-w[i]) : w[i];          // (ACT: bf16's softplus keeps its value)
                else if constexpr (ACT == NFA_ACT_RELU) dz = (a.mask ? ((s[k][0] >> i) & 1u) == 0 : w[i] <= 0.0f) ? 0.0f : dz;
                else if constexpr (ACT != NFA_ACT_NONE) dz *= act_slope_of_kept<ACT>(w[i]);
                each(k, dz, i);
                if constexpr (SPLIT) hi.v[i] = from_f<bf16>(fabsf(dz) > kLargest ? copysignf(kLargest, dz) : dz);
                else hi.v[i] = from_f<T>(dz);
                if constexpr (SPLIT) lo.v[i] = from_f<bf16>(dz - to_f(hi.v[i]));
            }
            if constexpr (SPLIT || ACT != NFA_ACT_NONE) g[k] = __builtin_bit_cast(u32x4, hi);
            if constexpr (SPLIT) rest[k] = __builtin_bit_cast(u32x4, lo);
        }
    };
    if constexpr (sizeof(T) == 4) {
        with_act(a.act, with);
    } else if constexpr (SPLIT) {
        if (std::is_same_v<T, bf16> && a.act == NFA_ACT_SOFTPLUS) with(std::integral_constant<int, NFA_ACT_SOFTPLUS>{});
        else with(std::integral_constant<int, NFA_ACT_NONE>{});
    } else {
        if (a.act == NFA_ACT_RELU) with(std::integral_constant<int, NFA_ACT_RELU>{});
        else with(std::integral_constant<int, NFA_ACT_NONE>{});
    }
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
// ds_read_b64_tr_b16: sixteen lanes read four rows of four times four columns, lane i gets the i-th column of the four rows
__device__ __forceinline__ s16x4 read_transposed(const char *at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
}

// y = act(z) (+ residual) of N chunks in place; `kept`: what the backward pass wants of them (bits: in the first word of a chunk)
template <class T, int N>
__device__ __forceinline__ void finish_chunks(const DenseArgs &a, float (&z)[N][kChunk<T>], const u32x4 (&res)[N], u32x4 (&y)[N],
                                              u32x4 (&kept)[N * kKept<T>]) {
    with_act(a.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        constexpr bool SMOOTH = ACT != NFA_ACT_NONE && ACT != NFA_ACT_RELU;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            Frag<T> out, keep;
            Frag<float> slope[2];
            const Frag<T> add = __builtin_bit_cast(Frag<T>, res[k]);
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < kChunk<T>; ++i) {
                const float v = act_fwd<ACT>(z[k][i]);
                out.v[i] = from_f<T>(a.residual ? v + to_f(add.v[i]) : v);
                if constexpr (ACT == NFA_ACT_RELU) bits |= (v <= 0.0f ? 0u : 1u) << i;     // (NaN passes its gradient on)
                z[k][i] = ACT == NFA_ACT_RELU || ACT == NFA_ACT_EXP || (ACT == NFA_ACT_SOFTPLUS && kKept<T> == 1) ? v : z[k][i];
            }
            y[k] = __builtin_bit_cast(u32x4, out);
            if (!a.saved_out) continue;
#pragma unroll
            for (int i = 0; i < kChunk<T>; ++i) {           // (exp: z is its value by now)
                if constexpr (SMOOTH && kKept<T> == 2) slope[i / 4].v[i % 4] = ACT == NFA_ACT_EXP ? z[k][i] : act_slope<ACT>(z[k][i]);
                else if constexpr (SMOOTH && sizeof(T) == 2) keep.v[i] = from_f<T>(act_from_value(ACT) ? z[k][i] : act_slope<ACT>(z[k][i]));
                else keep.v[i] = from_f<T>(z[k][i]);
            }
            if constexpr (SMOOTH && kKept<T> == 2) {
                kept[2 * k] = __builtin_bit_cast(u32x4, slope[0]);
                kept[2 * k + 1] = __builtin_bit_cast(u32x4, slope[1]);
            } else {
                kept[kKept<T> * k] = __builtin_bit_cast(u32x4, keep);
                if (a.mask) kept[kKept<T> * k][0] = bits;
            }
        }
    });
}
// a chunk of a contiguous output row, as far as it lies inside
template <class T, bool VEC>
__device__ __forceinline__ void store_chunk(T *row, int q, int n_q, u32x4 v) {
    if constexpr (VEC) {
        if (q < n_q) *reinterpret_cast<u32x4 *>(row + q) = v;
    } else if (q + kChunk<T> <= n_q) {
        __builtin_memcpy(row + q, &v, 16);
    } else {
        const Frag<T> f = __builtin_bit_cast(Frag<T>, v);
#pragma unroll
        for (int i = 0; i < kChunk<T>; ++i)
            if (q + i < n_q) row[q + i] = f.v[i];
    }
}
// the epilogue of N chunks of row p (columns q[k] ..): acc in, outputs and the saved numbers out
template <class T, int MODE, bool VEC, int N>
__device__ __forceinline__ void epilogue(const DenseArgs &a, int64_t p, const int (&q)[N], int n_q, float (&z)[N][kChunk<T>], const u32x4 (&res)[N]) {
    u32x4 y[N], kept[N * kKept<T>];
    T *out = reinterpret_cast<T *>(a.out) + p * a.n_q;
    if constexpr (MODE == kForward) {
        finish_chunks<T, N>(a, z, res, y, kept);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            store_chunk<T, VEC>(out, q[k], n_q, y[k]);
            if (!a.saved_out) continue;
            if (a.mask) {
                if (q[k] < n_q) reinterpret_cast<uint8_t *>(a.saved_out)[p * a.ld_saved + q[k] / kChunk<T>] = (uint8_t)kept[kKept<T> * k][0];
            } else if (kKept<T> == 2 && a.act != NFA_ACT_RELU) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    store_chunk<float, VEC>(reinterpret_cast<float *>(a.saved_out) + p * a.n_q, q[k] + 4 * i, n_q, kept[kKept<T> * k + (kKept<T> - 1) * i]);
            } else {
                store_chunk<T, VEC>(reinterpret_cast<T *>(a.saved_out) + p * a.n_q, q[k], n_q, kept[kKept<T> * k]);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            Frag<T> o;
#pragma unroll
            for (int i = 0; i < kChunk<T>; ++i) o.v[i] = from_f<T>(z[k][i]);
            store_chunk<T, VEC>(out, q[k], n_q, __builtin_bit_cast(u32x4, o));
        }
    }
}

// Columns of a group of 32 and the two fragments that compute them.  A lane of a fragment's result holds four neighbouring of its
// sixteen columns; 16-bit types exchange columns between the two fragments so that a lane's eight are neighbours (one 16-byte store).
// column of number r of lane group g in fragment j
template <class T> __device__ __forceinline__ int column_of(int j, int g, int r) { return sizeof(T) == 2 ? g * 8 + j * 4 + r : j * 16 + g * 4 + r; }
// place (16 j + row of the fragment) of column c
template <class T> __device__ __forceinline__ int place_of_column(int c) {
    return sizeof(T) == 2 ? ((c >> 2) & 1) * 16 + (c >> 3) * 4 + (c & 3) : c;
}

// ---- the weight stays in LDS -------------------------------------------------------------------------------------------
// LDS: forward, rows of the weight in the order of place_of_column, 16 KS-byte-chunked along c; dgrad, rows along c as they are, read
// transposed.  Chunks are exchanged inside a row so that the lanes of one read lie in different banks.
// What bounds it: reading x (and the residual) and writing y, and in dgrad reading dy and what was saved and writing dx, at 4.1 and 2.9
// TB/s at 2^18 x 256 x 256 bf16; dgrad's transposed reads of the weight share LDS banks two by two.
constexpr int kResidentBytes = 144 * 1024;
template <class T, int KS>
__device__ __forceinline__ int weight_offset(int row, int chunk) {                   // forward
    constexpr int CH = KS * 4, L = CH >= 16 ? 4 : (CH == 8 ? 3 : 2);
    return (row * CH + (chunk ^ ((row >> (4 - L)) & ((1 << L) - 1)))) * 16;
}
template <class T>
__device__ __forceinline__ int weight_offset_t(int row, int chunk, int pitch) {      // dgrad; pitch: chunks in a row, 4, 8 or a multiple of 16
    if (sizeof(T) == 2) return (row * pitch + (chunk ^ (pitch >= 16 ? (row & 3) << 2 : pitch == 8 ? ((row >> 1) & 1) << 2 : 0))) * 16;
    return (row * pitch + (chunk ^ (pitch >= 16 ? ((row >> 2) & 3) << 2 : pitch == 8 ? ((row >> 2) & 1) << 2 : 0))) * 16;
}

// waves of a CU: sixteen for short rows, eight for long ones (each with twice the loads in flight): 2^18 x 64 x 64 bf16 15.1 us against
// 16.5 with eight, 2^18 x 128 x 128 fp32 98 against 104 with sixteen
constexpr int resident_waves(int ks) { return ks <= 2 ? 16 : 8; }
template <class T, int MODE, int KS, bool SPLIT, bool VEC>
__global__ __launch_bounds__(512) void resident_kernel(DenseArgs a) {
    constexpr int CE = kChunk<T>, RT = SPLIT || KS == 16 ? 1 : 2;       // rows of a wave: RT fragments of sixteen
    constexpr int NC = sizeof(T) == 2 ? 1 : 2;                          // chunks of a lane in a group of 32 columns
    // groups of 32 columns at a time: two for long rows (whole 128-byte lines in a store, twice the independent products: 130 -> 106 us at
    // 2^18 x 256 x 256 bf16), one for short ones (31 against 41 us at 100003 x 63 x 65 fp16, where the second is mostly empty)
    constexpr int NG = KS >= 4 ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = lane_id(), i = lane & 15, g = lane >> 4;
    const int q0 = blockIdx.y * a.block_q, nq = a.n_q - q0 < a.block_q ? a.n_q - q0 : a.block_q;
    const int q_rows = (nq + 31) & ~31, pitch = a.block_q / CE;         // (dgrad: block_q is 32, 64 or a multiple of 128)
    constexpr bool BOTH = kSplitBoth<T, SPLIT>;                         // the weight's second parts behind the first
    using M = Fed<T, SPLIT>;
    const int second = a.block_q * (KS * 4 * CE * (int)sizeof(T));
    const T *Q = reinterpret_cast<const T *>(a.q), *P = reinterpret_cast<const T *>(a.p);
    if (MODE == kForward) {
        for (int e = threadIdx.x; e < q_rows * KS * 4; e += blockDim.x) {
            const int q = e / (KS * 4), chunk = e % (KS * 4);
            const u32x4 v = only_inside<VEC>(load_chunk<T, VEC>(Q, q0 + q, q0 + nq, a.ld_q, chunk * CE, a.n_c), q < nq && chunk * CE < a.n_c);
            *reinterpret_cast<u32x4 *>(lds + weight_offset<T, KS>((q & ~31) + place_of_column<T>(q & 31), chunk)) = v;
        }
    } else {
        for (int e = threadIdx.x; e < KS * 4 * CE * pitch; e += blockDim.x) {
            const int n = e / pitch, chunk = e - n * pitch;
            const u32x4 v = only_inside<VEC>(load_chunk<T, VEC>(Q + q0, n, a.n_c, a.ld_q, chunk * CE, nq), n < a.n_c && chunk * CE < nq);
            char *at = lds + weight_offset_t<T>(n, chunk, pitch);
            if constexpr (BOTH) split_chunk(v, *reinterpret_cast<u32x4 *>(at), *reinterpret_cast<u32x4 *>(at + second));
            else *reinterpret_cast<u32x4 *>(at) = v;
        }
    }
    float *bias = reinterpret_cast<float *>(lds + second);
    if (MODE == kForward)
        for (int c = threadIdx.x; c < a.block_q; c += blockDim.x) bias[c] = a.bias && c < nq ? to_f(reinterpret_cast<const T *>(a.bias)[q0 + c]) : 0.0f;
    __syncthreads();

    const bool whole = a.n_c == KS * 4 * CE;
    const int64_t waves = (int64_t)gridDim.x * (blockDim.x >> 6);
    for (int64_t tile = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave_in_block(); tile < a.tiles; tile += waves) {
        const int64_t p0 = tile * (16 * RT);
        u32x4 x[RT * KS], lo[SPLIT ? RT * KS : 1];
        if (VEC && whole) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int64_t p = p0 + r * 16 + i;
                const T *row = P + (p < a.n_p ? p : a.n_p - 1) * a.ld_p + g * CE;
#pragma unroll
                for (int k = 0; k < KS; ++k) x[r * KS + k] = *reinterpret_cast<const u32x4 *>(row + k * 4 * CE);
            }
        } else {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int k = 0; k < KS; ++k)
                    x[r * KS + k] = only_inside<VEC>(load_chunk<T, VEC>(P, p0 + r * 16 + i, a.n_p, a.ld_p, (k * 4 + g) * CE, a.n_c), (k * 4 + g) * CE < a.n_c);
        }
        if constexpr (MODE == kDgrad) {
            if (a.act != NFA_ACT_NONE) {
                constexpr int NS = kSaved<T, SPLIT>;
                u32x4 s[RT * KS * NS];
                if (!SPLIT && KS >= 4 && a.mask && whole && a.ld_saved % 16 == 0 && (uintptr_t)a.saved % 16 == 0) {
                    // relu's bits, four steps of the contraction in one access: word k of a row, byte g
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const int64_t p = p0 + r * 16 + i;
                        const u32x4 *row = reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint8_t *>(a.saved) + (p < a.n_p ? p : a.n_p - 1) * a.ld_saved);
#pragma unroll
                        for (int k = 0; k < KS; k += 4) {
                            const u32x4 b = row[k / 4];
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (k + e < KS) s[r * KS + k + e] = u32x4{b[e] >> (8 * g), 0, 0, 0};
                        }
                    }
                } else
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        load_saved<T, SPLIT, VEC>(a, p0 + r * 16 + i, a.n_p, (k * 4 + g) * CE, a.n_c, &s[(r * KS + k) * NS]);
#pragma unroll
                        for (int h = 0; h < NS; ++h) s[(r * KS + k) * NS + h] = only_inside<VEC>(s[(r * KS + k) * NS + h], (k * 4 + g) * CE < a.n_c);
                    }
                form_dz<T, SPLIT, RT * KS>(a, x, s, lo, [](int, float, int) {});
            }
        }
        u32x4 ahead[MODE == kForward ? RT * NC * NG : 1];
        auto load_residual = [&](int q) {                   // of the columns q .. q + 32 NG - 1
            if constexpr (MODE == kForward) {
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int c = 0; c < NC * NG; ++c)
                        ahead[r * NC * NG + c] = load_chunk<T, VEC>(reinterpret_cast<const T *>(a.residual), p0 + r * 16 + i, a.n_p, a.ld_residual,
                                                                   q0 + q + (c / NC) * 32 + column_of<T>(c % NC, g, 0), a.n_q);
            }
        };
        if (MODE == kForward && a.residual) load_residual(0);
        for (int q = 0; q < nq; q += 32 * NG) {
            f32x4 acc[RT][2 * NG];
            u32x4 res[RT * NC * NG];
            const bool both = q + 32 < nq;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
#pragma unroll
                for (int j = 0; j < 2 * NG; ++j) acc[r][j] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < NC * NG; ++c) res[r * NC * NG + c] = MODE == kForward && a.residual ? ahead[r * NC * NG + c] : u32x4{0, 0, 0, 0};
            }
            if (MODE == kForward && a.residual && q + 32 * NG < nq) load_residual(q + 32 * NG);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if (k * 4 * CE >= a.n_c) continue;
                u32x4 w[2 * NG], w2[BOTH ? 2 * NG : 1];
#pragma unroll
                for (int j = 0; j < 2 * NG; ++j) {
                    if (j >= 2 && !both) continue;
                    const int qj = q + (j >> 1) * 32;
                    if constexpr (MODE == kForward) {
                        w[j] = *reinterpret_cast<const u32x4 *>(lds + weight_offset<T, KS>(qj + (j & 1) * 16 + i, k * 4 + g));
                    } else if constexpr (sizeof(T) == 2) {
                        s16x4 h[2], h2[2];
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const int n = k * 32 + g * 8 + s * 4 + (i >> 2), c = qj + (i & 3) * 8 + (j & 1) * 4;
                            const char *at = lds + weight_offset_t<T>(n, c >> 3, pitch) + (c & 7) * 2;
                            h[s] = read_transposed(at);
                            if constexpr (BOTH) h2[s] = read_transposed(at + second);
                        }
                        w[j] = __builtin_bit_cast(u32x4, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
                        if constexpr (BOTH) w2[j] = __builtin_bit_cast(u32x4, __builtin_shufflevector(h2[0], h2[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    } else {
                        f32x4 e;
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            const int n = k * 16 + g * 4 + s, c = qj + (j & 1) * 16 + i;
                            e[s] = *reinterpret_cast<const float *>(lds + weight_offset_t<T>(n, c >> 2, pitch) + (c & 3) * 4);
                        }
                        w[j] = __builtin_bit_cast(u32x4, e);
                    }
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int j = 0; j < 2 * NG; ++j) {
                        if (j >= 2 && !both) continue;
                        acc[r][j] = multiply<M>(w[j], x[r * KS + k], acc[r][j]);
                        if constexpr (SPLIT) acc[r][j] = multiply<M>(w[j], lo[r * KS + k], acc[r][j]);
                        if constexpr (BOTH) acc[r][j] = multiply<M>(w2[j], x[r * KS + k], acc[r][j]);
                    }
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int64_t p = p0 + r * 16 + i;
                float z[NC * NG][CE];
                int col[NC * NG];
                u32x4 add[NC * NG];
#pragma unroll
                for (int c = 0; c < NC * NG; ++c) {
                    col[c] = q0 + q + (c / NC) * 32 + column_of<T>(c % NC, g, 0);
                    add[c] = res[r * NC * NG + c];
                }
#pragma unroll
                for (int j = 0; j < 2 * NG; ++j) {
                    f32x4 b = {0, 0, 0, 0};
                    if (MODE == kForward && (j < 2 || both)) b = *reinterpret_cast<const f32x4 *>(bias + q + (j >> 1) * 32 + column_of<T>(j & 1, g, 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[NC == 1 ? j >> 1 : j][NC == 1 ? (j & 1) * 4 + e : e] = acc[r][j][e] + b[e];
                }
                if (p < a.n_p) epilogue<T, MODE, VEC, NC * NG>(a, p, col, q0 + nq, z, add);
            }
        }
    }
}

// ---- tile by tile ------------------------------------------------------------------------------------------------------
// LDS layouts.  c-contiguous tiles: 128-byte rows, the 16-byte chunks of row r exchanged by r / 2 & 7: sixteen rows of one chunk lie
// in all banks.  DEAL: so do the sixteen rows that dealt_row() names.  Transposed tiles (rows along c, 64 or 128 columns): the 32-byte (16-bit types) or 64-byte units of a row exchanged so that the rows that one instruction reads
// lie in different banks.
template <class T, int COLS>
__device__ __forceinline__ int unit_swizzle(int row) {
    if (sizeof(T) == 4) return (row >> 2) & 3;
    if (COLS >= 128) return (row & 3) | (((row >> 3) & 1) << 2);
    return ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
}
// forward, 16-bit types: the columns (rows of the weight's tile) of a pair of fragments are dealt out so that a lane's results of both
// are eight neighbours, one 16-byte store of the result straight from its registers
template <class T> __device__ __forceinline__ int dealt_row(int c0, int i) { return (c0 & ~31) + column_of<T>((c0 >> 4) & 1, i >> 2, i & 3); }
template <class T, bool TR, int ROWS, bool DEAL = false>
__device__ __forceinline__ int stage_offset(int row, int chunk) {        // byte offset of a chunk in its tile
    if (DEAL) return row * kRowBytes + ((chunk ^ (((row >> 1) & 1) | ((row >> 2) & 6))) << 4);
    if (!TR) return row * kRowBytes + ((chunk ^ ((row >> 1) & 7)) << 4);
    if (sizeof(T) == 4) return row * ROWS * 4 + (((chunk >> 2) ^ unit_swizzle<T, ROWS>(row)) << 6) + ((chunk & 3) << 4);
    return row * ROWS * 2 + (((chunk >> 1) ^ unit_swizzle<T, ROWS>(row)) << 5) + ((chunk & 1) << 4);
}

// the sixteen bytes that lane l feeds to the matrix units for rows (or columns) c0 .. c0 + 15 and half `ks` of the tile
template <class T, bool TR, int ROWS, bool DEAL = false>
__device__ __forceinline__ u32x4 read_frag(const char *tile, int c0, int ks, int lane) {
    const int i = lane & 15, g = lane >> 4;
    u32x4 v;
    if (DEAL) {
        v = *reinterpret_cast<const u32x4 *>(tile + stage_offset<T, false, ROWS, true>(dealt_row<T>(c0, i), ks * 4 + g));
    } else if (!TR) {
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
        s16x4 h[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int row = ks * 32 + g * 8 + s * 4 + (i >> 2);
            h[s] = read_transposed(tile + row * ROWS * 2 + (((c0 >> 4) ^ unit_swizzle<T, ROWS>(row)) << 5) + ((i & 3) << 3));
        }
        v = __builtin_bit_cast(u32x4, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return v;
}

// WP x WQ waves, each with BP / WP x BQ / WQ of the tile.  A step is 128 bytes of the contraction: staged from registers into LDS one or
// two steps ahead, one barrier each.  65536 x 1024 x 1024 bf16 takes 186 us (740 TF): a workgroup fills its CU, so that its first loads and
// its epilogue (the whole chip's 34 MB of y at once) are not hidden behind another one's products; without it that takes 125 to 135 us.
template <class T, int MODE, int BP, int BQ, int WP, int WQ, bool SPLIT, bool VEC, bool DEEP>
__global__ __launch_bounds__(WP * WQ * kWave, 2) void tile_kernel(DenseArgs a) {
    constexpr int TH = WP * WQ * kWave;
    constexpr bool PT = MODE == kWgrad, QT = MODE != kForward, FUSE = MODE != kForward, DEAL = MODE == kForward && sizeof(T) == 2;
    constexpr int CE = kChunk<T>, ST = kStage<T>;
    constexpr int CP = BP * 8 / TH, CQ = BQ * 8 / TH;       // chunks a thread stages per tile
    constexpr int NP = BP / WP / 16, NQ = BQ / WQ / 16;     // sixteen-wide fragments of a wave
    constexpr bool BOTH = kSplitBoth<T, SPLIT>;
    constexpr int kP = BP * kRowBytes, kQ = BQ * kRowBytes, kAtQ = kP * (SPLIT ? 2 : 1), kBuf = kAtQ + kQ * (BOTH ? 2 : 1);
    using M = Fed<T, SPLIT>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = lane_id(), wave = wave_in_block();
    const int wp = wave / WQ, wq = wave % WQ;

    // tile (and, for wgrad, stretch of rows) of this workgroup: eight runs of them, one per XCD (workgroups are dealt to the XCDs in
    // turn), so that the tiles that read the same rows share an L2
    const int per = (int)((gridDim.x + kNumXCD - 1) / kNumXCD);
    const int64_t at = (int64_t)(blockIdx.x % kNumXCD) * per + blockIdx.x / kNumXCD;
    if (at >= (int64_t)a.tiles * a.splits) return;
    const int64_t stretch = at / a.tiles;
    const int tile = (int)(at - stretch * a.tiles);
    const int64_t p0 = (int64_t)(tile / a.tiles_q) * BP;
    const int q0 = (tile % a.tiles_q) * BQ;
    const int64_t c_begin = MODE == kWgrad ? stretch * a.split : 0;
    const int64_t c_end = MODE == kWgrad ? (c_begin + a.split < a.n_c ? c_begin + a.split : a.n_c) : a.n_c;

    const T *P = reinterpret_cast<const T *>(a.p), *Q = reinterpret_cast<const T *>(a.q);
    constexpr int NS = kSaved<T, SPLIT>;
    struct Staged { u32x4 p[CP], s[FUSE ? CP * NS : 1], q[CQ]; };
    f32x4 acc[NP][NQ];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    float db[MODE == kWgrad ? CE : 1];
#pragma unroll
    for (int i = 0; i < (MODE == kWgrad ? CE : 1); ++i) db[i] = 0.0f;

    // which row and chunk of a tile this thread stages in its k-th turn
    auto place = [&](bool tr, int rows, int k, int &row, int &chunk) {
        const int per_row = tr ? rows / CE : 8;
        chunk = tid % per_row;
        row = tid / per_row + k * (TH / per_row);
    };
    auto load = [&](Staged &t, int64_t c) {
#pragma unroll
        for (int k = 0; k < CP; ++k) {
            int row, chunk;
            place(PT, BP, k, row, chunk);
            const int64_t r = PT ? c + row : p0 + row, col = PT ? p0 + chunk * CE : c + chunk * CE;
            const int64_t rows = PT ? c_end : a.n_p, cols = PT ? a.n_p : a.n_c;
            t.p[k] = load_chunk<T, VEC>(P, r, rows, a.ld_p, col, cols);
            if constexpr (FUSE) load_saved<T, SPLIT, VEC>(a, r, rows, col, cols, &t.s[k * NS]);
        }
#pragma unroll
        for (int k = 0; k < CQ; ++k) {
            int row, chunk;
            place(QT, BQ, k, row, chunk);
            const int64_t r = QT ? c + row : q0 + row, col = QT ? q0 + chunk * CE : c + chunk * CE;
            const int64_t rows = QT ? c_end : a.n_q, cols = QT ? a.n_q : a.n_c;
            t.q[k] = load_chunk<T, VEC>(Q, r, rows, a.ld_q, col, cols);
        }
    };
    auto store = [&](Staged &t, char *buf, int64_t c) {
        u32x4 lo[SPLIT ? CP : 1];
#pragma unroll
        for (int k = 0; k < CP; ++k) {
            int row, chunk;
            place(PT, BP, k, row, chunk);
            const bool inside = PT ? c + row < c_end && p0 + chunk * CE < a.n_p : p0 + row < a.n_p && c + chunk * CE < a.n_c;
            t.p[k] = only_inside<VEC>(t.p[k], inside);
            if constexpr (FUSE)
#pragma unroll
                for (int h = 0; h < NS; ++h) t.s[k * NS + h] = only_inside<VEC>(t.s[k * NS + h], inside);
        }
        if constexpr (FUSE)
            form_dz<T, SPLIT, CP>(a, t.p, t.s, lo, [&](int, float dz, int e) {
                if constexpr (MODE == kWgrad) db[e] += dz;
            });
#pragma unroll
        for (int k = 0; k < CP; ++k) {
            int row, chunk;
            place(PT, BP, k, row, chunk);
            *reinterpret_cast<u32x4 *>(buf + stage_offset<T, PT, BP>(row, chunk)) = t.p[k];
            if constexpr (SPLIT) *reinterpret_cast<u32x4 *>(buf + kP + stage_offset<T, PT, BP>(row, chunk)) = lo[k];
        }
#pragma unroll
        for (int k = 0; k < CQ; ++k) {
            int row, chunk;
            place(QT, BQ, k, row, chunk);
            const bool inside = QT ? c + row < c_end && q0 + chunk * CE < a.n_q : q0 + row < a.n_q && c + chunk * CE < a.n_c;
            char *at = buf + kAtQ + stage_offset<T, QT, BQ, DEAL>(row, chunk);
            const u32x4 v = only_inside<VEC>(t.q[k], inside);
            if constexpr (BOTH) split_chunk(v, *reinterpret_cast<u32x4 *>(at), *reinterpret_cast<u32x4 *>(at + kQ));
            else *reinterpret_cast<u32x4 *>(at) = v;
        }
    };
    auto compute = [&](const char *buf, int64_t c) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            if (c + ks * (ST / 2) >= c_end) break;          // a half that holds only zeros
            u32x4 fp[NP], fq[NQ], fq2[BOTH ? NQ : 1];
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                fq[j] = read_frag<T, QT, BQ, DEAL>(buf + kAtQ, wq * (BQ / WQ) + j * 16, ks, lane);
                if constexpr (BOTH) fq2[j] = read_frag<T, QT, BQ>(buf + kAtQ + kQ, wq * (BQ / WQ) + j * 16, ks, lane);
            }
#pragma unroll
            for (int half = 0; half < (SPLIT ? 2 : 1); ++half) {
#pragma unroll
                for (int i = 0; i < NP; ++i) fp[i] = read_frag<T, PT, BP>(buf + half * kP, wp * (BP / WP) + i * 16, ks, lane);
#pragma unroll
                for (int i = 0; i < NP; ++i)
#pragma unroll
                    for (int j = 0; j < NQ; ++j) {
                        acc[i][j] = multiply<M>(fq[j], fp[i], acc[i][j]);
                        if constexpr (BOTH)
                            if (half == 0) acc[i][j] = multiply<M>(fq2[j], fp[i], acc[i][j]);
                    }
            }
        }
    };

    if constexpr (DEEP) {
        // Two tiles in flight behind the one that is multiplied.  Every load is made, also behind the end (from a place that exists; what
        // lies outside is stored as zeros): with a branch around it the wait for one tile would be a wait for both.
        static_assert(VEC, "loads behind the end need places that exist");
        Staged even, odd;
        load(even, c_begin);
        load(odd, c_begin + ST);
        store(even, lds, c_begin);
        __syncthreads();
        auto step = [&](Staged &next, Staged &after, int64_t c, int cur) {       // tile c is in buffer `cur`, tile c + ST in `next`
            load(after, c + 2 * ST);
            compute(lds + cur * kBuf, c);
            store(next, lds + (cur ^ 1) * kBuf, c + ST);
            __syncthreads();
        };
        for (int64_t c = c_begin; c < c_end; c += 2 * ST) {
            step(odd, even, c, 0);
            step(even, odd, c + ST, 1);
        }
    } else {
        Staged t;
        load(t, c_begin);
        store(t, lds, c_begin);
        __syncthreads();
        int cur = 0;
        for (int64_t c = c_begin; c < c_end; c += ST) {
            const bool more = c + ST < c_end;
            if (more) load(t, c + ST);
            compute(lds + cur * kBuf, c);
            if (more) store(t, lds + (cur ^ 1) * kBuf, c + ST);
            __syncthreads();
            cur ^= 1;
        }
    }

    // lane l holds row p = l % 16 of each fragment and four neighbouring columns q
    const int i = lane & 15, g = lane >> 4;
    if constexpr (MODE == kWgrad) {
        float *part = a.partial + stretch * (a.n_p * a.n_q + a.n_p);
#pragma unroll
        for (int pi = 0; pi < NP; ++pi)
#pragma unroll
            for (int qi = 0; qi < NQ; ++qi) {
                const int64_t p = p0 + wp * (BP / WP) + pi * 16 + i;
                const int q = q0 + wq * (BQ / WQ) + qi * 16 + g * 4;
                if (p >= a.n_p) continue;
                if (VEC) {                                  // (whole chunks of 16 bytes: n_p and n_q divide by 4)
                    if (q < a.n_q) *reinterpret_cast<f32x4 *>(part + p * a.n_q + q) = acc[pi][qi];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (q + r < a.n_q) part[p * a.n_q + q + r] = acc[pi][qi][r];
                }
            }
        if (q0 == 0 && a.want_bias) {                       // db: the threads that staged the same columns, in order
            constexpr int per_row = BP / CE, n = TH / per_row;
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
    } else if constexpr (DEAL) {
        // straight from the registers, sixteen rows of each wave at a time (65536 x 1024 x 1024 bf16, back to back: 164 us, through LDS
        // as below 175; 65536 x 512 x 512 48 and 55)
        constexpr int N = NQ / 2;                           // chunks of a lane in a row
        const T *bias = reinterpret_cast<const T *>(a.bias);
        int col[N];
        float add[N][CE];
        u32x4 res[N] = {};
#pragma unroll
        for (int c = 0; c < N; ++c) {
            col[c] = q0 + wq * (BQ / WQ) + c * 32 + g * CE;
#pragma unroll
            for (int e = 0; e < CE; ++e) add[c][e] = bias && col[c] + e < a.n_q ? to_f(bias[col[c] + e]) : 0.0f;
        }
#pragma unroll 1
        for (int pi = 0; pi < NP; ++pi) {                   // (one body for all fragments: unrolled it would not fit the instruction cache)
            const int64_t p = p0 + wp * (BP / WP) + pi * 16 + i;
            float z[N][CE];
            if (a.residual)
#pragma unroll
                for (int c = 0; c < N; ++c) res[c] = load_chunk<T, VEC>(reinterpret_cast<const T *>(a.residual), p, a.n_p, a.ld_residual, col[c], a.n_q);
#pragma unroll
            for (int t = 0; t < NP; ++t) {
                if (t != pi) continue;
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z[j >> 1][(j & 1) * 4 + r] = acc[t][j][r] + add[j >> 1][(j & 1) * 4 + r];
            }
            if (p < a.n_p) epilogue<T, MODE, VEC, N>(a, p, col, a.n_q, z, res);
        }
    } else {
        // through LDS, so that a thread holds whole chunks of a row: sixteen rows of each wave at a time
        const T *bias = reinterpret_cast<const T *>(a.bias);
        constexpr int W = BQ / WQ + 4;                      // floats in a row: the wave's columns, shifted by a bank group per row
        float *mine = reinterpret_cast<float *>(lds) + wave * 16 * W;
#pragma unroll 1
        for (int pi = 0; pi < NP; ++pi) {                   // (one body for all fragments: unrolled it would not fit the instruction cache)
#pragma unroll
            for (int t = 0; t < NP; ++t) {
                if (t != pi) continue;
#pragma unroll
                for (int qi = 0; qi < NQ; ++qi) *reinterpret_cast<f32x4 *>(mine + i * W + qi * 16 + g * 4) = acc[t][qi];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            constexpr int per_row = BQ / WQ / CE;           // chunks of a row
#pragma unroll
            for (int k = 0; k < 16 * per_row / kWave; ++k) {
                const int e = k * kWave + lane, row = e / per_row, chunk = e % per_row;
                const int64_t p = p0 + wp * (BP / WP) + pi * 16 + row;
                const int col[1] = {q0 + wq * (BQ / WQ) + chunk * CE};
                float z[1][CE];
                u32x4 res[1] = {{0, 0, 0, 0}};
                if (MODE == kForward && a.residual)
                    res[0] = load_chunk<T, VEC>(reinterpret_cast<const T *>(a.residual), p, a.n_p, a.ld_residual, col[0], a.n_q);
#pragma unroll
                for (int v = 0; v < CE; ++v)
                    z[0][v] = mine[row * W + chunk * CE + v] + (MODE == kForward && bias && col[0] + v < a.n_q ? to_f(bias[col[0] + v]) : 0.0f);
                if (p < a.n_p && col[0] < a.n_q) epilogue<T, MODE, VEC, 1>(a, p, col, a.n_q, z, res);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---- few rows, a long contraction ----------------------------------------------------------------------------------------
// A tile of a long contraction is one step after the other, and few tiles leave the chip empty meanwhile: here sixteen rows and 32
// columns are a workgroup, whose four waves take every fourth step each, straight from memory, and join their sums in LDS in order.
// Latency bounds it: 200 x 1024 x 1024 bf16 7.9 us, fp32 13.3; 1 x 256 x 256 4.4 us, most of it the launch.
template <class T, bool VEC>
__global__ __launch_bounds__(kBlock) void stream_kernel(DenseArgs a) {
    constexpr int CE = kChunk<T>, NC = sizeof(T) == 2 ? 1 : 2, kDeep = 4;      // kDeep: a wave's steps in flight
    __shared__ f32x4 sums[kWavesPerBlock][2][kWave];
    const int lane = lane_id(), i = lane & 15, g = lane >> 4, wave = wave_in_block();
    const int64_t p0 = (int64_t)(blockIdx.x / a.tiles_q) * 16;
    const int q0 = (int)(blockIdx.x % a.tiles_q) * 32;
    const T *P = reinterpret_cast<const T *>(a.p), *Q = reinterpret_cast<const T *>(a.q);
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const int64_t steps = (a.n_c + 4 * CE - 1) / (4 * CE);
    for (int64_t k0 = wave; k0 < steps; k0 += kWavesPerBlock * kDeep) {
        u32x4 x[kDeep], w[kDeep][2];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const int64_t c = ((k0 + d * kWavesPerBlock) * 4 + g) * CE;
            x[d] = load_chunk<T, VEC>(P, p0 + i, a.n_p, a.ld_p, c, a.n_c);
#pragma unroll
            for (int j = 0; j < 2; ++j) w[d][j] = load_chunk<T, VEC>(Q, q0 + column_of<T>(j, i >> 2, i & 3), a.n_q, a.ld_q, c, a.n_c);
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const bool inside = ((k0 + d * kWavesPerBlock) * 4 + g) * CE < a.n_c;
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[j] = multiply<T>(only_inside<VEC>(w[d][j], inside), only_inside<VEC>(x[d], inside), acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    const int64_t p = p0 + i;
    if (wave != 0 || p >= a.n_p) return;
    float z[NC][CE];
    int col[NC];
    u32x4 res[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        col[c] = q0 + column_of<T>(c, g, 0);
        res[c] = u32x4{0, 0, 0, 0};
        if (a.residual) res[c] = load_chunk<T, VEC>(reinterpret_cast<const T *>(a.residual), p, a.n_p, a.ld_residual, col[c], a.n_q);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = q0 + column_of<T>(j, g, e);
            float v = a.bias && c < a.n_q ? to_f(reinterpret_cast<const T *>(a.bias)[c]) : 0.0f, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kWavesPerBlock; ++k) sum += sums[k][j][lane][e];
            z[NC == 1 ? 0 : j][NC == 1 ? j * 4 + e : e] = sum + v;
        }
    epilogue<T, kForward, VEC, NC>(a, p, col, a.n_q, z, res);
}

// ---- the weight gradient of a narrow layer in 32 bits ------------------------------------------------------------------------
// dW[n][k] = sum_m dz[m][n] x[m][k] with n and k of up to 64.  One matrix instruction takes four rows, a lane a column of one of them: so
// a lane loads NP (NQ) neighbouring columns of its row straight from memory, fragment f takes the f-th of them (its columns are f, NP + f,
// 2 NP + f, ...), nothing goes through LDS, and columns are padded to 16 and not to the 64 of a tile.  Reading dy and x once bounds it:
// 2^18 x 8 x 32 takes 14.4 us with its join, 42 MB at 2.9 TB/s (33 us by tiles).
// The four waves of a workgroup take every fourth sixteen rows each and join their sums in LDS in order.
template <int NP, int NQ>
__global__ __launch_bounds__(kBlock, 2) void narrow_wgrad_kernel(DenseArgs a) {
    constexpr int kSteps = 4;                               // four rows each, loaded together
    struct alignas(NP * 4) PVec { float v[NP]; };
    struct alignas(NQ * 4) QVec { float v[NQ]; };
    struct Rows { PVec p[kSteps], s[kSteps]; uint32_t bits[kSteps]; QVec q[kSteps]; };
    __shared__ f32x4 sums[kWavesPerBlock][NP * NQ][kWave];
    const int lane = lane_id(), i = lane & 15, g = lane >> 4, wave = wave_in_block();
    const int64_t stretch = blockIdx.x, begin = stretch * a.split, end = begin + a.split < a.n_c ? begin + a.split : a.n_c;
    const int p = i * NP < a.n_p ? i * NP : 0, q = i * NQ < a.n_q ? i * NQ : 0;      // (columns that do not exist are read from one that does)
    const bool value = a.act != NFA_ACT_NONE && !a.mask;
    f32x4 acc[NP][NQ];
    float db[NP];
#pragma unroll
    for (int f = 0; f < NP; ++f) {
        db[f] = 0.0f;
#pragma unroll
        for (int e = 0; e < NQ; ++e) acc[f][e] = f32x4{0, 0, 0, 0};
    }
    auto load = [&](Rows &r, int64_t row0) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int64_t want = row0 + k * 4 + g, row = want < end ? want : end - 1;
            r.p[k] = *reinterpret_cast<const PVec *>(reinterpret_cast<const float *>(a.p) + row * a.ld_p + p);
            r.q[k] = *reinterpret_cast<const QVec *>(reinterpret_cast<const float *>(a.q) + row * a.ld_q + q);
            if (a.mask) r.bits[k] = reinterpret_cast<const uint8_t *>(a.saved)[row * a.ld_saved + (p >> 2)];
            if (value) r.s[k] = *reinterpret_cast<const PVec *>(reinterpret_cast<const float *>(a.saved) + row * a.ld_saved + p);
        }
    };
    auto add = [&](Rows &r, int64_t row0) {
        with_act(a.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int f = 0; f < NP; ++f) {
                    float &dz = r.p[k].v[f];
                    if constexpr (ACT == NFA_ACT_RELU) dz = (a.mask ? ((r.bits[k] >> ((p & 3) + f)) & 1u) == 0 : r.s[k].v[f] <= 0.0f) ? 0.0f : dz;
                    else if constexpr (ACT != NFA_ACT_NONE) dz *= act_slope_of_kept<ACT>(r.s[k].v[f]);
                }
        });
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const bool inside = row0 + k * 4 + g < end;
#pragma unroll
            for (int f = 0; f < NP; ++f) db[f] += r.p[k].v[f] = inside ? r.p[k].v[f] : 0.0f;
#pragma unroll
            for (int e = 0; e < NQ; ++e) {
                const float x = inside ? r.q[k].v[e] : 0.0f;
#pragma unroll
                for (int f = 0; f < NP; ++f) acc[f][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, r.p[k].v[f], acc[f][e], 0, 0, 0);
            }
        }
    };
    constexpr int kEach = kSteps * 4, kStride = kEach * kWavesPerBlock;
    Rows now, next;
    int64_t row = begin + wave * kEach;
    load(now, row);
    for (; row < end; row += kStride) {
        load(next, row + kStride);
        add(now, row);
        now = next;
    }
#pragma unroll
    for (int f = 0; f < NP; ++f)
#pragma unroll
        for (int e = 0; e < NQ; ++e) sums[wave][f * NQ + e][lane] = acc[f][e];
    __syncthreads();
    float *part = a.partial + stretch * (a.n_p * a.n_q + a.n_p);
    for (int t = wave; t < NP * NQ; t += kWavesPerBlock) {
        f32x4 v = sums[0][t][lane];
#pragma unroll
        for (int w = 1; w < kWavesPerBlock; ++w) v += sums[w][t][lane];
        const int col = i * NP + t / NQ;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = (g * 4 + r) * NQ + t % NQ;
            if (col < a.n_p && at < a.n_q) part[(int64_t)col * a.n_q + at] = v[r];
        }
    }
    if (!a.want_bias) return;
    __syncthreads();
    float *join = reinterpret_cast<float *>(sums);          // [wave][fragment][lane]
#pragma unroll
    for (int f = 0; f < NP; ++f) join[(wave * NP + f) * kWave + lane] = db[f];
    __syncthreads();
    const int c = threadIdx.x;
    if (c < a.n_p) {
        float v = 0.0f;
        for (int w = 0; w < kWavesPerBlock; ++w)
#pragma unroll
            for (int r = 0; r < 4; ++r) v += join[(w * NP + c % NP) * kWave + r * 16 + c / NP];
        part[a.n_p * a.n_q + c] = v;
    }
}

// Columns by lane, sixteen rows side by side; a column's sum is formed in the same order every time.  A workgroup sums the rows
// [first, first + each) of its 64 columns, first = blockIdx.y * each; of many rows a first launch leaves each stretch's sum in the
// stretch's own first row (nobody else reads it), a second one sums those.  The columns go to up to three outputs, one behind the other
// (nullptr: not wanted).  Latency bounds it: 256 rows of 65792 columns (67 MB) take 7.5 us, 512 rows of 288 4 us.
struct Outputs { void *to[3]; int64_t cols[3]; };
template <class T, bool LAST>
__global__ __launch_bounds__(1024) void reduce_rows_kernel(float *part, int64_t rows, int64_t each, int64_t step, int64_t ld, Outputs o) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane, first = blockIdx.y * each, end = first + each < rows ? first + each : rows;
    float v = 0.0f;
    if (c < ld) {
#pragma unroll 8
        for (int64_t r = first + grp * step; r < end; r += 16 * step) v += part[r * ld + c];
    }
    sum[grp][lane] = v;
    __syncthreads();
    if (grp == 0 && c < ld) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += sum[k][lane];
        if (!LAST) {
            part[first * ld + c] = t;
            return;
        }
        int64_t at = c;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (at >= 0 && at < o.cols[k] && o.to[k]) reinterpret_cast<T *>(o.to[k])[at] = from_f<T>(t);
            at -= o.cols[k];
        }
    }
}

// the same for few rows of many columns: a thread a column, its rows in order
template <class T>
__global__ __launch_bounds__(kBlock) void reduce_few_rows_kernel(const float *__restrict__ part, int64_t rows, int64_t ld, Outputs o) {
    const int64_t c = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (c >= ld) return;
    float v = 0.0f;
#pragma unroll 8
    for (int64_t r = 0; r < rows; ++r) v += part[r * ld + c];
    int64_t at = c;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (at >= 0 && at < o.cols[k] && o.to[k]) reinterpret_cast<T *>(o.to[k])[at] = from_f<T>(v);
        at -= o.cols[k];
    }
}

bool aligned(const void *p, int64_t ld, int64_t cols, int64_t bytes, int64_t to) {
    return (uintptr_t)p % to == 0 && ld * bytes % to == 0 && cols * bytes % to == 0;
}

template <class K>
int allow_lds(K kernel, size_t bytes) {
    if (bytes <= 64 * 1024) return NFA_OK;
    const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == hipSuccess ? NFA_OK : fail(NFA_ERR_LAUNCH, "linear: %zu bytes of LDS: %s", bytes, hipGetErrorString(e));
}

template <class T, int MODE, int BP, int BQ, int WP, int WQ, bool SPLIT>
int launch_tiles(DenseArgs a, int64_t splits, hipStream_t s) {
    const int64_t tiles_p = ceil_div(a.n_p, BP);
    a.tiles_q = (int32_t)ceil_div(a.n_q, BQ);
    NFA_REQUIRE(tiles_p * a.tiles_q * std::max<int64_t>(splits, 1) < kMaxThreads / (WP * WQ * kWave), "linear: too many rows for one launch");
    a.tiles = (int32_t)(tiles_p * a.tiles_q);
    const int64_t steps = MODE == kWgrad ? a.split : a.n_c;
    const size_t bytes = (size_t)(BP * (SPLIT ? 2 : 1) + BQ * (kSplitBoth<T, SPLIT> ? 2 : 1)) * kRowBytes * (steps > kStage<T> ? 2 : 1);
    auto kernel = tile_kernel<T, MODE, BP, BQ, WP, WQ, SPLIT, true, false>;
    if constexpr (BP < 256)                                 // (the largest tiles are for aligned rows)
        if (!a.vec) kernel = tile_kernel<T, MODE, BP, BQ, WP, WQ, SPLIT, false, false>;
    // two tiles ahead where one workgroup is all a CU holds and the contraction is long enough: weight gradient of 2^18 x 256 x 256 104 -> 90
    // us, 65536 x 1024 x 1024 forward 226 -> 219 then (dgrad has no registers left for it)
    if constexpr (BP * BQ >= 128 * 256 && sizeof(T) == 2 && MODE != kDgrad)
        if (a.vec && steps >= 8 * kStage<T>) kernel = tile_kernel<T, MODE, BP, BQ, WP, WQ, SPLIT, true, true>;
    if (int rc = allow_lds(kernel, bytes)) return rc;
    a.splits = (int32_t)splits;
    const unsigned grid = (unsigned)(ceil_div(a.tiles * splits, kNumXCD) * kNumXCD);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(WP * WQ * kWave), bytes, s, a);
    return check_launch("tile_kernel");
}

template <class T, int MODE, int KS, bool SPLIT>
int launch_resident(DenseArgs a, hipStream_t s) {
    constexpr int RT = SPLIT || KS == 16 ? 1 : 2, C = KS * 4 * kChunk<T>, kWeight = C * (int)sizeof(T) * (kSplitBoth<T, SPLIT> ? 2 : 1);
    const int64_t tiles = ceil_div(a.n_p, 16 * RT);
    NFA_REQUIRE(tiles < (1ll << 31), "linear: too many rows for one launch");
    a.tiles = (int32_t)tiles;
    // columns of a workgroup: all that fit, fewer where the rows alone do not give every SIMD a wave (4096 x 256 x 256 bf16 7.5 us, 17.6
    // with all columns)
    auto round_q = [](int64_t q) { return q <= 32 ? 32 : q <= 64 ? 64 : ceil_div(q, 128) * 128; };
    int64_t block = round_q(a.n_q), most = 32;
    while (round_q(most + 32) * kWeight <= kResidentBytes && most < block) most = round_q(most + 32);
    if (block > most) block = most;
    while (block > 32 && tiles * ceil_div(a.n_q, block) < kNumCU * 4) block = block > 128 ? round_q(block / 2) : block / 2;
    a.block_q = (int32_t)block;
    const int64_t blocks_q = ceil_div(a.n_q, block);
    const size_t bytes = (size_t)(block * (kWeight + 4));                      // and the bias in 32 bits
    const auto kernel = a.vec ? resident_kernel<T, MODE, KS, SPLIT, true> : resident_kernel<T, MODE, KS, SPLIT, false>;
    if (int rc = allow_lds(kernel, bytes)) return rc;
    const int per_cu = bytes <= 36 * 1024 ? 4 : bytes <= 72 * 1024 ? 2 : 1, threads = std::min(512, resident_waves(KS) * kWave / per_cu);
    int64_t grid = ceil_div((int64_t)kNumCU * per_cu, blocks_q);
    const int64_t need = ceil_div(tiles, threads / kWave);
    if (grid > need) grid = need;
    NFA_REQUIRE(blocks_q < 65536, "linear: too many features for one launch");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid, (unsigned)blocks_q), dim3(threads), bytes, s, a);
    return check_launch("resident_kernel");
}

template <class T>
int launch_stream(DenseArgs a, hipStream_t s) {
    a.tiles_q = (int32_t)ceil_div(a.n_q, 32);
    NFA_REQUIRE(ceil_div(a.n_p, 16) * a.tiles_q < kMaxThreads / kBlock, "linear: too many rows for one launch");
    const auto kernel = a.vec ? stream_kernel<T, true> : stream_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(ceil_div(a.n_p, 16) * a.tiles_q)), dim3(kBlock), 0, s, a);
    return check_launch("stream_kernel");
}

// forward or dgrad: the weight in LDS for contractions of up to 256, tiles beyond
template <class T, int MODE, bool SPLIT>
int launch_rows(const DenseArgs &a, hipStream_t s) {
    constexpr int step = 4 * kChunk<T>;
    // few rows: neither a weight for every CU nor a tile, but rows, columns and the contraction over many workgroups.  In bf16 while every
    // CU gets one (1000 x 128 x 128: 4.5 us against 4.7 with the weight in LDS, 1000 x 256 x 256, 504 workgroups, 5.6 against 6.5, but
    // 1500 x 128 x 128, 376 of them, 5.4 against 4.7), in fp32, whose weight takes twice as long to LDS, four (1000 x 256 x 256 5.9
    // against 10.0, 400 x 128 x 1024, 800 workgroups, 8.6 against 9.0, 1000 x 128 x 1024, 2016, 14.4 against 12.9)
    if (MODE == kForward && ceil_div(a.n_p, 16) * ceil_div(a.n_q, 32) <= (sizeof(T) == 4 ? 4 : 1) * kNumCU) return launch_stream<T>(a, s);
    // the weight in LDS; 2^18 x 256 x 256 bf16 forward 66 us against 88 by tiles, dgrad 62 against 81; fp32 316 against 339
    if (a.n_c <= step) return launch_resident<T, MODE, 1, SPLIT>(a, s);
    if (a.n_c <= 2 * step) return launch_resident<T, MODE, 2, SPLIT>(a, s);
    if (a.n_c <= 4 * step) return launch_resident<T, MODE, 4, SPLIT>(a, s);
    if (a.n_c <= 8 * step) return launch_resident<T, MODE, 8, SPLIT>(a, s);
    // (dgrad in fp32 reads a number of a column at a time from LDS, here for every sixteen rows, by tiles for 64: 2^18 x 256 x 256 608 us
    // against 439 by tiles, 2^18 x 64 x 256 220 against 144, 4096 x 256 x 256 35 against 12)
    if constexpr (sizeof(T) == 4 && MODE == kForward)
        if (a.n_c <= 16 * step) return launch_resident<T, MODE, 16, SPLIT>(a, s);
    // long contractions.  Few tiles: 4096 x 1024 x 256, 64 of them: fp32 49 us against 84 by tiles (whose steps are four times as long as
    // those of 16-bit types), bf16 25 against 20.  In fp32 any number of rows too, where the 32 columns of one workgroup are all there
    // are: 75956 x 751 x 4 61 us against 98, 75956 x 752 x 32 63 against 89; in bf16 41 against 26 and 36 against 25
    if (MODE == kForward && ((sizeof(T) == 4 && a.n_q <= 32 && a.n_p < (1ll << 27)) ||
                             ceil_div(a.n_p, 128) * ceil_div(a.n_q, 128) < (sizeof(T) == 4 ? kNumCU : kNumCU / 4))) return launch_stream<T>(a, s);
    // 16-bit types, aligned and large enough for every CU: 256 x 256 by eight waves, whose fragments are used often enough that the matrix
    // units and not LDS set the pace (16384 x 1024 x 1024 bf16 43.9 us against 51.8 by 128 x 128, 65536 x 512 x 512 56.5 against 62.7)
    constexpr int BP = SPLIT ? 64 : 128;
    if constexpr (sizeof(T) == 2 && !SPLIT)
        if (a.vec && a.n_q > 128 && ceil_div(a.n_p, 256) * ceil_div(a.n_q, 256) >= kNumCU) return launch_tiles<T, MODE, 256, 256, 2, 4, SPLIT>(a, 1, s);
    // dgrad of few rows: smaller tiles, so that more CUs get one (2000 x 512 x 512 fp32 22 us against 50 by 128 x 128, bf16 8.8 against 15;
    // 588 x 908 x 804 34 against 79, 18 against 35)
    if constexpr (MODE == kDgrad && !SPLIT)
        if (ceil_div(a.n_p, BP) * ceil_div(a.n_q, 128) < kNumCU) return launch_tiles<T, MODE, 64, 64, 2, 2, SPLIT>(a, 1, s);
    // both sides in two parts fill 96 KiB of LDS with 64 x 128, one wave per SIMD: eight waves by 128 x 128 (65536 x 1024 x 1024 fp16 671 us
    // against 1091, 65536 x 512 x 512 176 against 286)
    if constexpr (kSplitBoth<T, SPLIT>)
        if (a.n_q > 64) return launch_tiles<T, MODE, 128, 128, 2, 4, SPLIT>(a, 1, s);
    // (64 columns where there are no more: 65536 x 512 x 64 fp32 45 us against 79)
    return a.n_q <= 64 ? launch_tiles<T, MODE, BP, 64, 2, 2, SPLIT>(a, 1, s) : launch_tiles<T, MODE, BP, 128, 2, 2, SPLIT>(a, 1, s);
}

template <int NP>
int launch_narrow_wgrad(DenseArgs a, int64_t splits, hipStream_t s) {
    const auto kernel = a.n_q <= 16 ? narrow_wgrad_kernel<NP, 1> : a.n_q <= 32 ? narrow_wgrad_kernel<NP, 2> : narrow_wgrad_kernel<NP, 4>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)splits), dim3(kBlock), 0, s, a);
    return check_launch("narrow_wgrad_kernel");
}

// rows of the long axis that one workgroup of the weight gradient sums: enough workgroups for every CU twice, and not so many that
// their partial sums (a whole weight each) outweigh the rows read
struct WgradPlan { int64_t split, splits, bp, bq; };
bool narrow_layer(int64_t n, int64_t k) { return n <= 64 && k <= 64 && n % 4 == 0 && k % 4 == 0; }
WgradPlan wgrad_plan(int64_t rows, int64_t n, int64_t k, int32_t dtype, bool two_parts) {
    const int64_t stage = dtype == NFA_DTYPE_F32 ? 32 : 64;
    WgradPlan w;
    // large tiles read dy and x fewer times (2^18 x 256 x 256 bf16 by 64 x 64, 128 x 128, 128 x 256: 173, 130, 91 us; fp32 418, 402, 368),
    // but in fp32, which the matrix units bound, not at the price of padding (2^18 x 129 x 32: 92 us by 64 x 64, 117 by 64 x 128),
    auto pad = [](int64_t x, int64_t b) { return ceil_div(x, b) * b; };
    const bool f32 = dtype == NFA_DTYPE_F32;
    // dz in two parts: 64 rows.  fp16, x in two parts too, 128 x 128 by eight waves (2^18 x 256 x 256 184 us against 288 by 64 x 128), 64 x 64
    // where one side is narrow (2^18 x 256 -> 64 73 us against 76 by 64 x 128, 2^18 x 65 -> 63 60 against 84)
    const bool both = two_parts && dtype == NFA_DTYPE_F16;
    w.bp = n <= 64 || (two_parts && !both) ? 64 : 128;
    w.bq = k <= 64 ? 64 : k <= 128 || two_parts || w.bp == 64 ? 128 : 256;
    if (both && w.bp != w.bq) w.bp = w.bq = 64;
    if (f32)
        while (w.bq > 64 && pad(k, w.bq / 2) < pad(k, w.bq)) w.bq /= 2;
    // and not where the rows are too few for a workgroup on every CU (4096 x 256 x 256 bf16 12 us by 64 x 64, 18 by 128 x 256)
    const int64_t most = ceil_div(rows, 4 * stage);
    if (ceil_div(n, w.bp) * ceil_div(k, w.bq) * most < kNumCU) w.bp = w.bq = 64;
    const int64_t tiles = ceil_div(n, w.bp) * ceil_div(k, w.bq);
    // workgroups on a CU: one of 128 x 256; two otherwise (2^18 x 64 x 64 bf16 20 us, 25 with four; narrow layers 2^18 x 8 x 32 14.4, 15.5
    // with four), but four of 64 x 64 in fp32, whose steps are short (2^18 x 129 x 32: 109 us, 129 with two)
    const int64_t per_cu = w.bq == 256 || (both && w.bq == 128) ? 1 : f32 && w.bp == 64 && w.bq == 64 && !narrow_layer(n, k) ? 4 : 2;
    int64_t splits = ceil_div(per_cu * kNumCU, tiles);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    w.split = ceil_div(ceil_div(rows, splits), stage) * stage;
    w.splits = ceil_div(rows, w.split);
    return w;
}

// relu keeps a bit of each number, a byte a chunk.  Rows that do not divide into chunks are differentiated from the value instead, but in
// fp16, where values below 2^-25 round to 0
bool keeps_bits(int64_t out_features, int32_t dtype, int32_t act) {
    return act == NFA_ACT_RELU && (dtype == NFA_DTYPE_F16 || out_features % (16 / dtype_bytes(dtype)) == 0);
}
int64_t bit_bytes(int64_t out_features, int32_t dtype) { return ceil_div(out_features, 16 / dtype_bytes(dtype)); }     // of a row
bool two_parts(int32_t dtype, int32_t act) { return dtype != NFA_DTYPE_F32 && act != NFA_ACT_NONE && act != NFA_ACT_RELU; }
bool keeps_slopes(int32_t dtype, int32_t act) { return dtype == NFA_DTYPE_F16 && two_parts(dtype, act); }     // in 32 bits

}  // namespace

__global__ __launch_bounds__(kBlock) void zero_kernel(uint16_t *p, int64_t n) {
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < n; e += (int64_t)gridDim.x * kBlock) p[e] = 0;
}
void launch_zero(void *p, int64_t n, int32_t dtype, hipStream_t s) {
    n *= dtype_bytes(dtype) / 2;
    if (p && n > 0) hipLaunchKernelGGL(zero_kernel, dim3(blocks_for(n)), dim3(kBlock), 0, s, (uint16_t *)p, n);
}

void launch_reduce_rows(float *part, int64_t rows, std::initializer_list<std::pair<void *, int64_t>> outputs, int32_t dtype, hipStream_t s) {
    Outputs o{};
    int64_t cols = 0, k = 0;
    for (auto &p : outputs) {
        o.to[k] = p.first;
        o.cols[k++] = p.second;
        cols += p.second;
    }
    const unsigned blocks = (unsigned)ceil_div(cols, 64);
    // few rows of many columns, a thread a column: the weight gradient of 4096 x 1024 x 1024 bf16, 8 rows of 2^20 columns, takes 34 us
    // against 63 with sixteen groups a column, that of 65536 x 256 x 512, 64 rows of 2^17, 49 against 52
    if (rows <= 64 && cols >= 64 * kNumCU) {
        with_dtype(dtype, [&](auto t) {
            hipLaunchKernelGGL((reduce_few_rows_kernel<decltype(t)>), dim3((unsigned)ceil_div(cols, kBlock)), dim3(kBlock), 0, s, part, rows, cols, o);
        });
        return;
    }
    // one launch while it fills the chip or its rows are few: 4096 rows of 1152 columns take 19 us in one, 10 in two
    int64_t step = 1;
    if (rows >= 1024 && blocks < 2 * kNumCU) {
        step = 128;
        hipLaunchKernelGGL((reduce_rows_kernel<float, false>), dim3(blocks, (unsigned)ceil_div(rows, step)), dim3(1024), 0, s, part, rows, step, (int64_t)1, cols, o);
    }
    with_dtype(dtype, [&](auto t) {
        hipLaunchKernelGGL((reduce_rows_kernel<decltype(t), true>), dim3(blocks), dim3(1024), 0, s, part, rows, rows, step, cols, o);
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
    if (keeps_bits(out_features, dtype, activation)) return rows * bit_bytes(out_features, dtype);
    if (keeps_slopes(dtype, activation)) return rows * out_features * 4;
    if (activation == NFA_ACT_NONE || (act_from_value(activation) && !has_residual)) return 0;
    return rows * out_features * dtype_bytes(dtype);
}

NFA_EXPORT int nfa_linear_fwd(const nfa_linear_args *a, void *outputs, void *saved, void *stream) {
    if (int rc = check_linear(a, "linear_fwd")) return rc;
    if (a->rows == 0) return NFA_OK;
    NFA_REQUIRE(outputs, "linear_fwd: NULL pointer");
    NFA_REQUIRE(!a->residual || a->residual_stride >= a->out_features || a->rows == 1, "linear_fwd: residual_stride < out_features");
    const int64_t bytes = dtype_bytes(a->dtype);
    if (nfa_linear_saved_bytes(a->rows, a->out_features, a->dtype, a->activation, a->residual != nullptr) == 0) saved = nullptr;
    DenseArgs d{};
    d.p = a->inputs; d.ld_p = a->inputs_stride;
    d.q = a->weight; d.ld_q = a->in_features;
    d.bias = a->bias; d.residual = a->residual; d.ld_residual = a->residual_stride;
    d.out = outputs; d.saved_out = saved;
    d.n_p = a->rows; d.n_q = a->out_features; d.n_c = a->in_features;
    d.act = a->activation;
    d.mask = keeps_bits(a->out_features, a->dtype, a->activation);
    d.ld_saved = d.mask ? bit_bytes(a->out_features, a->dtype) : a->out_features;
    d.vec = aligned(d.p, d.ld_p, a->in_features, bytes, 16) && aligned(d.q, d.ld_q, a->in_features, bytes, 16) &&
            aligned(outputs, d.n_q, d.n_q, bytes, 16) && (!saved || d.mask || aligned(saved, d.n_q, d.n_q, keeps_slopes(a->dtype, a->activation) ? 4 : bytes, 16)) &&
                (!a->residual || aligned(a->residual, a->residual_stride, d.n_q, bytes, 16));
    int rc = NFA_OK;
    with_dtype(a->dtype, [&](auto t) { rc = launch_rows<decltype(t), kForward, false>(d, (hipStream_t)stream); });
    return rc;
}

NFA_EXPORT int64_t nfa_linear_bwd_workspace_bytes(int64_t rows, int32_t in_features, int32_t out_features, int32_t dtype, int32_t activation) {
    if (rows <= 0 || in_features <= 0 || out_features <= 0) return 0;
    const WgradPlan w = wgrad_plan(rows, out_features, in_features, dtype, two_parts(dtype, activation));
    return w.splits * ((int64_t)out_features * in_features + out_features) * 4;
}

NFA_EXPORT int nfa_linear_bwd(const nfa_linear_args *a, const void *saved, void *grad_inputs, void *grad_weight, void *grad_bias,
                              void *workspace, void *stream) {
    if (int rc = check_linear(a, "linear_bwd")) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (a->rows == 0) {
        launch_zero(grad_weight, (int64_t)a->out_features * a->in_features, a->dtype, s);
        launch_zero(grad_bias, a->out_features, a->dtype, s);
        return check_launch("zero_kernel");
    }
    NFA_REQUIRE(a->grad_outputs, "linear_bwd: NULL pointer");
    NFA_REQUIRE(a->grad_outputs_stride >= a->out_features || a->rows == 1, "linear_bwd: grad_outputs_stride < out_features");
    NFA_REQUIRE(saved || a->activation == NFA_ACT_NONE, "linear_bwd: the activation needs what the forward call saved");
    NFA_REQUIRE(workspace || !(grad_weight || grad_bias), "linear_bwd: NULL workspace");
    NFA_REQUIRE(!(grad_weight || grad_bias) || ((int64_t)a->in_features + 1) * a->out_features < kMaxThreads - kBlock,
                "linear_bwd: too many weights for one launch");
    const int64_t bytes = dtype_bytes(a->dtype), n = a->out_features, k = a->in_features;
    const bool split = two_parts(a->dtype, a->activation);
    DenseArgs d{};
    d.p = a->grad_outputs; d.ld_p = a->grad_outputs_stride;
    d.saved = saved;
    d.act = a->activation;
    d.mask = keeps_bits(n, a->dtype, a->activation);
    d.ld_saved = d.mask ? bit_bytes(n, a->dtype) : n;
    const bool vec = aligned(a->grad_outputs, a->grad_outputs_stride, n, bytes, 16) &&
              (!saved || a->activation == NFA_ACT_NONE || d.mask || aligned(saved, n, n, keeps_slopes(a->dtype, a->activation) ? 4 : bytes, 16));
    int rc = NFA_OK;
    if (grad_inputs) {
        DenseArgs e = d;
        e.q = a->weight; e.ld_q = k;
        e.out = grad_inputs;
        e.vec = vec && aligned(a->weight, k, k, bytes, 16) && aligned(grad_inputs, k, k, bytes, 16);
        e.n_p = a->rows; e.n_q = (int32_t)k; e.n_c = n;
        with_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            if constexpr (sizeof(T) == 2)
                if (split) { rc = launch_rows<T, kDgrad, true>(e, s); return; }
            rc = launch_rows<T, kDgrad, false>(e, s);
        });
        if (rc) return rc;
    }
    if (grad_weight || grad_bias) {
        const WgradPlan w = wgrad_plan(a->rows, n, k, a->dtype, split);
        DenseArgs e = d;
        e.q = a->inputs; e.ld_q = a->inputs_stride;
        e.vec = vec && aligned(a->inputs, a->inputs_stride, k, bytes, 16);
        e.partial = (float *)workspace;
        e.n_p = n; e.n_q = (int32_t)k; e.n_c = a->rows;
        e.split = w.split;
        e.want_bias = grad_bias != nullptr;
        with_dtype(a->dtype, [&](auto t) {
            using T = decltype(t);
            if constexpr (sizeof(T) == 2)
                if (split) {
                    if (w.bq == 64) rc = launch_tiles<T, kWgrad, 64, 64, 2, 2, true>(e, w.splits, s);
                    else if constexpr (std::is_same_v<T, f16>) rc = launch_tiles<T, kWgrad, 128, 128, 2, 4, true>(e, w.splits, s);
                    else rc = launch_tiles<T, kWgrad, 64, 128, 2, 2, true>(e, w.splits, s);
                    return;
                }
            // 2^18 x 8 x 32: 14.4 us against 33 by tiles of 64 x 64, 32 x 32 17.4 against 34, 64 x 64 39.3 against 39.7
            if constexpr (sizeof(T) == 4)
                if (e.vec && narrow_layer(n, k)) {
                    rc = n <= 16 ? launch_narrow_wgrad<1>(e, w.splits, s) : n <= 32 ? launch_narrow_wgrad<2>(e, w.splits, s) : launch_narrow_wgrad<4>(e, w.splits, s);
                    return;
                }
            if (w.bp == 64) rc = w.bq == 64 ? launch_tiles<T, kWgrad, 64, 64, 2, 2, false>(e, w.splits, s) : launch_tiles<T, kWgrad, 64, 128, 2, 2, false>(e, w.splits, s);
            else if (w.bq == 64) rc = launch_tiles<T, kWgrad, 128, 64, 2, 2, false>(e, w.splits, s);
            else rc = w.bq == 128 ? launch_tiles<T, kWgrad, 128, 128, 2, 2, false>(e, w.splits, s) : launch_tiles<T, kWgrad, 128, 256, 2, 4, false>(e, w.splits, s);
        });
        if (rc) return rc;
        launch_reduce_rows(e.partial, w.splits, {{grad_weight, n * k}, {grad_bias, n}}, a->dtype, s);
        return check_launch("reduce_rows_kernel");
    }
    return NFA_OK;
}
