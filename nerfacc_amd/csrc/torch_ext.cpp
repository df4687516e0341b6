// torch_ext.cpp — the PyTorch-ROCm C++ extension in front of libnerfacc_hip.so (module `nerfacc_amd._hip`).
//
// Same role as the reference's pybind module `nerfacc.csrc` (nerfacc/cuda/csrc/nerfacc.cpp:126-163): the 21
// names of that module with the same argument order, plus the fused entry points of this implementation.
// The reference's functions take torch::Tensor, allocate their outputs from the caching allocator, launch on
// the current stream under a device guard and block the host only where a size is needed (data_spec.hpp:91);
// so do these.  All kernels live behind the C ABI of include/nerfacc_hip.h — this file is host plumbing only:
// argument checks (CHECK_INPUT, utils_cuda.cuh:12-17), allocation, the readback of the few integers that size
// an output, the cache of the bit-packed occupancy grid.  No CPU path: a host tensor is an error.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <chrono>
#include <limits>
#include <map>
#include <mutex>
#include <optional>
#include <set>
#include <string>
#include <thread>
#include <tuple>
#include <vector>

#include "../../include/nerfacc_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------------------------------
// small helpers
// ---------------------------------------------------------------------------------------------------
inline void check_rc(int rc) {
    TORCH_CHECK(rc == NFA_OK, "nerfacc_amd: ", nfa_last_error());
}

// the library's option table (nfa_set_option): 0 = launch the emit pass after the read-back of the totals
inline bool speculative_emit_allowed() {
    int64_t v = 1;
    int32_t is_set = 0;
    nfa_get_option("speculative_emit", &v, &is_set);
    return !is_set || v != 0;
}

inline void check_input(const Tensor &t, const char *name, std::optional<at::ScalarType> dtype = std::nullopt) {
    TORCH_CHECK(t.defined(), name, " is undefined");
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA/HIP tensor (nerfacc_amd has no CPU kernels)");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    if (dtype) TORCH_CHECK(t.scalar_type() == *dtype, name, " must have dtype ", *dtype, ", got ", t.scalar_type());
}

// 1-D (or [n, inner]) tensor of the given dtype with exactly n leading elements, on the reference tensor's device
inline void check_len(const Tensor &t, const char *name, at::ScalarType dtype, int64_t n, const Tensor &like, int64_t inner = 1) {
    check_input(t, name, dtype);
    TORCH_CHECK(t.numel() == n * inner, name, " must have ", n * inner, " elements, got ", t.numel());
    TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}
inline void check_len(const OptTensor &t, const char *name, at::ScalarType dtype, int64_t n, const Tensor &like, int64_t inner = 1) {
    if (t) check_len(*t, name, dtype, n, like, inner);
}

template <class T> inline T *ptr(const Tensor &t) { return t.defined() ? reinterpret_cast<T *>(t.data_ptr()) : nullptr; }
template <class T> inline T *ptr(const OptTensor &t) { return (t && t->defined()) ? reinterpret_cast<T *>(t->data_ptr()) : nullptr; }

inline hipStream_t stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

using Guard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

inline at::TensorOptions opts(const Tensor &like, at::ScalarType dt) { return like.options().dtype(dt); }

[[noreturn]] void raise_not_implemented(const char *msg) {
    PyErr_SetString(PyExc_NotImplementedError, msg);
    throw py::error_already_set();
}

// ---------------------------------------------------------------------------------------------------
// optional HIP-event timing of named single-kernel calls (bench.py's live roofline measurement).  Events are
// recorded on the stream the kernel is launched on; nothing is synchronised until timing_summary().
// ---------------------------------------------------------------------------------------------------
struct Timing {
    std::mutex mu;
    bool on = false;
    std::vector<std::string> names;
    std::map<std::string, std::vector<std::pair<hipEvent_t, hipEvent_t>>> records;
} g_timing;

struct Timed {
    const char *name;
    hipStream_t s;
    hipEvent_t e0 = nullptr, e1 = nullptr;
    Timed(const char *n, hipStream_t st) : name(n), s(st) {
        if (!g_timing.on) return;
        std::lock_guard<std::mutex> l(g_timing.mu);
        bool want = false;
        for (auto &x : g_timing.names) want |= (x == n);
        if (!want) return;
        hipEventCreate(&e0);
        hipEventCreate(&e1);
        hipEventRecord(e0, s);
    }
    ~Timed() {
        if (!e0) return;
        hipEventRecord(e1, s);
        std::lock_guard<std::mutex> l(g_timing.mu);
        g_timing.records[name].emplace_back(e0, e1);
    }
};

// names = None stops recording and KEEPS what was recorded (timing_summary reads it); a list starts afresh
void set_timing(std::optional<std::vector<std::string>> names) {
    std::lock_guard<std::mutex> l(g_timing.mu);
    if (names.has_value()) {
        for (auto &kv : g_timing.records)
            for (auto &p : kv.second) { hipEventDestroy(p.first); hipEventDestroy(p.second); }
        g_timing.records.clear();
    }
    g_timing.on = names.has_value();
    g_timing.names = names.value_or(std::vector<std::string>{});
}

py::dict timing_summary() {
    hipDeviceSynchronize();
    std::lock_guard<std::mutex> l(g_timing.mu);
    py::dict out;
    for (auto &kv : g_timing.records) {
        double total = 0.0;
        for (auto &p : kv.second) { float ms = 0.f; hipEventElapsedTime(&ms, p.first, p.second); total += ms; }
        const size_t n = kv.second.size();
        out[py::str(kv.first)] = py::make_tuple(n, n ? total / n : 0.0);
    }
    return out;
}

// ---------------------------------------------------------------------------------------------------
// host readback of the few integers a call needs (sample totals, kept counts): the kernels store them straight
// into pinned host memory, so the readback is a stream wait plus a CPU load.  One slot per (device, stream,
// host thread): the calls stay re-entrant across threads and streams like the reference's stateless functions.
// ---------------------------------------------------------------------------------------------------
// false once a slot had to be allocated without hipHostMallocCoherent: a polling host may then never see a running kernel's
// store, so wait_stamp synchronises the stream straight away instead of spinning for its 2 ms first
std::atomic<bool> g_host_ints_coherent{true};

int64_t *host_ints(int device, hipStream_t s, int which = 0) {
    // which = 1: the slot of a count pass launched AHEAD of its call (sample_occgrid's next-chunk prefetch): the calls in between
    // (visibility_compact of the current chunk) keep using slot 0
    thread_local std::map<std::tuple<int, hipStream_t, int>, int64_t *> slots;
    auto key = std::make_tuple(device, s, which);
    auto it = slots.find(key);
    if (it != slots.end()) return it->second;
    int64_t *p = nullptr;
    // coherent (fine-grained) pinned memory: a kernel's store is visible to a polling host while the kernel runs (wait_stamp)
    if (hipHostMalloc(reinterpret_cast<void **>(&p), 8 * sizeof(int64_t), hipHostMallocCoherent) != hipSuccess) {
        (void)hipGetLastError();
        TORCH_CHECK(hipHostMalloc(reinterpret_cast<void **>(&p), 8 * sizeof(int64_t), hipHostMallocDefault) == hipSuccess,
                    "nerfacc_amd: hipHostMalloc failed");
        g_host_ints_coherent = false;
    }
    for (int i = 0; i < 8; ++i) p[i] = 0;
    if (slots.size() > 64) slots.clear();      // (slots of dead streams are leaked: 64 B each)
    slots[key] = p;
    return p;
}

// The read-backs of this file wait for ONE word: the kernel that produces the integers stores the caller's stamp behind them
// (system-scope fence), and the host polls that word instead of asking the runtime to synchronise the stream — 1-2 us instead of
// the 8-9 us a hipStreamSynchronize takes to come back (tools/sync_latency.py), and the host is released when the integers exist,
// not when the kernel that wrote them (and goes on to write its outputs) has finished.  Bounded: after ~2 ms of polling the
// stream is synchronised the ordinary way (a launch that failed, a size range whose kernels do not stamp).
inline int64_t next_stamp() {
    thread_local int64_t seq = 0;
    return ++seq;
}
inline void wait_stamp(const int64_t *slot, int64_t stamp, hipStream_t s) {
    py::gil_scoped_release nogil;
    const volatile int64_t *p = slot;
    const auto t0 = std::chrono::steady_clock::now();
    for (int64_t spins = 0; g_host_ints_coherent.load(std::memory_order_relaxed); ++spins) {
        if (*p == stamp) { std::atomic_thread_fence(std::memory_order_acquire); return; }
        if ((spins & 1023) == 1023 && std::chrono::steady_clock::now() - t0 > std::chrono::milliseconds(2)) break;
    }
    TORCH_CHECK(hipStreamSynchronize(s) == hipSuccess, "nerfacc_amd: hipStreamSynchronize failed");
}

inline void wait_stream(hipStream_t s) {
    py::gil_scoped_release nogil;               // other Python threads may run while this one waits for its stream
    TORCH_CHECK(hipStreamSynchronize(s) == hipSuccess, "nerfacc_amd: hipStreamSynchronize failed");
}

// ---------------------------------------------------------------------------------------------------
// occupancy bricks: packed once per distinct state of a `binaries` tensor (identity + in-place version)
// ---------------------------------------------------------------------------------------------------
struct BrickEntry {
    c10::weak_intrusive_ptr<c10::TensorImpl> ref;
    c10::TensorImpl *impl;
    uint32_t version;
    Tensor bricks;
    int64_t nonempty;
    int64_t level_counts[8];
    hipStream_t stream;
    hipEvent_t event;
};
std::mutex g_brick_mu;
std::vector<BrickEntry> g_bricks;     // most recently used first
constexpr size_t kBrickSlots = 4;

// caller holds g_brick_mu: makes `bricks` (packed on stream s) the front entry for this state of `binaries`
void insert_brick_entry(const Tensor &binaries, const Tensor &bricks, hipStream_t s) {
    c10::TensorImpl *impl = binaries.unsafeGetTensorImpl();
    hipEvent_t ev;
    hipEventCreateWithFlags(&ev, hipEventDisableTiming);
    hipEventRecord(ev, s);
    // drop slots whose tensor is gone or is this tensor in an older state, then the oldest
    std::vector<BrickEntry> keep;
    for (auto &c : g_bricks) {
        if (c.ref.expired() || c.impl == impl) { hipEventDestroy(c.event); continue; }
        keep.push_back(std::move(c));
    }
    g_bricks = std::move(keep);
    BrickEntry e{c10::weak_intrusive_ptr<c10::TensorImpl>(binaries.getIntrusivePtr()), impl, binaries._version(), bricks, -1,
                 {0, 0, 0, 0, 0, 0, 0, 0}, s, ev};
    g_bricks.insert(g_bricks.begin(), std::move(e));
    while (g_bricks.size() > kBrickSlots) { hipEventDestroy(g_bricks.back().event); g_bricks.pop_back(); }
}

// returns (bricks, number of non-empty bricks); reads the count back once per grid state
std::pair<Tensor, int64_t> brick_entry(const Tensor &binaries, bool need_count) {
    check_input(binaries, "binaries", at::kBool);
    TORCH_CHECK(binaries.dim() == 4, "binaries must have shape [n_grids, resx, resy, resz]");
    Guard g(device_of(binaries));                       // events and the copy below belong to the tensor's device
    std::lock_guard<std::mutex> l(g_brick_mu);
    hipStream_t s = stream_of(binaries);
    c10::TensorImpl *impl = binaries.unsafeGetTensorImpl();
    const uint32_t ver = binaries._version();
    size_t hit = g_bricks.size();
    for (size_t k = 0; k < g_bricks.size(); ++k) {
        auto &c = g_bricks[k];
        if (c.impl == impl && c.version == ver && !c.ref.expired()) { hit = k; break; }
    }
    if (hit == g_bricks.size()) {
        const int G = (int)binaries.size(0), rx = (int)binaries.size(1), ry = (int)binaries.size(2), rz = (int)binaries.size(3);
        const int64_t words = nfa_packed_grid_words(G, rx, ry, rz);
        Tensor bricks = at::empty({words}, opts(binaries, at::kLong));
        check_rc(nfa_pack_binaries(ptr<uint8_t>(binaries), G, rx, ry, rz, ptr<uint64_t>(bricks), s));
        insert_brick_entry(binaries, bricks, s);
        hit = 0;
    } else if (hit != 0) {
        BrickEntry e = std::move(g_bricks[hit]);
        g_bricks.erase(g_bricks.begin() + hit);
        g_bricks.insert(g_bricks.begin(), std::move(e));
        hit = 0;
    }
    auto &c = g_bricks[0];
    if (c.stream != s) hipStreamWaitEvent(s, c.event, 0);      // packed on another stream: order this one after the pack
    if (need_count && c.nonempty < 0) {
        const int64_t nb = binaries.size(0) * ((binaries.size(1) + 3) / 4) * ((binaries.size(2) + 3) / 4) * ((binaries.size(3) + 3) / 4);
        // header of the packed grid: [0] non-empty bricks, [1..8] occupied voxels per level
        int64_t hdr[9];
        TORCH_CHECK(hipMemcpyAsync(hdr, ptr<int64_t>(c.bricks) + nb, sizeof(hdr), hipMemcpyDeviceToHost, s) == hipSuccess,
                    "nerfacc_amd: readback of the packed-grid header failed");
        // (the GIL stays held: releasing it while holding g_brick_mu would let another Python thread block on the mutex
        // with the GIL, and this thread could then never take the GIL back.  Once per grid state, ~20 us.)
        TORCH_CHECK(hipStreamSynchronize(s) == hipSuccess, "nerfacc_amd: hipStreamSynchronize failed");
        c.nonempty = hdr[0];
        for (int g = 0; g < 8; ++g) c.level_counts[g] = hdr[1 + g];
    }
    return {c.bricks, c.nonempty};
}

Tensor packed_bricks(const Tensor &binaries) { return brick_entry(binaries, true).first; }

// occupied voxels per level of `binaries` (what nonzero(binaries[level]) would count), from the packed grid's header: one
// read-back per grid state, shared with the traversal's
std::vector<int64_t> grid_occupied_counts(const Tensor &binaries) {
    brick_entry(binaries, true);
    std::lock_guard<std::mutex> l(g_brick_mu);
    c10::TensorImpl *impl = binaries.unsafeGetTensorImpl();
    for (auto &c : g_bricks)
        if (c.impl == impl && c.version == binaries._version() && !c.ref.expired())
            return std::vector<int64_t>(c.level_counts, c.level_counts + std::min<int64_t>(binaries.size(0), 8));
    TORCH_CHECK(false, "nerfacc_amd: packed grid vanished from the cache");
}

void *sync_block(const Tensor &like, hipStream_t s);

// the occupied cells of level `lvl`, ascending (torch.nonzero(binaries[lvl].flatten())[:, 0], occ_grid.py:356) without rocprim's
// partition and without a read-back: the count comes from the packed grid's header
Tensor grid_occupied_cells(const Tensor &binaries, int64_t lvl) {
    check_input(binaries, "binaries", at::kBool);
    TORCH_CHECK(binaries.dim() == 4 && lvl >= 0 && lvl < binaries.size(0), "binaries must be [levels, rx, ry, rz] and lvl one of its levels");
    const std::vector<int64_t> counts = grid_occupied_counts(binaries);
    TORCH_CHECK(lvl < (int64_t)counts.size(), "grid_occupied_cells: level counts are kept for the first 8 levels");
    const int64_t n_cells = binaries.size(1) * binaries.size(2) * binaries.size(3), cnt = counts[lvl];
    Tensor out = at::empty({cnt}, opts(binaries, at::kLong));
    if (cnt == 0) return out;
    Guard g(device_of(binaries));
    hipStream_t s = stream_of(binaries);
    check_rc(nfa_grid_occupied_cells((const uint8_t *)binaries.data_ptr() + lvl * n_cells, n_cells, ptr<int64_t>(out), cnt, sync_block(binaries, s), s));
    return out;
}

// ---------------------------------------------------------------------------------------------------
// RaySegmentsSpec (data_spec.hpp:6-14; nerfacc.cpp:128-137): seven optional tensors
// ---------------------------------------------------------------------------------------------------
struct RaySegmentsSpec {
    OptTensor vals, is_left, is_right, is_valid, chunk_starts, chunk_cnts, ray_indices;

    void check() const {      // data_spec.hpp:15-51
        TORCH_CHECK(vals.has_value(), "RaySegmentsSpec.vals is not set");
        check_input(*vals, "vals", at::kFloat);
        if (vals->dim() > 1) return;
        TORCH_CHECK(chunk_starts && chunk_cnts, "flattened RaySegmentsSpec needs chunk_starts and chunk_cnts");
        check_input(*chunk_starts, "chunk_starts", at::kLong);
        check_input(*chunk_cnts, "chunk_cnts", at::kLong);
        TORCH_CHECK(chunk_starts->dim() == 1 && chunk_cnts->dim() == 1, "chunk_starts / chunk_cnts must be 1-D");
        TORCH_CHECK(chunk_starts->numel() == chunk_cnts->numel(), "chunk_starts and chunk_cnts differ in length");
        auto same = [&](const OptTensor &t, const char *n, at::ScalarType dt) {
            if (!t) return;
            check_input(*t, n, dt);
            TORCH_CHECK(t->dim() == 1 && t->numel() == vals->numel(), n, " must be 1-D with as many elements as vals");
        };
        same(ray_indices, "ray_indices", at::kLong);
        same(is_left, "is_left", at::kBool);
        same(is_right, "is_right", at::kBool);
        same(is_valid, "is_valid", at::kBool);
    }

    nfa_ray_segments view() const {
        nfa_ray_segments s{};
        s.vals = ptr<float>(vals);
        s.n_edges = vals->numel();
        if (vals->dim() > 1) {
            s.n_edges_per_ray = vals->size(-1);
            s.n_rays = vals->numel() / std::max<int64_t>(vals->size(-1), 1);
        } else {
            s.chunk_starts = ptr<int64_t>(chunk_starts);
            s.chunk_cnts = ptr<int64_t>(chunk_cnts);
            s.ray_indices = ptr<int64_t>(ray_indices);
            s.n_rays = chunk_cnts->numel();
        }
        return s;
    }
};

// ---------------------------------------------------------------------------------------------------
// grid
// ---------------------------------------------------------------------------------------------------
std::vector<Tensor> ray_aabb_intersect(const Tensor &rays_o, const Tensor &rays_d, const Tensor &aabbs, double near_plane,
                                       double far_plane, double miss_value) {   // nerfacc.cpp:63-69
    check_input(rays_o, "rays_o", at::kFloat);
    check_input(rays_d, "rays_d", at::kFloat);
    check_input(aabbs, "aabbs", at::kFloat);
    const int64_t R = rays_o.size(0), G = aabbs.size(0);
    Tensor t_mins = at::empty({R, G}, rays_o.options()), t_maxs = at::empty({R, G}, rays_o.options());
    Tensor hits = at::empty({R, G}, opts(rays_o, at::kBool));
    Guard g(device_of(rays_o));
    check_rc(nfa_ray_aabb_intersect(ptr<float>(rays_o), ptr<float>(rays_d), R, ptr<float>(aabbs), G, (float)near_plane,
                                    (float)far_plane, (float)miss_value, ptr<float>(t_mins), ptr<float>(t_maxs), ptr<uint8_t>(hits),
                                    stream_of(rays_o)));
    return {t_mins, t_maxs, hits};
}

nfa_traverse_args traverse_args(const Tensor &rays_o, const Tensor &rays_d, const OptTensor &rays_mask, const Tensor &binaries,
                                const Tensor &aabbs, const OptTensor &t_sorted, const OptTensor &t_indices, const OptTensor &hits,
                                const OptTensor &near_planes, const OptTensor &far_planes, double step_size, double cone_angle,
                                int64_t limit, Tensor &bricks_keepalive, double near_plane = 0.0,
                                double far_plane = std::numeric_limits<double>::infinity(), const OptTensor &t_min = std::nullopt,
                                const OptTensor &t_max = std::nullopt, const OptTensor &jitter = std::nullopt, double jitter_scale = 0.0) {
    check_input(rays_o, "rays_o", at::kFloat);
    check_input(rays_d, "rays_d", at::kFloat);
    check_input(aabbs, "aabbs", at::kFloat);
    const int64_t R = rays_o.size(0), G = binaries.size(0);
    auto per_ray = [&](const OptTensor &t, const char *name) {
        if (!t) return;
        check_input(*t, name, at::kFloat);
        TORCH_CHECK(t->numel() == R, name, " must have n_rays elements");
    };
    per_ray(near_planes, "near_planes");
    per_ray(far_planes, "far_planes");
    per_ray(t_min, "t_min");
    per_ray(t_max, "t_max");
    per_ray(jitter, "jitter");
    TORCH_CHECK(rays_o.dim() == 2 && rays_o.size(1) == 3 && rays_d.sizes() == rays_o.sizes(), "rays_o / rays_d must have shape [n_rays, 3]");
    TORCH_CHECK(rays_d.device() == rays_o.device() && binaries.device() == rays_o.device() && aabbs.device() == rays_o.device(),
                "rays_o, rays_d, binaries and aabbs must live on the same device");
    TORCH_CHECK(aabbs.dim() == 2 && aabbs.size(0) == G && aabbs.size(1) == 6, "aabbs must have shape [n_grids, 6]");
    nfa_traverse_args a{};
    a.near_plane = (float)near_plane;
    a.far_plane = (float)far_plane;
    a.t_min = ptr<float>(t_min);
    a.t_max = ptr<float>(t_max);
    a.jitter = ptr<float>(jitter);
    a.jitter_scale = (float)jitter_scale;
    a.n_rays = R;
    a.rays_o = ptr<float>(rays_o);
    a.rays_d = ptr<float>(rays_d);
    if (rays_mask) {
        check_input(*rays_mask, "rays_mask", at::kBool);
        a.rays_mask = ptr<uint8_t>(*rays_mask);
    }
    auto be = brick_entry(binaries, true);
    bricks_keepalive = be.first;
    a.n_grids = (int32_t)G;
    a.res[0] = (int32_t)binaries.size(1); a.res[1] = (int32_t)binaries.size(2); a.res[2] = (int32_t)binaries.size(3);
    a.bricks = ptr<uint64_t>(be.first);
    a.n_nonempty_bricks = be.second;
    a.aabbs = ptr<float>(aabbs);
    if (t_sorted) {
        TORCH_CHECK(t_indices && hits, "t_sorted, t_indices and hits must be given together");
        check_input(*t_sorted, "t_sorted", at::kFloat);
        check_input(*t_indices, "t_indices", at::kLong);
        check_input(*hits, "hits", at::kBool);
        TORCH_CHECK(t_sorted->dim() == 2 && t_sorted->size(0) == R && t_sorted->size(1) == 2 * G && t_indices->sizes() == t_sorted->sizes()
                        && hits->dim() == 2 && hits->size(0) == R && hits->size(1) == G,
                    "t_sorted/t_indices must be [n_rays, 2*n_grids], hits [n_rays, n_grids]");
        a.t_sorted = ptr<float>(*t_sorted);
        a.t_indices = ptr<int64_t>(*t_indices);
        a.hits = ptr<uint8_t>(*hits);
    }
    a.near_planes = ptr<float>(near_planes);
    a.far_planes = ptr<float>(far_planes);
    a.step_size = (float)step_size;
    a.cone_angle = (float)cone_angle;
    a.traverse_steps_limit = (int32_t)limit;
    return a;
}

// nerfacc.cpp:71-98 / grid.cu:320-474.  Two-pass mode: count -> offsets (device) -> ONE readback -> allocate -> fill; as
// in the reference it ignores rays_mask (grid.cu:418,450).
std::tuple<RaySegmentsSpec, RaySegmentsSpec, OptTensor> traverse_grids(
    const Tensor &rays_o, const Tensor &rays_d, const Tensor &rays_mask, const Tensor &binaries, const Tensor &aabbs,
    const OptTensor &t_sorted, const OptTensor &t_indices, const OptTensor &hits, const Tensor &near_planes, const Tensor &far_planes,
    double step_size, double cone_angle, bool compute_intervals, bool compute_samples, bool compute_terminate_planes,
    int64_t traverse_steps_limit, bool over_allocate) {
    TORCH_CHECK(!over_allocate || traverse_steps_limit > 0, "traverse_steps_limit must be > 0 when over_allocate is true");   // grid.cu:345
    check_input(rays_o, "rays_o", at::kFloat);
    const int64_t R = rays_o.size(0);
    const auto i64 = opts(rays_o, at::kLong), f32 = rays_o.options(), b8 = opts(rays_o, at::kBool);
    RaySegmentsSpec intervals, samples;
    OptTensor terminate;
    if (compute_terminate_planes) terminate = at::empty({R}, f32);
    Guard g(device_of(rays_o));
    hipStream_t s = stream_of(rays_o);
    Tensor keep;
    nfa_traverse_args a = traverse_args(rays_o, rays_d, over_allocate ? OptTensor(rays_mask) : std::nullopt, binaries, aabbs, t_sorted,
                                        t_indices, hits, OptTensor(near_planes), OptTensor(far_planes), step_size, cone_angle,
                                        traverse_steps_limit, keep);
    Tensor iv_cnts, iv_starts, sm_cnts, sm_starts, ws;
    int64_t n_edges = 0, n_samples = 0, n_overflow = 0;
    if (over_allocate) {
        // grid.cu:364-404: fixed-size slots, single pass, then starts from the actual counts
        Tensor maskl = rays_mask.to(at::kLong);
        iv_cnts = maskl * (2 * traverse_steps_limit);
        sm_cnts = maskl * traverse_steps_limit;
        iv_starts = at::empty_like(iv_cnts);
        sm_starts = at::empty_like(sm_cnts);
        int64_t *h = host_ints(rays_o.device().index(), s);
        check_rc(nfa_exclusive_sum_i64(ptr<int64_t>(iv_cnts), R, ptr<int64_t>(iv_starts), h, s));
        check_rc(nfa_exclusive_sum_i64(ptr<int64_t>(sm_cnts), R, ptr<int64_t>(sm_starts), h + 1, s));
        wait_stream(s);
        n_edges = h[0];
        n_samples = h[1];
    } else {
        if (compute_intervals) { iv_cnts = at::empty({R}, i64); iv_starts = at::empty({R}, i64); }
        sm_cnts = at::empty({R}, i64);
        sm_starts = at::empty({R}, i64);
        a.workspace_bytes = nfa_traverse_workspace_bytes_for(&a);
        ws = at::empty({std::max<int64_t>(a.workspace_bytes, 16)}, opts(rays_o, at::kByte));
        int64_t *h = host_ints(rays_o.device().index(), s);
        a.iv_cnts = ptr<int64_t>(iv_cnts); a.iv_starts = ptr<int64_t>(iv_starts);
        a.sm_cnts = ptr<int64_t>(sm_cnts); a.sm_starts = ptr<int64_t>(sm_starts);
        a.totals = h;
        a.terminate_planes = ptr<float>(terminate);
        check_rc(nfa_traverse_count(&a, ws.data_ptr(), s));
        check_rc(nfa_traverse_offsets(&a, ws.data_ptr(), s));
        wait_stream(s);                                       // the one host sync (data_spec.hpp:91)
        n_edges = h[0]; n_samples = h[1]; n_overflow = h[2];
    }
    a.iv_cnts = ptr<int64_t>(iv_cnts); a.iv_starts = ptr<int64_t>(iv_starts);
    a.sm_cnts = ptr<int64_t>(sm_cnts); a.sm_starts = ptr<int64_t>(sm_starts);
    auto alloc = [&](int64_t n, const at::TensorOptions &o) { return over_allocate ? at::zeros({n}, o) : at::empty({n}, o); };
    if (compute_intervals) {
        intervals.vals = alloc(n_edges, f32);
        intervals.ray_indices = alloc(n_edges, i64);
        Tensor flags = at::zeros({2, n_edges}, b8);
        intervals.is_left = flags[0];
        intervals.is_right = flags[1];
        a.iv_vals = ptr<float>(intervals.vals); a.iv_ray_indices = ptr<int64_t>(intervals.ray_indices);
        a.iv_is_left = ptr<uint8_t>(intervals.is_left); a.iv_is_right = ptr<uint8_t>(intervals.is_right);
    }
    if (compute_samples) {
        samples.vals = alloc(n_samples, f32);
        samples.ray_indices = alloc(n_samples, i64);
        samples.is_valid = alloc(n_samples, b8);
        a.sm_vals = ptr<float>(samples.vals); a.sm_ray_indices = ptr<int64_t>(samples.ray_indices);
        a.sm_is_valid = ptr<uint8_t>(samples.is_valid);
    }
    a.terminate_planes = ptr<float>(terminate);
    if (over_allocate) {
        if (R > 0) check_rc(nfa_traverse_fill(&a, 0, 1, nullptr, 0, 0, s));
        check_rc(nfa_exclusive_sum_i64(ptr<int64_t>(iv_cnts), R, ptr<int64_t>(iv_starts), nullptr, s));
        check_rc(nfa_exclusive_sum_i64(ptr<int64_t>(sm_cnts), R, ptr<int64_t>(sm_starts), nullptr, s));
    } else if (R > 0 && (compute_intervals || compute_samples) && n_samples > 0) {
        check_rc(nfa_traverse_fill(&a, 1, 0, ws.data_ptr(), n_samples, n_overflow, s));
    }
    if (compute_intervals) { intervals.chunk_cnts = iv_cnts; intervals.chunk_starts = iv_starts; }
    if (compute_samples) { samples.chunk_cnts = sm_cnts; samples.chunk_starts = sm_starts; }
    return {intervals, samples, terminate};
}

// k float rows of n elements from one allocation, each row 16-byte aligned (the tiled kernels then use vector accesses: 2 or 4 elements per lane)
struct Rows {
    Tensor buf;
    int64_t pitch, n;
    Rows(int64_t k, int64_t n_, const at::TensorOptions &o) : pitch((n_ + 3) & ~int64_t(3)), n(n_) { buf = at::empty({k, pitch}, o); }
    Rows(Tensor adopted, int64_t n_) : buf(std::move(adopted)), pitch(buf.size(1)), n(n_) {}      // a [k, pitch] tensor allocated ahead
    float *p(int64_t r) const { return buf.data_ptr<float>() + r * pitch; }
    Tensor row(int64_t r) const { return buf[r].narrow(0, 0, n); }
};

// The traversal's scratch (run records, block sums: nfa_traverse_workspace_bytes_for, up to 256 MB) is the same few MB call after
// call: one slab per (host thread, device, stream), grown when a call needs more, instead of an allocation per call.  Everything that
// touches it — count, offsets, emit of one call, then the next call's — is enqueued on that one stream, in order.
// A call that needs more than kWorkspaceKeep gets its own allocation (stream-ordered by torch's caching allocator, returned to it when
// the call ends): one frame-sized call does not pin a quarter of a GB for the life of the thread.
constexpr int64_t kWorkspaceKeep = 64ll << 20;
using SlabMap = std::map<std::pair<int, hipStream_t>, Tensor>;
SlabMap &workspace_slabs() {
    thread_local SlabMap slabs;
    return slabs;
}
Tensor traverse_workspace(const Tensor &like, hipStream_t s, int64_t bytes) {
    if (bytes > kWorkspaceKeep) return at::empty({bytes}, opts(like, at::kByte));
    Tensor &t = workspace_slabs()[{(int)like.device().index(), s}];
    if (!t.defined() || t.numel() < bytes)
        t = at::empty({std::min<int64_t>(std::max<int64_t>(bytes + bytes / 4, 1 << 16), kWorkspaceKeep)}, opts(like, at::kByte));
    return t;
}
// drops this host thread's retained slabs (and with them any count pass launched ahead: its records lived there)
void release_workspace();

// The sync block of the single-launch forms (include/nerfacc_hip.h: NFA_SYNC_BYTES, zero before its first use, left zero by every
// kernel that uses it): one per (host thread, device, stream), allocated zero-filled once.  Everything that touches it is enqueued
// on that one stream, in order.
SlabMap &sync_blocks() {
    thread_local SlabMap blocks;
    return blocks;
}
// Outputs of the NEXT single-launch sampling call of the same kind, allocated while the current call's launch is counting: the
// single launch needs its outputs to exist before it starts (the three-kernel form allocates them behind the count kernel's launch,
// for free), and two allocations in front of the launch are 4-5 us on the step's critical path — host wake-up to host wake-up is what
// bounds a training step at this size (tools/path_ab.py).  One set per (host thread, device, kind of call), at most kNextOutKeep bytes.
constexpr int64_t kNextOutKeep = 64ll << 20;
struct NextOut {
    Tensor ray_indices, rows;      // [cap] int64, [2, pitch] float
    int64_t cap = 0;
    hipStream_t stream = nullptr;
};
std::map<int, NextOut> &next_outputs() {
    thread_local std::map<int, NextOut> m;
    return m;
}

void *sync_block(const Tensor &like, hipStream_t s) {
    Tensor &t = sync_blocks()[{(int)like.device().index(), s}];
    if (!t.defined()) t = at::zeros({(int64_t)NFA_SYNC_BYTES}, opts(like, at::kByte));
    return t.data_ptr();
}

// The reference's eval loop (examples/utils.py:80-88) calls `estimator.sampling` on consecutive 8192-ray SLICES of one ray array, and
// every call has to wait for its count pass before it can size its outputs (~40 us of 205 per chunk with the host idle, profiles/
// r03_host_share.md).  When a call's rays start exactly where the previous call's ended — the second consecutive slice — the count
// and offsets kernels of the NEXT slice are launched at the end of the call, behind its own work; the next call, if it asks for
// exactly those rays (same pointers and count, same tensor versions, same grid, same scalars), finds its totals waiting.  A guess
// that is not taken up costs one count pass of GPU time and nothing else: nothing it wrote is looked at.  Only plain calls qualify
// (no jitter, masks, per-ray planes or step limits: training batches are fresh tensors and never match).  `chunk_prefetch` = 0
// switches it off.
struct ChunkPrefetch {
    bool valid = false;
    const void *o_ptr = nullptr, *d_ptr = nullptr, *aabbs_ptr = nullptr;
    const void *bin_impl = nullptr;
    int64_t R = 0;
    uint32_t o_ver = 0, d_ver = 0, bin_ver = 0, aabbs_ver = 0;
    double step = 0, cone = 0, near_plane = 0, far_plane = 0;
    int64_t stamp = 0, ws_bytes = 0;
    Tensor ws_keep;                     // the workspace the guess's run records live in (held: the taking call uses exactly this one)
    Tensor packed;
    const void *expect_o = nullptr;     // where the next slice of the caller's loop would start (set by every qualifying call)
    // The guess is keyed on IDENTITY, not only on addresses: weak references to the storages of both ray arrays, of the boxes and to
    // the grid tensor.  A weak reference keeps the (small) StorageImpl / TensorImpl object alive, so a live guess's pointer cannot be
    // handed to another object, and an expired one says the memory behind the recorded address may have been freed and re-used (a
    // fresh tensor at the same address starts at version 0 again).  It does not keep the caller's memory alive.
    c10::weak_intrusive_ptr<c10::StorageImpl> o_st{c10::intrusive_ptr<c10::StorageImpl>()}, d_st{c10::intrusive_ptr<c10::StorageImpl>()},
        aabbs_st{c10::intrusive_ptr<c10::StorageImpl>()};
    c10::weak_intrusive_ptr<c10::TensorImpl> bin_ref{c10::intrusive_ptr<c10::TensorImpl>()};
    bool same_storage(const c10::weak_intrusive_ptr<c10::StorageImpl> &w, const Tensor &t) const {
        return !w.expired() && w._unsafe_get_target() == t.storage().unsafeGetStorageImpl();
    }
    void drop() {
        valid = false;
        packed = Tensor();
        ws_keep = Tensor();
        o_st = d_st = aabbs_st = c10::weak_intrusive_ptr<c10::StorageImpl>(c10::intrusive_ptr<c10::StorageImpl>());
        bin_ref = c10::weak_intrusive_ptr<c10::TensorImpl>(c10::intrusive_ptr<c10::TensorImpl>());
    }
};
std::map<std::pair<int, hipStream_t>, ChunkPrefetch> &prefetch_slots() {
    thread_local std::map<std::pair<int, hipStream_t>, ChunkPrefetch> slots;
    return slots;
}
ChunkPrefetch &chunk_prefetch(int device, hipStream_t s) {
    auto &slots = prefetch_slots();
    if (slots.size() > 64) slots.clear();
    return slots[{device, s}];
}
void release_workspace() {
    prefetch_slots().clear();
    workspace_slabs().clear();
    sync_blocks().clear();
    next_outputs().clear();
}
inline bool chunk_prefetch_allowed() {
    int64_t v = 1;
    int32_t is_set = 0;
    nfa_get_option("chunk_prefetch", &v, &is_set);
    return !is_set || v != 0;
}

// traverse_grids + the two is_left / is_right compactions of occ_grid.py:164-177 in one count pass and one emit pass:
// (ray_indices, t_starts, t_ends, packed_info[, terminate_planes]).  rays_mask / traverse_steps_limit give one round of the
// test-time marcher (examples/utils.py:349-372) with exactly sized outputs.
py::tuple sample_occgrid(const Tensor &rays_o, const Tensor &rays_d, const Tensor &binaries, const Tensor &aabbs,
                         const OptTensor &near_planes, const OptTensor &far_planes, double step_size, double cone_angle,
                         const OptTensor &rays_mask, int64_t traverse_steps_limit, bool with_terminate_planes, double near_plane,
                         double far_plane, const OptTensor &t_min, const OptTensor &t_max, const OptTensor &jitter, double jitter_scale) {
    check_input(rays_o, "rays_o", at::kFloat);
    const int64_t R = rays_o.size(0);
    const auto i64 = opts(rays_o, at::kLong), f32 = rays_o.options();
    Guard g(device_of(rays_o));
    hipStream_t s = stream_of(rays_o);
    Tensor keep;
    nfa_traverse_args a = traverse_args(rays_o, rays_d, rays_mask, binaries, aabbs, std::nullopt, std::nullopt, std::nullopt,
                                        near_planes, far_planes, step_size, cone_angle, traverse_steps_limit, keep, near_plane, far_plane,
                                        t_min, t_max, jitter, jitter_scale);
    // a plain call (what the reference's eval loop makes): may take up, and leave behind, a count pass launched ahead
    // (tensors created under torch.inference_mode() carry no version counter — `_version()` throws for them — so a call with any
    //  of them neither takes up nor leaves a guess: ADVICE r4.  Writes that bypass the version counter — `x.data.copy_`, raw-pointer
    //  kernels, DLPack consumers — are invisible to this key: such callers set chunk_prefetch = 0.)
    const bool plain = R > 0 && !rays_mask && !near_planes && !far_planes && !t_min && !t_max && !jitter && traverse_steps_limit <= 0 &&
                       !with_terminate_planes && !rays_o.is_inference() && !rays_d.is_inference() && !aabbs.is_inference() &&
                       !binaries.is_inference();
    ChunkPrefetch &pf = chunk_prefetch(rays_o.device().index(), s);
    a.workspace_bytes = nfa_traverse_workspace_bytes_for(&a);
    const bool taken = plain && pf.valid && pf.o_ptr == rays_o.data_ptr() && pf.d_ptr == rays_d.data_ptr() && pf.R == R &&
                       pf.same_storage(pf.o_st, rays_o) && pf.same_storage(pf.d_st, rays_d) && pf.same_storage(pf.aabbs_st, aabbs) &&
                       !pf.bin_ref.expired() && pf.bin_impl == (const void *)binaries.unsafeGetTensorImpl() &&
                       pf.o_ver == rays_o._version() && pf.d_ver == rays_d._version() && pf.bin_ver == binaries._version() &&
                       pf.aabbs_ptr == aabbs.data_ptr() && pf.aabbs_ver == aabbs._version() && pf.step == step_size &&
                       pf.cone == cone_angle && pf.near_plane == near_plane && pf.far_plane == far_plane &&
                       pf.ws_bytes == a.workspace_bytes && pf.ws_keep.defined();
    Tensor ws = taken ? pf.ws_keep : traverse_workspace(rays_o, s, a.workspace_bytes);
    Tensor packed = taken ? pf.packed : at::empty({2, R}, i64);           // [starts; cnts], handed out transposed as [R, 2]
    const int64_t pf_stamp = pf.stamp;
    pf.drop();                                        // taken up or stale: either way it is spent
    int64_t *h = host_ints(rays_o.device().index(), s, taken ? 1 : 0);
    a.sm_starts = ptr<int64_t>(packed);
    a.sm_cnts = ptr<int64_t>(packed) + R;
    a.totals = h;
    Tensor term;
    if (with_terminate_planes) {
        TORCH_CHECK(near_planes.has_value(), "with_terminate_planes needs near_planes as a tensor");
        term = near_planes->clone();
        a.terminate_planes = ptr<float>(term);
    }
    // The emit pass runs BEFORE the read-back, into outputs sized from the previous call on this device (training
    // steps draw about the same number of samples every time): the GPU goes from counting straight into it
    // instead of idling through the host's wake-up, allocation and launch (16 us, tools/step_timeline.py), and the host —
    // released by the stamp behind the totals, not by the end of the emit pass — prepares the caller's next kernels while it
    // runs.  A guess that is too small costs nothing but the second launch the old order always needed.
    // The guess is SAMPLES PER RAY of the previous call of the same kind on this device (training batches, eval chunks and
    // marcher rounds differ by orders of magnitude in size but much less in samples per ray), times this call's ray count.
    thread_local std::map<int, double> last_spr;
    const int dev = rays_o.device().index() * 4 + (rays_mask.has_value() ? 1 : 0) + (traverse_steps_limit > 0 ? 2 : 0);
    const bool speculate = R > 0 && last_spr.count(dev) && last_spr[dev] > 0.0 && speculative_emit_allowed();
    int64_t cap = speculate ? (int64_t)(1.25 * last_spr[dev] * (double)R) + 1024 : 0;
    Tensor ray_indices;
    Rows ts(2, 0, f32);
    auto speculative_outputs = [&]() {
        ts = Rows(2, cap, f32);
        if (!speculate) return;
        ray_indices = at::empty({cap}, i64);
        a.sm_ray_indices = ptr<int64_t>(ray_indices);
        a.t_starts = ts.p(0);
        a.t_ends = ts.p(1);
    };
    int64_t stamp;
    if (taken) {
        stamp = pf_stamp;                             // count and offsets of exactly this call ran behind the previous one
        speculative_outputs();
        a.terminate_planes = nullptr;
        if (speculate) {
            Timed t("traverse_fill", s);
            check_rc(nfa_traverse_emit_speculative(&a, ws.data_ptr(), cap, s));
        }
    } else if (nfa_traverse_sample_fused(&a)) {
        // ONE launch counts, forms the offsets (look-back over the count kernel's workgroups) and expands every wave's own rays
        // (round 6; three launches before): the outputs have to exist first — normally they do, allocated behind the previous
        // call's launch (next_outputs)
        NextOut &no = next_outputs()[dev];
        if (speculate && no.ray_indices.defined() && no.stream == s && no.cap >= cap && no.cap <= 2 * cap + 4096) {
            cap = no.cap;
            ray_indices = std::move(no.ray_indices);
            ts = Rows(std::move(no.rows), cap);
            a.sm_ray_indices = ptr<int64_t>(ray_indices);
            a.t_starts = ts.p(0);
            a.t_ends = ts.p(1);
        } else {
            speculative_outputs();
        }
        no = NextOut{};
        stamp = next_stamp();
        h[3] = 0;
        int32_t did = 0;
        {
            Timed t("traverse_sample", s);
            check_rc(nfa_traverse_sample(&a, ws.data_ptr(), cap, stamp, sync_block(rays_o, s), &did, s));
        }
        a.terminate_planes = nullptr;                 // written by the count pass only
        if (speculate && 16 * cap <= kNextOutKeep) {  // (while the launch counts)
            no.cap = cap;
            no.stream = s;
            no.ray_indices = at::empty({cap}, i64);
            no.rows = at::empty({2, (cap + 3) & ~int64_t(3)}, f32);
        }
    } else {
        {
            Timed t("traverse_count", s);
            check_rc(nfa_traverse_count(&a, ws.data_ptr(), s));
        }
        stamp = next_stamp();
        h[3] = 0;
        check_rc(nfa_traverse_offsets_stamped(&a, ws.data_ptr(), stamp, s));
        speculative_outputs();                        // (allocated while the count pass runs)
        a.terminate_planes = nullptr;                 // written by the count pass only
        if (speculate) {
            Timed t("traverse_fill", s);
            check_rc(nfa_traverse_emit_speculative(&a, ws.data_ptr(), cap, s));
        }
    }
    if (R > 0) wait_stamp(h + 3, stamp, s);
    else wait_stream(s);
    bool emitted = speculate;
    if (R > 0 && h[1] < 0) {
        // the fused launch's look-back gave up (a bounded wait: include/nerfacc_hip.h); counts and run records are complete —
        // offsets by their own kernel, emit pass below
        stamp = next_stamp();
        h[3] = 0;
        check_rc(nfa_traverse_offsets_stamped(&a, ws.data_ptr(), stamp, s));
        wait_stamp(h + 3, stamp, s);
        emitted = false;
    }
    const int64_t n = h[1], n_overflow = h[2];
    // (totals that cannot be — seen once in ~60 runs of eight processes sharing one GPU, when the count launch lost one XCD's share of
    //  its workgroups' stores, profiles/r06_oversubscription.md: an error the caller can see instead of outputs sized by garbage)
    TORCH_CHECK(n >= 0 && n_overflow >= 0 && n_overflow <= R && h[0] >= n,
                "nerfacc_amd: sample_occgrid read back inconsistent totals (edges ", h[0], ", samples ", n, ", overflow rays ", n_overflow, " of ", R,
                " rays): the count pass's outputs are corrupt");
    last_spr[dev] = R > 0 ? (double)n / (double)R : 0.0;
    if (emitted && n <= cap) {
        if (n_overflow > 0) check_rc(nfa_traverse_fill(&a, 1, 0, ws.data_ptr(), 0, n_overflow, s));     // the rays the count pass flagged
        ray_indices = ray_indices.narrow(0, 0, n);
        ts.n = n;
        if (cap > (1 << 20) && n < cap / 4) {
            // a guess far too large: the caller would keep the whole over-sized storage alive through these views
            // (and torch.save would write it) — hand out right-sized copies instead
            ray_indices = ray_indices.clone();
            Rows exact(2, n, f32);
            exact.row(0).copy_(ts.row(0));
            exact.row(1).copy_(ts.row(1));
            ts = exact;
        }
    } else {
        ray_indices = at::empty({n}, i64);
        ts = Rows(2, n, f32);
        a.sm_ray_indices = ptr<int64_t>(ray_indices);
        a.t_starts = ts.p(0);
        a.t_ends = ts.p(1);
        if (n > 0) {
            Timed t("traverse_fill", s);
            check_rc(nfa_traverse_fill(&a, 1, 0, ws.data_ptr(), n, n_overflow, s));
        }
    }
    if (plain) {
        // the next slice of the caller's loop, if this call continued one (its rays start where the previous call's ended) and both
        // ray arrays have rows left behind this slice
        const float *o_end = ptr<float>(rays_o) + 3 * R, *d_end = ptr<float>(rays_d) + 3 * R;
        const bool continued = pf.expect_o == rays_o.data_ptr();
        pf.expect_o = o_end;
        auto rows_left = [&](const Tensor &t) {
            const int64_t used = (t.storage_offset() + 3 * R) * 4;
            return ((int64_t)t.storage().nbytes() - used) / 12;
        };
        const int64_t Rn = std::min<int64_t>(R, std::min(rows_left(rays_o), rows_left(rays_d)));
        nfa_traverse_args a2 = a;
        a2.n_rays = Rn;
        a2.rays_o = o_end;
        a2.rays_d = d_end;
        a2.sm_ray_indices = nullptr; a2.t_starts = nullptr; a2.t_ends = nullptr; a2.terminate_planes = nullptr;
        if (Rn > 0) a2.workspace_bytes = nfa_traverse_workspace_bytes_for(&a2);
        // (a slice whose workspace is beyond what a thread retains gets a per-call allocation: a guess would pin it between calls and
        //  behind the loop's last slice — exactly what the cap is there to prevent: no count pass ahead for such slices)
        if (continued && Rn > 0 && chunk_prefetch_allowed() && a2.workspace_bytes <= kWorkspaceKeep) {
            pf.packed = at::empty({2, Rn}, i64);
            a2.sm_starts = ptr<int64_t>(pf.packed);
            a2.sm_cnts = ptr<int64_t>(pf.packed) + Rn;
            int64_t *h2 = host_ints(rays_o.device().index(), s, 1);
            a2.totals = h2;
            Tensor ws2 = traverse_workspace(rays_o, s, a2.workspace_bytes);      // (the same slab: this call's kernels are enqueued before)
            pf.stamp = next_stamp();
            h2[3] = 0;
            // count + offsets of the next slice: one launch where the fused form exists (capacity 0: nothing is expanded), else two
            check_rc(nfa_traverse_sample(&a2, ws2.data_ptr(), 0, pf.stamp, sync_block(rays_o, s), nullptr, s));
            pf.o_ptr = o_end; pf.d_ptr = d_end; pf.R = Rn;
            pf.o_ver = rays_o._version(); pf.d_ver = rays_d._version();
            pf.bin_impl = (const void *)binaries.unsafeGetTensorImpl(); pf.bin_ver = binaries._version();
            pf.aabbs_ptr = aabbs.data_ptr(); pf.aabbs_ver = aabbs._version();
            pf.step = step_size; pf.cone = cone_angle; pf.near_plane = near_plane; pf.far_plane = far_plane;
            pf.ws_bytes = a2.workspace_bytes;
            pf.ws_keep = ws2;
            pf.o_st = rays_o.storage().getWeakStorageImpl();
            pf.d_st = rays_d.storage().getWeakStorageImpl();
            pf.aabbs_st = aabbs.storage().getWeakStorageImpl();
            pf.bin_ref = c10::weak_intrusive_ptr<c10::TensorImpl>(binaries.getIntrusivePtr());
            pf.valid = true;
        }
    } else {
        pf.expect_o = nullptr;
    }
    if (with_terminate_planes) return py::make_tuple(ray_indices, ts.row(0), ts.row(1), packed.t(), term);
    return py::make_tuple(ray_indices, ts.row(0), ts.row(1), packed.t());
}

// ---------------------------------------------------------------------------------------------------
// scans (nerfacc.cpp:17-60)
// ---------------------------------------------------------------------------------------------------
Tensor scan_packed(const Tensor &chunk_starts, const Tensor &chunk_cnts, const Tensor &inputs, int op, bool inclusive, bool reverse,
                   bool normalize) {
    check_input(chunk_starts, "chunk_starts", at::kLong);
    check_input(chunk_cnts, "chunk_cnts", at::kLong);
    check_input(inputs, "inputs", at::kFloat);
    TORCH_CHECK(chunk_starts.dim() == 1 && chunk_cnts.dim() == 1 && inputs.dim() == 1, "chunk_starts, chunk_cnts and inputs must be 1-D");
    TORCH_CHECK(chunk_starts.size(0) == chunk_cnts.size(0), "chunk_starts and chunk_cnts differ in length");
    Tensor out = at::empty_like(inputs);
    Guard g(device_of(inputs));
    check_rc(nfa_scan_packed(ptr<int64_t>(chunk_starts), ptr<int64_t>(chunk_cnts), chunk_cnts.size(0), ptr<float>(inputs), ptr<float>(out),
                             inputs.size(0), op, inclusive, reverse, normalize, stream_of(inputs)));
    return out;
}

Tensor scan_keyed(const Tensor &indices, const Tensor &inputs, int op, bool inclusive, bool reverse) {
    check_input(indices, "indices", at::kLong);
    check_input(inputs, "inputs", at::kFloat);
    TORCH_CHECK(indices.dim() == 1 && inputs.dim() == 1 && indices.size(0) == inputs.size(0), "indices and inputs must be 1-D with the same length");
    TORCH_CHECK(indices.device() == inputs.device(), "indices and inputs must live on the same device");
    Tensor out = at::empty_like(inputs);
    Guard g(device_of(inputs));
    check_rc(nfa_scan_keyed(ptr<int64_t>(indices), ptr<float>(inputs), ptr<float>(out), inputs.size(0), op, inclusive, reverse, stream_of(inputs)));
    return out;
}

Tensor prod_bwd(const OptTensor &indices, const OptTensor &chunk_starts, const OptTensor &chunk_cnts, const Tensor &inputs,
                const Tensor &outputs, const Tensor &grad_outputs, bool inclusive) {
    check_input(inputs, "inputs", at::kFloat);
    const int64_t n = inputs.numel();
    check_len(indices, "indices", at::kLong, n, inputs);
    if (chunk_starts) check_input(*chunk_starts, "chunk_starts", at::kLong);
    if (chunk_cnts) check_input(*chunk_cnts, "chunk_cnts", at::kLong);
    TORCH_CHECK(chunk_starts.has_value() == chunk_cnts.has_value() && (!chunk_starts || chunk_starts->numel() == chunk_cnts->numel()),
                "chunk_starts and chunk_cnts must be given together with the same length");
    check_len(outputs, "outputs", at::kFloat, n, inputs);
    check_len(grad_outputs, "grad_outputs", at::kFloat, n, inputs);
    Tensor gin = at::empty_like(grad_outputs);
    Guard g(device_of(inputs));
    check_rc(nfa_prod_backward(ptr<int64_t>(indices), ptr<int64_t>(chunk_starts), ptr<int64_t>(chunk_cnts), chunk_cnts ? chunk_cnts->size(0) : 0,
                               ptr<float>(inputs), ptr<float>(outputs), ptr<float>(grad_outputs), ptr<float>(gin), inputs.size(0), inclusive,
                               stream_of(inputs)));
    return gin;
}

// ---------------------------------------------------------------------------------------------------
// pdf (nerfacc.cpp:100-117)
// ---------------------------------------------------------------------------------------------------
std::vector<RaySegmentsSpec> importance_sampling(const RaySegmentsSpec &seg, const Tensor &cdfs, const py::object &n_intervals, bool stratified) {
    seg.check();
    check_input(cdfs, "cdfs", at::kFloat);
    TORCH_CHECK(cdfs.numel() == seg.vals->numel(), "cdfs and ray_segments.vals must have the same number of elements");
    if (!py::isinstance<py::int_>(n_intervals)) {
        // per-ray counts (nerfacc.cpp:100-105): flattened outputs sized from the counts — one host read of their sum, as the
        // reference's memalloc_data_from_chunk does (data_spec.hpp:86-97)
        Tensor cnts = n_intervals.cast<Tensor>();
        TORCH_CHECK(cnts.is_cuda() && cnts.device() == cdfs.device(), "n_intervals_per_ray must live on the device of cdfs");
        nfa_ray_segments view = seg.view();
        TORCH_CHECK(at::isIntegralType(cnts.scalar_type(), /*includeBool=*/false), "n_intervals_per_ray must be an integer tensor, got ",
                    cnts.scalar_type(), " (a float count would be truncated silently)");
        cnts = cnts.to(at::kLong).reshape({-1}).contiguous();
        TORCH_CHECK(cnts.numel() == view.n_rays, "n_intervals_per_ray must hold one count per ray (", view.n_rays, "), got ", cnts.numel());
        RaySegmentsSpec samples, intervals;
        samples.chunk_cnts = cnts;
        Tensor cs = at::cumsum(cnts, 0);
        samples.chunk_starts = cs - cnts;
        intervals.chunk_cnts = (cnts + 1) * (cnts > 0).to(at::kLong);
        Tensor ics = at::cumsum(*intervals.chunk_cnts, 0);
        intervals.chunk_starts = ics - *intervals.chunk_cnts;
        // ONE read-back: the smallest count and the two totals together (three blocking .item() calls before)
        int64_t n_s = 0, n_e = 0;
        if (cnts.numel()) {
            const Tensor three = at::stack({cnts.min(), cs[-1], ics[-1]}).cpu();
            const int64_t *h3 = three.data_ptr<int64_t>();
            TORCH_CHECK(h3[0] >= 0, "n_intervals_per_ray must not be negative");
            n_s = h3[1];
            n_e = h3[2];
        }
        const auto i64 = opts(cdfs, at::kLong), b8 = opts(cdfs, at::kBool);
        samples.vals = at::empty({n_s}, cdfs.options());
        samples.ray_indices = at::empty({n_s}, i64);
        intervals.vals = at::empty({n_e}, cdfs.options());
        intervals.ray_indices = at::empty({n_e}, i64);
        intervals.is_left = at::empty({n_e}, b8);
        intervals.is_right = at::empty({n_e}, b8);
        Tensor jitter;
        if (stratified) jitter = at::rand({view.n_rays}, cdfs.options());
        Guard g(device_of(cdfs));
        check_rc(nfa_importance_sampling_ragged(&view, ptr<float>(cdfs), ptr<int64_t>(samples.chunk_starts), ptr<int64_t>(cnts),
                                                ptr<int64_t>(intervals.chunk_starts), n_s, ptr<float>(jitter), ptr<float>(samples.vals),
                                                ptr<int64_t>(samples.ray_indices), ptr<float>(intervals.vals), ptr<int64_t>(intervals.ray_indices),
                                                (uint8_t *)intervals.is_left->data_ptr(), (uint8_t *)intervals.is_right->data_ptr(), stream_of(cdfs)));
        return {intervals, samples};
    }
    const int64_t n = n_intervals.cast<int64_t>();
    nfa_ray_segments view = seg.view();
    std::vector<int64_t> lead;
    if (seg.vals->dim() > 1) lead.assign(seg.vals->sizes().begin(), seg.vals->sizes().end() - 1);
    else lead = {view.n_rays};
    auto with_last = [&](int64_t k) { auto v = lead; v.push_back(k); return v; };
    RaySegmentsSpec samples, intervals;
    samples.vals = at::empty(with_last(n), cdfs.options());
    intervals.vals = at::empty(with_last(n + 1), cdfs.options());
    Tensor jitter;
    // one uniform per ray from torch's generator (the reference draws it with Philox inside the kernel, pdf.cu:138-144)
    if (stratified) jitter = at::rand({view.n_rays}, cdfs.options());
    Guard g(device_of(cdfs));
    check_rc(nfa_importance_sampling(&view, ptr<float>(cdfs), n, ptr<float>(jitter), ptr<float>(intervals.vals), ptr<float>(samples.vals),
                                     stream_of(cdfs)));
    return {intervals, samples};
}

std::vector<Tensor> searchsorted(const RaySegmentsSpec &query, const RaySegmentsSpec &key) {
    query.check();
    key.check();
    Tensor l = at::empty(query.vals->sizes(), opts(*query.vals, at::kLong)), r = at::empty_like(l);
    nfa_ray_segments q = query.view(), k = key.view();
    Guard g(device_of(*query.vals));
    check_rc(nfa_searchsorted(&q, &k, ptr<int64_t>(l), ptr<int64_t>(r), stream_of(*query.vals)));
    return {l, r};
}

Tensor transform_stot(const Tensor &s_vals, double t_min, double t_max, bool lindisp) {
    check_input(s_vals, "s_vals", at::kFloat);
    Tensor t = at::empty_like(s_vals);
    Guard g(device_of(s_vals));
    // (the reference's scalars are Python floats: 1 / t is formed in double inside the library call)
    check_rc(nfa_transform_stot(ptr<float>(s_vals), s_vals.numel(), t_min, t_max, lindisp ? 1 : 0, ptr<float>(t), stream_of(s_vals)));
    return t;
}

// (cdfs [R, S + 1], trans [R, S] or undefined)
std::vector<Tensor> edge_cdfs_fwd(const Tensor &t_edges, const Tensor &sigmas, bool want_trans) {
    check_input(t_edges, "t_edges", at::kFloat);
    check_input(sigmas, "sigmas", at::kFloat);
    TORCH_CHECK(sigmas.dim() == 2 && t_edges.dim() == 2 && t_edges.size(0) == sigmas.size(0) && t_edges.size(1) == sigmas.size(1) + 1 &&
                sigmas.size(1) >= 1 && t_edges.device() == sigmas.device(), "edge_cdfs: t_edges must be [n_rays, n + 1] and sigmas [n_rays, n]");
    Tensor cdfs = at::empty_like(t_edges), trans;
    if (want_trans) trans = at::empty_like(sigmas);
    Guard g(device_of(sigmas));
    check_rc(nfa_edge_cdfs_fwd(ptr<float>(t_edges), ptr<float>(sigmas), sigmas.size(0), sigmas.size(1), ptr<float>(cdfs), ptr<float>(trans),
                               stream_of(sigmas)));
    return {cdfs, trans};
}

Tensor edge_cdfs_bwd(const Tensor &t_edges, const Tensor &trans, const Tensor &g_cdfs) {
    check_input(t_edges, "t_edges", at::kFloat);
    check_input(trans, "trans", at::kFloat);
    check_input(g_cdfs, "g_cdfs", at::kFloat);
    TORCH_CHECK(trans.dim() == 2 && t_edges.dim() == 2 && t_edges.size(0) == trans.size(0) && t_edges.size(1) == trans.size(1) + 1 &&
                g_cdfs.sizes() == t_edges.sizes(), "edge_cdfs_bwd: shape mismatch");
    Tensor g_sig = at::empty_like(trans);
    Guard g(device_of(trans));
    check_rc(nfa_edge_cdfs_bwd(ptr<float>(t_edges), ptr<float>(trans), ptr<float>(g_cdfs), trans.size(0), trans.size(1), ptr<float>(g_sig),
                               stream_of(trans)));
    return g_sig;
}

// (loss [R, Nq], ids_left, ids_right (int32), coef) — the last three undefined unless want_grad
std::vector<Tensor> pdf_loss_fwd(const Tensor &q, const Tensor &cq, const Tensor &k, const Tensor &ck, double eps, bool want_grad) {
    check_input(q, "query vals", at::kFloat);
    check_input(cq, "cdfs_query", at::kFloat);
    check_input(k, "key vals", at::kFloat);
    check_input(ck, "cdfs_key", at::kFloat);
    TORCH_CHECK(q.dim() == 2 && k.dim() == 2 && cq.sizes() == q.sizes() && ck.sizes() == k.sizes() && q.size(0) == k.size(0) && q.size(1) >= 2 &&
                k.size(1) >= 2, "pdf_loss: batched [n_rays, n + 1] edges and cdfs expected");
    const int64_t R = q.size(0), nq = q.size(1) - 1, nk = k.size(1) - 1;
    Tensor loss = at::empty({R, nq}, q.options()), il, ir, coef;
    if (want_grad) { il = at::empty({R, nq}, opts(q, at::kInt)); ir = at::empty_like(il); coef = at::empty_like(loss); }
    Guard g(device_of(q));
    check_rc(nfa_pdf_loss_fwd(ptr<float>(q), ptr<float>(cq), ptr<float>(k), ptr<float>(ck), R, nq, nk, (float)eps, ptr<float>(loss),
                              ptr<int32_t>(il), ptr<int32_t>(ir), ptr<float>(coef), stream_of(q)));
    return {loss, il, ir, coef};
}

Tensor pdf_loss_bwd(const Tensor &g_loss, const Tensor &il, const Tensor &ir, const Tensor &coef, int64_t n_key) {
    check_input(g_loss, "g_loss", at::kFloat);
    check_input(il, "ids_left", at::kInt);
    check_input(ir, "ids_right", at::kInt);
    check_input(coef, "coef", at::kFloat);
    TORCH_CHECK(g_loss.dim() == 2 && il.sizes() == g_loss.sizes() && ir.sizes() == g_loss.sizes() && coef.sizes() == g_loss.sizes() && n_key >= 1,
                "pdf_loss_bwd: shape mismatch");
    Tensor g_ck = at::empty({g_loss.size(0), n_key + 1}, g_loss.options());
    Guard g(device_of(g_loss));
    check_rc(nfa_pdf_loss_bwd(ptr<float>(g_loss), ptr<int32_t>(il), ptr<int32_t>(ir), ptr<float>(coef), g_loss.size(0), g_loss.size(1), n_key,
                              ptr<float>(g_ck), stream_of(g_loss)));
    return g_ck;
}

// ---------------------------------------------------------------------------------------------------
// pack / rendering (fused entry points: chains of ATen ops in the reference)
// ---------------------------------------------------------------------------------------------------
Tensor pack_info(const Tensor &ray_indices, int64_t n_rays) {
    check_input(ray_indices, "ray_indices", at::kLong);
    TORCH_CHECK(n_rays >= 0, "n_rays must be >= 0");
    Tensor out = at::empty({n_rays, 2}, ray_indices.options());
    Guard g(device_of(ray_indices));
    check_rc(nfa_pack_info(ptr<int64_t>(ray_indices), ray_indices.size(0), n_rays, ptr<int64_t>(out), stream_of(ray_indices)));
    return out;
}

Tensor unpack_info(const Tensor &chunk_starts, const Tensor &chunk_cnts, int64_t n) {
    check_input(chunk_starts, "chunk_starts", at::kLong);
    check_input(chunk_cnts, "chunk_cnts", at::kLong);
    TORCH_CHECK(chunk_starts.numel() == chunk_cnts.numel() && n >= 0, "chunk_starts and chunk_cnts differ in length (or n < 0)");
    Tensor out = at::empty({n}, chunk_starts.options());
    Guard g(device_of(chunk_starts));
    check_rc(nfa_unpack_info(ptr<int64_t>(chunk_starts), ptr<int64_t>(chunk_cnts), chunk_cnts.size(0), ptr<int64_t>(out), n, stream_of(chunk_starts)));
    return out;
}

py::tuple render_weight_from_density_fwd(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas,
                                         const OptTensor &prefix_trans) {
    check_input(sigmas, "sigmas", at::kFloat);
    const int64_t n = sigmas.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, sigmas);
    check_len(t_starts, "t_starts", at::kFloat, n, sigmas);
    check_len(t_ends, "t_ends", at::kFloat, n, sigmas);
    check_len(prefix_trans, "prefix_trans", at::kFloat, n, sigmas);
    Rows out(3, n, sigmas.options());
    Guard g(device_of(sigmas));
    check_rc(nfa_render_weight_from_density_fwd(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(sigmas),
                                                ptr<float>(prefix_trans), n, out.p(0), out.p(1), out.p(2), stream_of(sigmas)));
    return py::make_tuple(out.row(0), out.row(1), out.row(2));
}

Tensor render_weight_from_density_bwd(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas,
                                      const Tensor &trans, const Tensor &alphas, const OptTensor &g_w, const OptTensor &g_T, const OptTensor &g_a) {
    check_input(sigmas, "sigmas", at::kFloat);
    const int64_t n = sigmas.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, sigmas);
    check_len(t_starts, "t_starts", at::kFloat, n, sigmas);
    check_len(t_ends, "t_ends", at::kFloat, n, sigmas);
    check_len(trans, "trans", at::kFloat, n, sigmas);
    check_len(alphas, "alphas", at::kFloat, n, sigmas);
    for (auto *t : {&g_w, &g_T, &g_a}) check_len(*t, "grad", at::kFloat, n, sigmas);
    Tensor gs = at::empty_like(sigmas);
    Guard g(device_of(sigmas));
    check_rc(nfa_render_weight_from_density_bwd(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(sigmas),
                                                ptr<float>(trans), ptr<float>(alphas), ptr<float>(g_w), ptr<float>(g_T), ptr<float>(g_a),
                                                sigmas.size(0), ptr<float>(gs), stream_of(sigmas)));
    return gs;
}

py::object sample_positions(const Tensor &rays_o, const Tensor &rays_d, const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends,
                            bool with_dirs) {
    check_input(rays_o, "rays_o", at::kFloat);
    check_input(rays_d, "rays_d", at::kFloat);
    check_input(ray_indices, "ray_indices", at::kLong);
    check_input(t_starts, "t_starts", at::kFloat);
    check_input(t_ends, "t_ends", at::kFloat);
    const int64_t n = ray_indices.size(0);
    TORCH_CHECK(t_starts.size(0) == n && t_ends.size(0) == n && rays_o.sizes() == rays_d.sizes() && rays_o.dim() == 2 && rays_o.size(1) == 3,
                "sample_positions: rays [R,3] x2 and ray_indices / t_starts / t_ends [N] expected");
    Tensor pos = at::empty({n, 3}, rays_o.options()), dirs;
    if (with_dirs) dirs = at::empty({n, 3}, rays_o.options());
    Guard g(device_of(rays_o));
    check_rc(nfa_sample_positions(ptr<float>(rays_o), ptr<float>(rays_d), rays_o.size(0), ptr<int64_t>(ray_indices), ptr<float>(t_starts),
                                  ptr<float>(t_ends), n, ptr<float>(pos), ptr<float>(dirs), stream_of(rays_o)));
    if (with_dirs) return py::make_tuple(pos, dirs);
    return py::cast(pos);
}

// (ray_indices', t_starts', t_ends', mask or None); ONE host sync (the count)
py::tuple visibility_compact(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &dens, bool from_alpha,
                             double early_stop_eps, double alpha_thre, bool want_mask) {
    check_input(dens, "sigmas/alphas", at::kFloat);
    const int64_t n = dens.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, dens);
    check_len(t_starts, "t_starts", at::kFloat, n, dens);
    check_len(t_ends, "t_ends", at::kFloat, n, dens);
    Tensor o_idx = at::empty({n}, ray_indices.options());
    Rows o_t(2, n, dens.options());
    Tensor mask;
    if (want_mask) mask = at::empty({n}, opts(dens, at::kBool));
    Tensor ws = at::empty({std::max<int64_t>(nfa_visibility_workspace_bytes(n), 16)}, opts(dens, at::kByte));
    Guard g(device_of(dens));
    hipStream_t s = stream_of(dens);
    int64_t *h = host_ints(dens.device().index(), s);
    const int64_t stamp = next_stamp();
    {
        Timed t("visibility", s);
        h[1] = 0;
        // (one launch at the training size: mask pass, look-back over its workgroups and compaction — include/nerfacc_hip.h)
        check_rc(nfa_visibility_compact_sync(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(dens), from_alpha,
                                             n, (float)early_stop_eps, (float)alpha_thre, ptr<int64_t>(o_idx), o_t.p(0), o_t.p(1),
                                             ptr<uint8_t>(mask), h, stamp, ws.data_ptr(), n > 0 ? sync_block(dens, s) : nullptr, s));
    }
    if (n > 0) wait_stamp(h + 1, stamp, s);
    else wait_stream(s);
    if (n > 0 && h[0] < 0) {
        // the single launch's look-back gave up (a bounded wait): the compaction kernel over what it left in the workspace
        const int64_t stamp2 = next_stamp();
        h[1] = 0;
        check_rc(nfa_visibility_compact_resume(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(dens), from_alpha,
                                               n, (float)early_stop_eps, (float)alpha_thre, ptr<int64_t>(o_idx), o_t.p(0), o_t.p(1),
                                               ptr<uint8_t>(mask), h, stamp2, ws.data_ptr(), s));
        wait_stamp(h + 1, stamp2, s);
    }
    const int64_t k = n > 0 ? h[0] : 0;
    py::object m = want_mask ? py::cast(mask) : py::none();
    return py::make_tuple(o_idx.narrow(0, 0, k), o_t.row(0).narrow(0, 0, k), o_t.row(1).narrow(0, 0, k), m);
}

Tensor accumulate_along_rays(const Tensor &ray_indices, const Tensor &weights, const OptTensor &values, int64_t n_rays, const OptTensor &outputs) {
    check_input(weights, "weights", at::kFloat);
    const int64_t n = weights.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, weights);
    int64_t D = 1;
    if (values) {
        TORCH_CHECK(values->dim() >= 1, "values must be [n_samples, D]");
        D = values->size(-1);
        check_len(*values, "values", at::kFloat, n, weights, D);
    }
    Tensor out;
    if (outputs) {
        check_input(*outputs, "outputs", at::kFloat);
        TORCH_CHECK(outputs->dim() == 2 && outputs->size(1) == D && outputs->device() == weights.device(), "outputs must be [n_rays, ", D, "] on the inputs' device");
        out = *outputs;
    } else {
        TORCH_CHECK(n_rays >= 0, "n_rays must be >= 0");
        out = at::zeros({n_rays, D}, weights.options());
    }
    Guard g(device_of(weights));
    check_rc(nfa_accumulate_along_rays(ptr<int64_t>(ray_indices), ptr<float>(weights), ptr<float>(values), weights.size(0), (int32_t)D,
                                       out.size(0), ptr<float>(out), stream_of(weights)));
    return out;
}

py::tuple accumulate_along_rays_bwd(const Tensor &ray_indices, const Tensor &weights, const OptTensor &values, const Tensor &g_out, bool need_w,
                                    bool need_v) {
    check_input(g_out, "g_outputs", at::kFloat);
    check_input(weights, "weights", at::kFloat);
    TORCH_CHECK(g_out.dim() == 2, "g_outputs must be [n_rays, D]");
    const int64_t D = g_out.size(-1), n = weights.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, weights);
    check_len(values, "values", at::kFloat, n, weights, D);
    TORCH_CHECK(values.has_value() || D == 1, "g_outputs must be [n_rays, 1] when values is None");
    TORCH_CHECK(g_out.device() == weights.device(), "g_outputs must live on the inputs' device");
    Tensor g_w, g_v;
    if (need_w) g_w = at::empty_like(weights);
    if (need_v && values) g_v = at::empty_like(*values);
    Guard g(device_of(weights));
    check_rc(nfa_accumulate_along_rays_bwd(ptr<int64_t>(ray_indices), ptr<float>(weights), ptr<float>(values), ptr<float>(g_out), weights.size(0),
                                           (int32_t)D, g_out.size(0), ptr<float>(g_w), ptr<float>(g_v), stream_of(weights)));
    return py::make_tuple(g_w.defined() ? py::cast(g_w) : py::none(), g_v.defined() ? py::cast(g_v) : py::none());
}

std::vector<Tensor> rendering_fwd_core(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas,
                                       const Tensor &rgbs, int64_t n_rays, const OptTensor &bkgd, bool expected_depths) {
    check_input(sigmas, "sigmas", at::kFloat);
    const int64_t n = sigmas.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, sigmas);
    check_len(t_starts, "t_starts", at::kFloat, n, sigmas);
    check_len(t_ends, "t_ends", at::kFloat, n, sigmas);
    check_len(rgbs, "rgbs", at::kFloat, n, sigmas, 3);
    check_len(bkgd, "render_bkgd", at::kFloat, 1, sigmas, 3);
    TORCH_CHECK(n_rays >= 0, "n_rays must be >= 0");
    Rows per(3, n, sigmas.options());
    Tensor colors = at::empty({n_rays, 3}, sigmas.options());
    Tensor od = at::empty({2, n_rays, 1}, sigmas.options());
    Guard g(device_of(sigmas));
    hipStream_t s = stream_of(sigmas);
    {
        Timed t("rendering_fwd", s);
        check_rc(nfa_rendering_fwd(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(sigmas), ptr<float>(rgbs), n,
                                   n_rays, ptr<float>(bkgd), expected_depths, per.p(0), per.p(1), per.p(2),
                                   ptr<float>(colors), ptr<float>(od), ptr<float>(od) + n_rays, s));
    }
    return {colors, od[0], od[1], per.row(0), per.row(1), per.row(2)};
}
py::tuple rendering_fwd(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas, const Tensor &rgbs,
                        int64_t n_rays, const OptTensor &bkgd, bool expected_depths) {
    const auto o = rendering_fwd_core(ray_indices, t_starts, t_ends, sigmas, rgbs, n_rays, bkgd, expected_depths);
    return py::make_tuple(o[0], o[1], o[2], o[3], o[4], o[5]);
}

std::pair<Tensor, Tensor> rendering_bwd_core(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas,
                                             const Tensor &rgbs, const Tensor &weights, const Tensor &trans, const Tensor &alphas,
                                             const Tensor &opacities, const Tensor &depths, int64_t n_rays, const OptTensor &bkgd,
                                             bool expected_depths, const OptTensor &g_colors, const OptTensor &g_opac, const OptTensor &g_depth,
                                             const OptTensor &g_w, const OptTensor &g_T, const OptTensor &g_a, bool need_sigma, bool need_rgb) {
    check_input(sigmas, "sigmas", at::kFloat);
    const int64_t n = sigmas.numel();
    check_len(ray_indices, "ray_indices", at::kLong, n, sigmas);
    check_len(t_starts, "t_starts", at::kFloat, n, sigmas);
    check_len(t_ends, "t_ends", at::kFloat, n, sigmas);
    check_len(rgbs, "rgbs", at::kFloat, n, sigmas, 3);
    check_len(weights, "weights", at::kFloat, n, sigmas);
    check_len(trans, "trans", at::kFloat, n, sigmas);
    check_len(alphas, "alphas", at::kFloat, n, sigmas);
    check_len(opacities, "opacities", at::kFloat, n_rays, sigmas);
    check_len(depths, "depths", at::kFloat, n_rays, sigmas);
    check_len(bkgd, "render_bkgd", at::kFloat, 1, sigmas, 3);
    check_len(g_colors, "g_colors", at::kFloat, n_rays, sigmas, 3);
    check_len(g_opac, "g_opacities", at::kFloat, n_rays, sigmas);
    check_len(g_depth, "g_depths", at::kFloat, n_rays, sigmas);
    for (auto *t : {&g_w, &g_T, &g_a}) check_len(*t, "grad", at::kFloat, n, sigmas);
    Tensor g_sig, g_rgb;
    if (need_sigma) g_sig = at::empty_like(sigmas);
    if (need_rgb) g_rgb = at::empty_like(rgbs);
    Guard g(device_of(sigmas));
    hipStream_t s = stream_of(sigmas);
    {
        Timed t("rendering_bwd", s);
        check_rc(nfa_rendering_bwd(ptr<int64_t>(ray_indices), ptr<float>(t_starts), ptr<float>(t_ends), ptr<float>(sigmas), ptr<float>(rgbs),
                                   ptr<float>(weights), ptr<float>(trans), ptr<float>(alphas), ptr<float>(opacities), ptr<float>(depths),
                                   sigmas.size(0), n_rays, ptr<float>(bkgd), expected_depths, ptr<float>(g_colors), ptr<float>(g_opac),
                                   ptr<float>(g_depth), ptr<float>(g_w), ptr<float>(g_T), ptr<float>(g_a), ptr<float>(g_sig), ptr<float>(g_rgb), s));
    }
    return {g_sig, g_rgb};
}
py::tuple rendering_bwd(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas, const Tensor &rgbs,
                        const Tensor &weights, const Tensor &trans, const Tensor &alphas, const Tensor &opacities, const Tensor &depths,
                        int64_t n_rays, const OptTensor &bkgd, bool expected_depths, const OptTensor &g_colors, const OptTensor &g_opac,
                        const OptTensor &g_depth, const OptTensor &g_w, const OptTensor &g_T, const OptTensor &g_a, bool need_sigma, bool need_rgb) {
    const auto r = rendering_bwd_core(ray_indices, t_starts, t_ends, sigmas, rgbs, weights, trans, alphas, opacities, depths, n_rays, bkgd,
                                      expected_depths, g_colors, g_opac, g_depth, g_w, g_T, g_a, need_sigma, need_rgb);
    return py::make_tuple(r.first.defined() ? py::cast(r.first) : py::none(), r.second.defined() ? py::cast(r.second) : py::none());
}

// ---------------------------------------------------------------------------------------------------
// rendering with its autograd node in C++ (volrend.py:104-164 after rgb_sigma_fn): what nerfacc.rendering calls on the
// training path.  The Python twin (nerfacc_amd/volrend.py::_Rendering) costs ~15 us of interpreter per forward and ~30 us
// per backward on a step whose GPU waits for the host there (tools/step_timeline.py).
// ---------------------------------------------------------------------------------------------------
struct RenderingFn : public torch::autograd::Function<RenderingFn> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, Tensor ray_indices, Tensor t_starts, Tensor t_ends,
                                                  Tensor sigmas, Tensor rgbs, int64_t n_rays, OptTensor bkgd, bool expected_depths) {
        ctx->set_materialize_grads(false);      // of six outputs a loss usually touches one: no zero fills for the rest
        ray_indices = ray_indices.contiguous();
        t_starts = t_starts.contiguous();
        t_ends = t_ends.contiguous();
        sigmas = sigmas.contiguous();
        rgbs = rgbs.contiguous();
        OptTensor bk;
        if (bkgd && bkgd->defined()) bk = bkgd->detach().to(at::kFloat).contiguous();
        std::vector<Tensor> o = rendering_fwd_core(ray_indices, t_starts, t_ends, sigmas, rgbs, n_rays, bk, expected_depths);
        ctx->saved_data["n_rays"] = n_rays;
        ctx->saved_data["expected_depths"] = expected_depths;
        ctx->saved_data["has_bkgd"] = bk.has_value();
        std::vector<Tensor> saved = {ray_indices, t_starts, t_ends, sigmas, rgbs, o[3], o[4], o[5], o[1], o[2]};
        if (bk) saved.push_back(*bk);
        ctx->save_for_backward(saved);
        return o;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list g) {
        const auto saved = ctx->get_saved_variables();
        const bool has_bkgd = ctx->saved_data["has_bkgd"].toBool();
        auto opt = [](const Tensor &t) -> OptTensor { return t.defined() ? OptTensor(t.contiguous()) : std::nullopt; };
        const bool need_sigma = ctx->needs_input_grad(3), need_rgb = ctx->needs_input_grad(4);
        Tensor g_sig, g_rgb;
        if (need_sigma || need_rgb) {            // (no Python object anywhere below: the autograd engine's thread does not hold the GIL)
            auto r = rendering_bwd_core(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], saved[8], saved[9],
                                        ctx->saved_data["n_rays"].toInt(), has_bkgd ? OptTensor(saved[10]) : std::nullopt,
                                        ctx->saved_data["expected_depths"].toBool(), opt(g[0]), opt(g[1]), opt(g[2]), opt(g[3]), opt(g[4]),
                                        opt(g[5]), need_sigma, need_rgb);
            g_sig = r.first;
            g_rgb = r.second;
        }
        return {Tensor(), Tensor(), Tensor(), g_sig, g_rgb, Tensor(), Tensor(), Tensor()};
    }
};

py::tuple rendering_autograd(const Tensor &ray_indices, const Tensor &t_starts, const Tensor &t_ends, const Tensor &sigmas, const Tensor &rgbs,
                             int64_t n_rays, const OptTensor &bkgd, bool expected_depths) {
    auto o = RenderingFn::apply(ray_indices, t_starts, t_ends, sigmas, rgbs, n_rays, bkgd, expected_depths);
    return py::make_tuple(o[0], o[1], o[2], o[3], o[4], o[5]);
}

// ---------------------------------------------------------------------------------------------------
// occupancy-grid maintenance (OccGridEstimator._update, occ_grid.py:366-404)
// ---------------------------------------------------------------------------------------------------
Tensor grid_cell_points(const OptTensor &cell_ids, const Tensor &jitter, const std::vector<int64_t> &resolution, const Tensor &aabb) {
    check_input(jitter, "jitter", at::kFloat);
    check_input(aabb, "aabb", at::kFloat);
    const int64_t n = jitter.size(0);
    if (cell_ids) {
        check_input(*cell_ids, "cell_ids", at::kLong);
        TORCH_CHECK(cell_ids->dim() == 1 && cell_ids->size(0) == n, "cell_ids must have shape [n] matching jitter [n, 3]");
    }
    TORCH_CHECK(jitter.dim() == 2 && jitter.size(1) == 3 && aabb.numel() == 6 && resolution.size() == 3, "jitter must be [n, 3] and aabb must hold 6 floats");
    Tensor points = at::empty({n, 3}, jitter.options());
    Guard g(device_of(jitter));
    hipStream_t s = stream_of(jitter);
    Timed t("grid_cell_points", s);
    check_rc(nfa_grid_cell_points(ptr<int64_t>(cell_ids), n, ptr<float>(jitter), (int32_t)resolution[0], (int32_t)resolution[1],
                                  (int32_t)resolution[2], ptr<float>(aabb), ptr<float>(points), s));
    return points;
}

void grid_ema_update(const Tensor &occs_level, const OptTensor &cell_ids, const Tensor &occ_new, double ema_decay) {
    check_input(occs_level, "occs", at::kFloat);
    check_input(occ_new, "occ_new", at::kFloat);
    const int64_t n = occ_new.numel();
    if (cell_ids) {
        check_input(*cell_ids, "cell_ids", at::kLong);
        TORCH_CHECK(cell_ids->numel() == n, "cell_ids and occ_new must have the same number of elements");
    } else {
        TORCH_CHECK(n <= occs_level.numel(), "occ_new has more elements than the level has cells");
    }
    Tensor scratch = at::empty({n}, occs_level.options());
    Guard g(device_of(occs_level));
    hipStream_t s = stream_of(occs_level);
    Timed t("grid_ema_update", s);
    check_rc(nfa_grid_ema_update(ptr<float>(occs_level), ptr<int64_t>(cell_ids), n, ptr<float>(occ_new), (float)ema_decay, ptr<float>(scratch), s));
}

void grid_mark_invisible(const Tensor &occs_level, const OptTensor &cell_ids, const std::vector<int64_t> &resolution, const Tensor &aabb,
                         const Tensor &w2c_R, const Tensor &w2c_T, const Tensor &K, double width, double height, double near_plane) {
    check_input(occs_level, "occs", at::kFloat);
    check_input(aabb, "aabb", at::kFloat);
    check_input(w2c_R, "w2c_R", at::kFloat);
    check_input(w2c_T, "w2c_T", at::kFloat);
    check_input(K, "K", at::kFloat);
    int64_t n = occs_level.numel();
    if (cell_ids) { check_input(*cell_ids, "cell_ids", at::kLong); n = cell_ids->numel(); }
    const int64_t C = w2c_R.size(0);
    TORCH_CHECK(w2c_R.numel() == 9 * C && w2c_T.numel() == 3 * C && (K.numel() == 9 || K.numel() == 9 * C) && resolution.size() == 3,
                "grid_mark_invisible: w2c_R [C,3,3], w2c_T [C,3,1], K [C or 1,3,3] expected");
    Guard g(device_of(occs_level));
    check_rc(nfa_grid_mark_invisible(ptr<float>(occs_level), ptr<int64_t>(cell_ids), n, (int32_t)resolution[0], (int32_t)resolution[1],
                                     (int32_t)resolution[2], ptr<float>(aabb), ptr<float>(w2c_R), ptr<float>(w2c_T), ptr<float>(K), (int32_t)C,
                                     (K.numel() == 9 && C != 1) ? 1 : 0, (float)width, (float)height, (float)near_plane, stream_of(occs_level)));
}

// shape = None: flat bool grid.  shape = (G, rx, ry, rz): the bool grid in that shape AND its bit-packed form, produced by
// the same pass and entered into the brick cache — the traversal that follows does not pack again.
py::tuple grid_threshold(const Tensor &occs, double occ_thre, const std::optional<std::vector<int64_t>> &shape) {
    check_input(occs, "occs", at::kFloat);
    const int64_t n = occs.numel();
    Tensor ws = at::empty({nfa_grid_threshold_workspace_bytes() / 8}, opts(occs, at::kDouble));
    Tensor thre = at::empty({1}, occs.options());
    Guard g(device_of(occs));
    hipStream_t s = stream_of(occs);
    Timed t("grid_threshold", s);
    if (shape) {
        TORCH_CHECK(shape->size() == 4 && (*shape)[0] * (*shape)[1] * (*shape)[2] * (*shape)[3] == n && n > 0,
                    "grid_threshold: shape must be (n_grids, resx, resy, resz) with as many cells as occs");
        const int G = (int)(*shape)[0], rx = (int)(*shape)[1], ry = (int)(*shape)[2], rz = (int)(*shape)[3];
        Tensor binaries = at::empty(*shape, opts(occs, at::kBool));
        Tensor bricks = at::empty({nfa_packed_grid_words(G, rx, ry, rz)}, opts(occs, at::kLong));
        check_rc(nfa_grid_threshold_packed(ptr<float>(occs), G, rx, ry, rz, (float)occ_thre, ws.data_ptr(), ptr<uint8_t>(binaries),
                                           ptr<float>(thre), ptr<uint64_t>(bricks), s));
        std::lock_guard<std::mutex> l(g_brick_mu);
        insert_brick_entry(binaries, bricks, s);
        return py::make_tuple(binaries, thre);
    }
    Tensor binaries = at::empty({n}, opts(occs, at::kBool));
    check_rc(nfa_grid_threshold(ptr<float>(occs), n, (float)occ_thre, ws.data_ptr(), ptr<uint8_t>(binaries), ptr<float>(thre), s));
    return py::make_tuple(binaries, thre);
}

// ---------------------------------------------------------------------------------------------------
// feature operators (dense.hip, conv.hip, selective.hip).  These calls check what would be read out of bounds; the whole operators further
// down, and nerfacc_amd/dense.py and selective.py for the ctypes face, check shapes and dtypes in the caller's terms.
// ---------------------------------------------------------------------------------------------------
inline int32_t dtype_of(const Tensor &t) {
    if (t.scalar_type() == at::kFloat) return NFA_DTYPE_F32;
    if (t.scalar_type() == at::kBFloat16) return NFA_DTYPE_BF16;
    TORCH_CHECK(t.scalar_type() == at::kHalf, "nerfacc_amd: float32, bfloat16 or float16 expected, got ", t.scalar_type());
    return NFA_DTYPE_F16;
}

// a number of features, channels or states for the C ABI, never cut off
inline int32_t i32(int64_t v) {
    TORCH_CHECK(v >= 0 && v < (1ll << 31), "nerfacc_amd: a size of ", v, " is over 2^31 - 1");
    return (int32_t)v;
}

// a [rows, cols] tensor whose rows are contiguous and do not overlap, at any row stride up to 2^25; copied if it is not one
inline Tensor as_rows(const Tensor &t, const char *name, int64_t rows, int64_t cols, const Tensor &like) {
    TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA/HIP tensor (nerfacc_amd has no CPU kernels)");
    TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type(), name, " differs in device or dtype");
    TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols, name, " must have shape [", rows, ", ", cols, "]");
    if ((t.stride(1) == 1 || cols == 1) && ((t.stride(0) >= cols && t.stride(0) <= (1 << 25)) || rows <= 1)) return t;
    return t.contiguous();
}
inline int64_t row_stride(const Tensor &t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

inline Tensor dense_of(const Tensor &t, const char *name, at::ScalarType dtype, int64_t n, const Tensor &like) {
    TORCH_CHECK(t.defined() && t.is_cuda(), name, " must be a CUDA/HIP tensor (nerfacc_amd has no CPU kernels)");
    TORCH_CHECK(t.device() == like.device() && t.scalar_type() == dtype && t.numel() == n, name, " differs in device, dtype or size");
    return t.contiguous();
}
inline OptTensor dense_of(const OptTensor &t, const char *name, at::ScalarType dtype, int64_t n, const Tensor &like) {
    if (!t || !t->defined()) return std::nullopt;
    return dense_of(*t, name, dtype, n, like);
}
inline OptTensor some(const Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// How many nodes of the autograd graphs behind `tensors` were recorded on another stream than the current one of their device.
// A backward pass that is captured into a graph waits for the streams of all of them; one outside the capture (a leaf whose
// accumulator an eager graph keeps alive) ends the capture, and on ROCm the process.
int64_t foreign_nodes(const std::vector<OptTensor> &tensors) {
    std::vector<torch::autograd::Node *> todo;
    std::set<torch::autograd::Node *> seen;
    std::vector<std::shared_ptr<torch::autograd::Node>> held;
    auto add = [&](torch::autograd::Node *n) { if (n && seen.insert(n).second) todo.push_back(n); };
    for (auto &t : tensors) {
        if (!t || !t->defined() || !t->requires_grad()) continue;
        if (auto fn = t->grad_fn()) { held.push_back(fn); add(fn.get()); }
        else if (auto acc = torch::autograd::impl::try_get_grad_accumulator(*t)) { held.push_back(acc); add(acc.get()); }
    }
    int64_t n = 0;
    while (!todo.empty()) {
        auto *node = todo.back();
        todo.pop_back();
        if (auto s = node->stream())
            n += s->device_type() != at::kCPU && s->id() != c10::hip::getCurrentHIPStream(s->device_index()).id();
        for (auto &e : node->next_edges()) add(e.function.get());
    }
    return n;
}

std::tuple<Tensor, OptTensor> linear_fwd(const Tensor &x_, const Tensor &w_, const OptTensor &b_, const OptTensor &r_, int64_t act, bool save) {
    TORCH_CHECK(x_.dim() == 2 && w_.dim() == 2, "linear: 2-D inputs and weight expected");
    const int64_t m = x_.size(0), k = w_.size(1), n = w_.size(0);
    const Tensor x = as_rows(x_, "inputs", m, k, x_), w = dense_of(w_, "weight", x_.scalar_type(), n * k, x_);
    const OptTensor b = dense_of(b_, "bias", x_.scalar_type(), n, x_);
    Tensor r;
    if (r_ && r_->defined()) r = as_rows(*r_, "residual", m, n, x_);
    Guard g(device_of(x_));
    Tensor out = at::empty({m, n}, x_.options()), saved;
    if (const int64_t bytes = save ? nfa_linear_saved_bytes(m, i32(n), dtype_of(x), (int32_t)act, r.defined()) : 0; bytes > 0)
        saved = at::empty({bytes}, opts(x, at::kByte));
    nfa_linear_args a{};
    a.rows = m; a.in_features = i32(k); a.out_features = i32(n);
    a.dtype = dtype_of(x); a.activation = (int32_t)act;
    a.inputs = x.data_ptr(); a.inputs_stride = row_stride(x);
    a.weight = w.data_ptr(); a.bias = ptr<void>(b);
    if (r.defined()) { a.residual = r.data_ptr(); a.residual_stride = row_stride(r); }
    check_rc(nfa_linear_fwd(&a, out.data_ptr(), ptr<void>(saved), stream_of(x)));
    return {out, some(saved)};
}

std::tuple<OptTensor, OptTensor, OptTensor> linear_bwd(const Tensor &g_, const Tensor &x_, const Tensor &w_, const OptTensor &saved_, int64_t act,
                                                       bool need_x, bool need_w, bool need_b) {
    TORCH_CHECK(x_.dim() == 2 && w_.dim() == 2, "linear: 2-D inputs and weight expected");
    const int64_t m = x_.size(0), k = w_.size(1), n = w_.size(0);
    const Tensor x = as_rows(x_, "inputs", m, k, x_), w = dense_of(w_, "weight", x_.scalar_type(), n * k, x_);
    const Tensor gy = as_rows(g_, "grad_outputs", m, n, x_);
    OptTensor saved;                            // what linear_fwd kept, or its outputs
    if (act != NFA_ACT_NONE && m > 0) {
        TORCH_CHECK(saved_ && saved_->defined() && saved_->is_cuda() && saved_->device() == x.device() && saved_->is_contiguous(), "linear: saved is missing");
        const int64_t kept = nfa_linear_saved_bytes(m, i32(n), dtype_of(x), (int32_t)act, 0);
        TORCH_CHECK((int64_t)saved_->nbytes() == (kept ? kept : m * n * (int64_t)x.element_size()), "linear: saved differs in size");
        saved = saved_;
    }
    Guard g(device_of(x_));
    Tensor gx, gw, gb;
    if (need_x) gx = at::empty({m, k}, x_.options());
    if (m == 0) {
        if (need_w) gw = at::zeros({n, k}, x_.options());
        if (need_b) gb = at::zeros({n}, x_.options());
        return {some(gx), some(gw), some(gb)};
    }
    if (need_w) gw = at::empty({n, k}, x_.options());
    if (need_b) gb = at::empty({n}, x_.options());
    nfa_linear_args a{};
    a.rows = m; a.in_features = i32(k); a.out_features = i32(n);
    a.dtype = dtype_of(x); a.activation = (int32_t)act;
    a.inputs = x.data_ptr(); a.inputs_stride = row_stride(x);
    a.weight = w.data_ptr();
    a.grad_outputs = gy.data_ptr(); a.grad_outputs_stride = row_stride(gy);
    Tensor ws;
    if (need_w || need_b) ws = at::empty({nfa_linear_bwd_workspace_bytes(m, i32(k), i32(n), a.dtype, a.activation)}, opts(x, at::kByte));
    check_rc(nfa_linear_bwd(&a, ptr<void>(saved), ptr<void>(gx), ptr<void>(gw), ptr<void>(gb), ptr<void>(ws), stream_of(x)));
    return {some(gx), some(gw), some(gb)};
}

std::tuple<Tensor, Tensor> row_map(const Tensor &info, int64_t rows) {
    check_input(info, "packed_info", at::kLong);
    TORCH_CHECK(info.dim() == 2 && info.size(1) == 2 && rows >= 0, "packed_info must be [n_rays, 2]");
    Guard g(device_of(info));
    Tensor ray = at::empty({rows}, opts(info, at::kInt)), pos = at::empty({rows}, opts(info, at::kInt));
    check_rc(nfa_row_map(ptr<int64_t>(info), info.size(0), rows, ptr<int32_t>(ray), ptr<int32_t>(pos), stream_of(info)));
    return {ray, pos};
}

Tensor ray_order(const Tensor &info, int64_t rows) {
    check_input(info, "packed_info", at::kLong);
    TORCH_CHECK(info.dim() == 2 && info.size(1) == 2 && rows >= 0, "packed_info must be [n_rays, 2]");
    Guard g(device_of(info));
    Tensor order = at::empty({info.size(0)}, opts(info, at::kInt));
    check_rc(nfa_ray_order(ptr<int64_t>(info), info.size(0), rows, ptr<int32_t>(order), stream_of(info)));
    return order;
}

// the sequences of a call: packed (info and its row map) or equal ones
struct Sequences {
    OptTensor info, ray, pos;
    int64_t n_rays;
    Sequences(const OptTensor &info_, const OptTensor &ray_, const OptTensor &pos_, int64_t n, int64_t rows, const Tensor &like) : n_rays(n) {
        info = dense_of(info_, "packed_info", at::kLong, 2 * n, like);
        TORCH_CHECK(n >= 0 && (info || (n > 0 && rows % n == 0)), "nerfacc_amd: rows do not divide into equal sequences");
        if (!info) return;
        ray = dense_of(ray_, "row_ray", at::kInt, rows, like);
        pos = dense_of(pos_, "row_pos", at::kInt, rows, like);
        TORCH_CHECK(ray && pos, "nerfacc_amd: packed sequences need their row map");
    }
    template <class A> void into(A &a) const {
        a.n_rays = n_rays;
        a.packed_info = ptr<int64_t>(info);
        a.row_ray = ptr<int32_t>(ray);
        a.row_pos = ptr<int32_t>(pos);
    }
};

std::tuple<Tensor, OptTensor> causal_conv_fwd(const Tensor &x_, const Tensor &w_, const OptTensor &b_, const OptTensor &init_, const OptTensor &info,
                                              const OptTensor &ray, const OptTensor &pos, int64_t n_rays, int64_t act, bool want_final) {
    TORCH_CHECK(x_.dim() == 2 && w_.dim() == 2, "causal_conv: 2-D inputs and weight expected");
    const int64_t n = x_.size(0), d = x_.size(1), width = w_.size(1);
    const auto dt = x_.scalar_type();
    const Tensor x = as_rows(x_, "inputs", n, d, x_), w = dense_of(w_, "weight", dt, d * width, x_);
    const OptTensor b = dense_of(b_, "bias", dt, d, x_), init = dense_of(init_, "initial_state", dt, n_rays * (width - 1) * d, x_);
    const Sequences seq(info, ray, pos, n_rays, n, x_);
    Guard g(device_of(x_));
    Tensor out = at::empty({n, d}, x_.options()), last;
    if (want_final) last = at::empty({n_rays, width - 1, d}, x_.options());
    if (n_rays == 0) return {out.zero_(), some(last)};
    nfa_causal_conv_args a{};
    seq.into(a);
    a.rows = n; a.channels = i32(d); a.width = i32(width); a.dtype = dtype_of(x); a.activation = (int32_t)act;
    a.inputs = x.data_ptr(); a.inputs_stride = row_stride(x);
    a.weight = w.data_ptr(); a.bias = ptr<void>(b); a.initial_state = ptr<void>(init);
    check_rc(nfa_causal_conv_fwd(&a, out.data_ptr(), ptr<void>(last), stream_of(x)));
    return {out, some(last)};
}

std::tuple<OptTensor, OptTensor, OptTensor, OptTensor> causal_conv_bwd(
    const Tensor &g_, const OptTensor &gfinal_, const Tensor &x_, const Tensor &w_, const OptTensor &b_, const OptTensor &init_, const OptTensor &info,
    const OptTensor &ray, const OptTensor &pos, int64_t n_rays, int64_t act, bool need_x, bool need_w, bool need_b, bool need_init) {
    TORCH_CHECK(x_.dim() == 2 && w_.dim() == 2, "causal_conv: 2-D inputs and weight expected");
    const int64_t n = x_.size(0), d = x_.size(1), width = w_.size(1), ns = n_rays * (width - 1) * d;
    const auto dt = x_.scalar_type();
    const Tensor x = as_rows(x_, "inputs", n, d, x_), w = dense_of(w_, "weight", dt, d * width, x_), gy = as_rows(g_, "grad_outputs", n, d, x_);
    const OptTensor b = dense_of(b_, "bias", dt, d, x_), init = dense_of(init_, "initial_state", dt, ns, x_),
                    gfinal = dense_of(gfinal_, "grad_final_state", dt, ns, x_);
    const Sequences seq(info, ray, pos, n_rays, n, x_);
    Guard g(device_of(x_));
    Tensor gx, gw, gb, gi, ws;
    const bool none = n == 0 || n_rays == 0;
    auto make = [&](at::IntArrayRef shape) { return none ? at::zeros(shape, x_.options()) : at::empty(shape, x_.options()); };
    if (need_x) gx = make({n, d});
    if (need_w) gw = make({d, width});
    if (need_b) gb = make({d});
    if (need_init) gi = make({n_rays, width - 1, d});
    if (n_rays == 0) return {some(gx), some(gw), some(gb), some(gi)};
    nfa_causal_conv_args a{};
    seq.into(a);
    a.rows = n; a.channels = i32(d); a.width = i32(width); a.dtype = dtype_of(x); a.activation = (int32_t)act;
    a.inputs = x.data_ptr(); a.inputs_stride = row_stride(x);
    a.weight = w.data_ptr(); a.bias = ptr<void>(b); a.initial_state = ptr<void>(init);
    a.grad_outputs = gy.data_ptr(); a.grad_outputs_stride = row_stride(gy); a.grad_final_state = ptr<void>(gfinal);
    if (need_w || need_b) ws = at::empty({nfa_causal_conv_bwd_workspace_bytes(n, a.channels, a.width, a.dtype)}, opts(x, at::kByte));
    check_rc(nfa_causal_conv_bwd(&a, ptr<void>(gx), ptr<void>(gw), ptr<void>(gb), ptr<void>(gi), ptr<void>(ws), stream_of(x)));
    return {some(gx), some(gw), some(gb), some(gi)};
}

Tensor causal_conv_step(const Tensor &x_, const Tensor &state_, const Tensor &w_, const OptTensor &b_, int64_t act, const Tensor &to) {
    TORCH_CHECK(x_.dim() == 2 && w_.dim() == 2, "causal_conv_step: 2-D inputs and weight expected");
    const int64_t r = x_.size(0), d = x_.size(1), width = w_.size(1), ns = r * (width - 1) * d;
    const auto dt = x_.scalar_type();
    const Tensor x = as_rows(x_, "inputs", r, d, x_), w = dense_of(w_, "weight", dt, d * width, x_), state = dense_of(state_, "state", dt, ns, x_);
    const OptTensor b = dense_of(b_, "bias", dt, d, x_);
    check_len(to, "out_state", dt, ns, x_);
    Guard g(device_of(x_));
    Tensor out = at::empty({r, d}, x_.options());
    nfa_causal_conv_args a{};
    a.n_rays = r; a.rows = r; a.channels = i32(d); a.width = i32(width); a.dtype = dtype_of(x); a.activation = (int32_t)act;
    a.inputs = x.data_ptr(); a.inputs_stride = row_stride(x);
    a.weight = w.data_ptr(); a.bias = ptr<void>(b);
    check_rc(nfa_causal_conv_step(&a, state.data_ptr(), out.data_ptr(), to.data_ptr(), stream_of(x)));
    return out;
}

// the tensors of a scan, checked and with contiguous rows
struct ScanInputs {
    int64_t n, d, s;
    Tensor u, dt, z, B, C, A;
    OptTensor D, bias, init;
    ScanInputs(const Tensor &u_, const Tensor &dt_, const OptTensor &z_, const Tensor &B_, const Tensor &C_, const Tensor &A_, const OptTensor &D_,
               const OptTensor &bias_, const OptTensor &init_, int64_t n_rays) {
        TORCH_CHECK(u_.dim() == 2 && A_.dim() == 2, "selective_scan: 2-D inputs and A expected");
        n = u_.size(0); d = u_.size(1); s = A_.size(1);
        u = as_rows(u_, "inputs", n, d, u_);
        dt = as_rows(dt_, "delta", n, d, u_);
        if (z_ && z_->defined()) z = as_rows(*z_, "gate", n, d, u_);
        B = as_rows(B_, "B", n, s, u_);
        C = as_rows(C_, "C", n, s, u_);
        A = dense_of(A_, "A", at::kFloat, d * s, u_);
        D = dense_of(D_, "D", at::kFloat, d, u_);
        bias = dense_of(bias_, "delta_bias", at::kFloat, d, u_);
        init = dense_of(init_, "initial_state", at::kFloat, n_rays * d * s, u_);
    }
    nfa_selective_scan_args args(bool softplus) const {
        nfa_selective_scan_args a{};
        a.rows = n; a.channels = i32(d); a.states = i32(s); a.dtype = dtype_of(u); a.delta_softplus = softplus;
        a.inputs = u.data_ptr(); a.inputs_stride = row_stride(u);
        a.delta = dt.data_ptr(); a.delta_stride = row_stride(dt);
        if (z.defined()) { a.gate = z.data_ptr(); a.gate_stride = row_stride(z); }
        a.B = B.data_ptr(); a.B_stride = row_stride(B);
        a.C = C.data_ptr(); a.C_stride = row_stride(C);
        a.A = ptr<float>(A); a.D = ptr<float>(D); a.delta_bias = ptr<float>(bias); a.initial_state = ptr<float>(init);
        return a;
    }
};

std::tuple<Tensor, OptTensor, OptTensor> selective_scan_fwd(
    const Tensor &u, const Tensor &dt, const OptTensor &z, const Tensor &B, const Tensor &C, const Tensor &A, const OptTensor &D, const OptTensor &bias,
    const OptTensor &init, const OptTensor &info, const OptTensor &ray, const OptTensor &pos, const OptTensor &order_, int64_t n_rays, bool softplus,
    bool want_final, bool keep) {
    const ScanInputs in(u, dt, z, B, C, A, D, bias, init, n_rays);
    const Sequences seq(info, ray, pos, n_rays, in.n, u);
    const OptTensor order = dense_of(order_, "ray_order", at::kInt, n_rays, u);
    Guard g(device_of(u));
    Tensor out = at::empty({in.n, in.d}, u.options()), last, kept, ws;
    if (want_final) last = at::empty({n_rays, in.d, in.s}, opts(u, at::kFloat));
    if (n_rays == 0) out.zero_();
    if (keep) kept = at::empty({nfa_selective_scan_checkpoint_bytes(in.n, i32(in.d), i32(in.s))}, opts(u, at::kByte));
    const int64_t bytes = nfa_selective_scan_workspace_bytes(n_rays, in.n, i32(in.d), i32(in.s), 0);
    if (bytes > 0) ws = at::empty({bytes}, opts(u, at::kByte));
    if (n_rays == 0) return {out, some(last), some(kept)};
    auto a = in.args(softplus);
    seq.into(a);
    a.ray_order = ptr<int32_t>(order);
    check_rc(nfa_selective_scan_fwd(&a, out.data_ptr(), ptr<float>(last), ptr<float>(kept), ptr<void>(ws), stream_of(u)));
    return {out, some(last), some(kept)};
}

// (inputs, delta, gate, B, C, A, D, delta_bias, initial_state)
std::vector<OptTensor> selective_scan_bwd(
    const Tensor &g_, const OptTensor &gfinal_, const Tensor &u, const Tensor &dt, const OptTensor &z, const Tensor &B, const Tensor &C, const Tensor &A,
    const OptTensor &D, const OptTensor &bias, const OptTensor &init, const Tensor &kept, const OptTensor &info, const OptTensor &ray, const OptTensor &pos,
    const OptTensor &order_, int64_t n_rays, bool softplus) {
    const ScanInputs in(u, dt, z, B, C, A, D, bias, init, n_rays);
    const Sequences seq(info, ray, pos, n_rays, in.n, u);
    const OptTensor order = dense_of(order_, "ray_order", at::kInt, n_rays, u);
    const Tensor gy = as_rows(g_, "grad_outputs", in.n, in.d, u);
    const OptTensor gfinal = dense_of(gfinal_, "grad_final_state", at::kFloat, n_rays * in.d * in.s, u);
    check_len(kept, "checkpoints", at::kByte, nfa_selective_scan_checkpoint_bytes(in.n, i32(in.d), i32(in.s)), u);
    Guard g(device_of(u));
    const auto f32 = opts(u, at::kFloat);
    const bool none = in.n == 0 || n_rays == 0;
    auto make = [&](at::IntArrayRef shape, at::TensorOptions o) { return none ? at::zeros(shape, o) : at::empty(shape, o); };
    Tensor gu = make({in.n, in.d}, u.options()), gdt = make({in.n, in.d}, u.options()), gz, gB = make({in.n, in.s}, u.options()),
           gC = make({in.n, in.s}, u.options()), gA = make({in.d, in.s}, f32), gD, gbias, ginit;
    if (in.z.defined()) gz = make({in.n, in.d}, u.options());
    if (in.D) gD = make({in.d}, f32);
    if (in.bias) gbias = make({in.d}, f32);
    if (in.init) {
        ginit = make({n_rays, in.d, in.s}, f32);
        if (none && gfinal) ginit.copy_(gfinal->view({n_rays, in.d, in.s}));
    }
    if (!none) {
        auto a = in.args(softplus);
        seq.into(a);
        a.ray_order = ptr<int32_t>(order);
        a.grad_outputs = gy.data_ptr(); a.grad_outputs_stride = row_stride(gy); a.grad_final_state = ptr<float>(gfinal);
        Tensor ws = at::empty({nfa_selective_scan_workspace_bytes(n_rays, in.n, a.channels, a.states, 1)}, opts(u, at::kByte));
        nfa_selective_scan_grads gr{};
        gr.inputs = gu.data_ptr(); gr.delta = gdt.data_ptr(); gr.gate = ptr<void>(gz); gr.B = gB.data_ptr(); gr.C = gC.data_ptr();
        gr.A = ptr<float>(gA); gr.D = ptr<float>(gD); gr.delta_bias = ptr<float>(gbias); gr.initial_state = ptr<float>(ginit);
        check_rc(nfa_selective_scan_bwd(&a, ptr<float>(kept), &gr, ws.data_ptr(), stream_of(u)));
    }
    return {gu, gdt, some(gz), gB, gC, gA, some(gD), some(gbias), some(ginit)};
}

Tensor selective_scan_step(const Tensor &u, const Tensor &dt, const OptTensor &z, const Tensor &B, const Tensor &C, const Tensor &A, const OptTensor &D,
                           const OptTensor &bias, const Tensor &state_, bool softplus, const Tensor &to) {
    const ScanInputs in(u, dt, z, B, C, A, D, bias, std::nullopt, u.dim() ? u.size(0) : 0);
    const int64_t ns = in.n * in.d * in.s;
    const Tensor state = dense_of(state_, "state", at::kFloat, ns, u);
    check_len(to, "out_state", at::kFloat, ns, u);
    Guard g(device_of(u));
    Tensor out = at::empty({in.n, in.d}, u.options());
    auto a = in.args(softplus);
    a.n_rays = in.n;
    check_rc(nfa_selective_scan_step(&a, ptr<float>(state), out.data_ptr(), ptr<float>(to), stream_of(u)));
    return out;
}

// ---------------------------------------------------------------------------------------------------
// the feature operators as a whole: refusals, autograd and the calls above in one go (the Python layer above this only names the
// activation; nerfacc_amd/dense.py and selective.py hold the same steps for the ctypes face)
// ---------------------------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline Tensor get(const OptTensor &t) { return t && t->defined() ? *t : Tensor(); }

void check_native(const char *op, const Tensor &x) {
    TORCH_CHECK(x.is_cuda(), op, ": inputs must be a CUDA/HIP tensor (nerfacc_amd has no CPU kernels)");
    const auto t = x.scalar_type();
    TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, op, ": inputs must be float32, bfloat16 or float16, got ", t);
}
void check_like(const char *op, const char *what, const Tensor &t, const Tensor &x, at::IntArrayRef shape, at::ScalarType dtype) {
    if (!t.defined()) return;
    TORCH_CHECK(t.device() == x.device(), op, ": ", what, " is on ", t.device(), ", inputs on ", x.device());
    TORCH_CHECK_TYPE(t.scalar_type() == dtype, op, ": ", what, " must have dtype ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.sizes() == shape, op, ": ", what, " must have shape ", shape, ", got ", t.sizes());
}
// a tangent would be dropped without a word
void refuse_forward(const char *op, std::initializer_list<OptTensor> tensors) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (auto &t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!(t && t->defined() && t->_fw_grad(0).defined()), op, ": forward mode derivatives are not implemented");
}
// whether autograd records the call; refuses one whose captured backward pass would end the process
bool records_grad(const char *op, const Tensor &x, std::initializer_list<OptTensor> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    bool any = false;
    for (auto &t : tensors) any |= t && t->defined() && t->requires_grad();
    if (!any) return false;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream_of(x), &status) != hipSuccess) (void)hipGetLastError();
    TORCH_CHECK(status == hipStreamCaptureStatusNone || foreign_nodes(std::vector<OptTensor>(tensors)) == 0, op,
                ": captured into a graph while an eager autograd graph of the same tensors lives (its backward pass could not be captured): drop the "
                "eager outputs first, or call under torch.no_grad()");
    return true;
}
// The results of a backward pass that differentiates once.  Under create_graph those that depend on something learnt (`depends`: through the
// tensors of the forward call; all of them where a gradient that came in requires one) are an error in another backward pass, as torch's
// once_differentiable makes those of the second kind: a penalty on them would have no effect otherwise.
variable_list once(variable_list grads, const variable_list &outer, std::initializer_list<bool> depends) {
    if (!at::GradMode::is_enabled()) return grads;
    bool any = false;
    for (auto &g : outer) any |= g.defined() && g.requires_grad();
    variable_list held;
    auto learnt = [&](size_t i) { return grads[i].defined() && (any || (i < depends.size() && depends.begin()[i])); };
    for (size_t i = 0; i < grads.size(); ++i)
        if (learnt(i)) held.push_back(grads[i].detach().requires_grad_(true));
    if (held.empty()) return grads;
    const size_t n = held.size();
    auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable", n);
    held = (*error)(std::move(held));
    for (size_t i = 0, k = 0; i < grads.size(); ++i)
        if (learnt(i)) grads[i] = held[k++];
    return grads;
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    enum : int64_t { kBias = 1 << 8, kResidual = 1 << 9, kSlope = 1 << 10, kInputs = 1 << 11, kWeight = 1 << 12 };     // beside the activation
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &b, const OptTensor &r, int64_t act, bool learns) {
        auto res = linear_fwd(x, w, b, r, act, learns);
        const Tensor out = std::get<0>(res), kept = get(std::get<1>(res));
        const bool smooth = act != NFA_ACT_NONE && act != NFA_ACT_RELU;         // (kSlope: act' depends on something learnt)
        ctx->saved_data["call"] = act | (b && b->defined() ? kBias : 0) | (r && r->defined() ? kResidual : 0) | (smooth && learns ? kSlope : 0) |
                                  (x.requires_grad() ? kInputs : 0) | (w.requires_grad() ? kWeight : 0);
        if (learns) ctx->save_for_backward({x, w, !kept.defined() && act != NFA_ACT_NONE ? out : kept});
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list out(6);
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const int64_t call = ctx->saved_data["call"].toInt();
        const bool has_bias = call & kBias, need_b = has_bias && ctx->needs_input_grad(2);
        if (need_x || need_w || need_b) {
            const auto saved = ctx->get_saved_variables();
            auto g = linear_bwd(grads[0], saved[0], saved[1], some(saved[2]), call & 255, need_x, need_w, need_b);
            out[0] = get(std::get<0>(g));
            out[1] = get(std::get<1>(g));
            out[2] = get(std::get<2>(g));
        }
        if ((call & kResidual) && ctx->needs_input_grad(has_bias ? 3 : 2)) out[3] = grads[0];     // (counts the given tensors)
        return once(out, grads, {(call & (kSlope | kWeight)) != 0, (call & (kSlope | kInputs)) != 0, (call & kSlope) != 0, false});
    }
};

Tensor linear(const Tensor &x, const Tensor &w, const OptTensor &b, const OptTensor &r, int64_t act) {
    refuse_forward("linear", {x, w, b, r});
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1), "linear: inputs (..., in) and weight (out, in) expected, got ", x.sizes(),
                      " and ", w.sizes());
    const int64_t n = w.size(0), k = w.size(1);
    TORCH_CHECK_VALUE(n > 0 && k > 0, "linear: in_features and out_features must be at least 1");
    TORCH_CHECK_VALUE(n <= (1 << 20) && k <= (1 << 20), "linear: more than 2^20 features");
    check_native("linear", x);
    at::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    const auto dt = x.scalar_type();
    check_like("linear", "weight", w, x, {n, k}, dt);
    check_like("linear", "bias", get(b), x, {n}, dt);
    check_like("linear", "residual", get(r), x, shape, dt);
    const bool flat = x.dim() == 2;
    const Tensor x2 = flat ? x : x.reshape({-1, k});
    OptTensor r2 = some(get(r));
    if (r2 && !flat) r2 = r2->reshape({-1, n});
    const OptTensor b2 = some(get(b));
    Tensor out;
    if (records_grad("linear", x, {x, w, b, r})) {
        const bool learns = x.requires_grad() || w.requires_grad() || (b2 && b2->requires_grad());
        out = LinearFn::apply(x2, w, b2, r2, act, learns);
    } else {
        out = std::get<0>(linear_fwd(x2, w, b2, r2, act, false));
    }
    return flat ? out : out.view(shape);
}

void check_channels(const char *op, int64_t d) { TORCH_CHECK_VALUE(d <= (1 << 23), op, ": more than 2^23 channels"); }
// number of sequences of a batched or packed tensor
int64_t sequences_of(const char *op, const Tensor &x, const OptTensor &info) {
    int64_t n = 0;
    if (!info || !info->defined()) {
        TORCH_CHECK_VALUE(x.dim() == 3, op, ": inputs must be (n_rays, n, channels), or (n_samples, channels) with packed_info; got ", x.sizes());
        n = x.size(0);
    } else {
        TORCH_CHECK_VALUE(x.dim() == 2, op, ": with packed_info inputs must be (n_samples, channels), got ", x.sizes());
        TORCH_CHECK_VALUE(info->dim() == 2 && info->size(1) == 2, op, ": packed_info must be 2-D with shape (n_rays, 2), got ", info->sizes());
        n = info->size(0);
    }
    TORCH_CHECK_VALUE(x.size(-1) > 0, op, ": at least one channel expected");
    check_channels(op, x.size(-1));
    TORCH_CHECK_VALUE(n < (1ll << 31) && x.numel() / x.size(-1) < (1ll << 31), op, ": more than 2^31 - 1 rays or samples");
    return n;
}
struct RowMap {
    OptTensor info, ray, pos;
    RowMap(const OptTensor &info_, const Tensor &x, int64_t n_rays) {
        if (info_ && info_->defined()) info = info_->contiguous();
        else if (n_rays == 0) info = at::empty({0, 2}, opts(x, at::kLong));
        if (info) std::tie(ray, pos) = row_map(*info, x.size(0));
    }
    // the dealing order of a scan: where whole rays are a few for each wave place of the chip, their lengths decide when the last one ends.
    // (64 channels, without and with the order, which takes 10 us by itself: 1024 ragged rays forward 115 and 114 us, backward 232 and 190;
    // 4096 195 and 130, 482 and 336; 16384 397 and 313; 131072 515 and 488, no longer worth one workgroup's pass over all rays)
    OptTensor order(int64_t n_rays, int64_t rows) const {
        if (!info || n_rays < 1024 || n_rays > 65536) return std::nullopt;
        return ray_order(*info, rows);
    }
};
inline Tensor flat_rows(const Tensor &t) { return !t.defined() || t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

struct CausalConvFn : torch::autograd::Function<CausalConvFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &b, const OptTensor &init, const OptTensor &info,
                                 const OptTensor &ray, const OptTensor &pos, int64_t n_rays, int64_t act, bool want_final) {
        ctx->set_materialize_grads(false);
        auto res = causal_conv_fwd(x, w, b, init, info, ray, pos, n_rays, act, want_final);
        ctx->save_for_backward({x, w, get(b), get(init), get(info), get(ray), get(pos)});
        ctx->saved_data["n_rays"] = n_rays;
        ctx->saved_data["act"] = act;
        if (!want_final) return {std::get<0>(res)};
        return {std::get<0>(res), *std::get<1>(res)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const bool has_b = s[2].defined(), has_init = s[3].defined();
        const Tensor gy = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
        auto g = causal_conv_bwd(gy, grads.size() > 1 ? some(grads[1]) : std::nullopt, s[0], s[1], some(s[2]), some(s[3]), some(s[4]), some(s[5]), some(s[6]),
                                 ctx->saved_data["n_rays"].toInt(), ctx->saved_data["act"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                                 has_b && ctx->needs_input_grad(2), has_init && ctx->needs_input_grad(has_b ? 3 : 2));
        variable_list out(10);
        out[0] = get(std::get<0>(g)); out[1] = get(std::get<1>(g)); out[2] = get(std::get<2>(g)); out[3] = get(std::get<3>(g));
        auto learns = [&](int i) { return s[i].defined() && s[i].requires_grad(); };
        const bool slope = ctx->saved_data["act"].toInt() != NFA_ACT_NONE && (learns(0) || learns(1) || learns(2) || learns(3));
        return once(out, grads, {slope || learns(1), slope || learns(0) || learns(3), slope, slope || learns(1)});
    }
};

int64_t check_width(const char *op, const Tensor &w, int64_t channels) {
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) == channels && w.size(1) >= 2 && w.size(1) <= 4, op, ": weight must be (channels, width) with ", channels,
                      " channels and width 2, 3 or 4, got ", w.sizes());
    return w.size(1);
}

std::tuple<Tensor, OptTensor> causal_conv(const Tensor &x_, const Tensor &w, const OptTensor &b, const OptTensor &info, const OptTensor &init, int64_t act,
                                          bool want_final) {
    refuse_forward("causal_conv", {x_, w, b, init});
    const int64_t n_rays = sequences_of("causal_conv", x_, info), d = x_.size(-1), width = check_width("causal_conv", w, d);
    check_native("causal_conv", x_);
    const auto dt = x_.scalar_type();
    check_like("causal_conv", "weight", w, x_, {d, width}, dt);
    check_like("causal_conv", "bias", get(b), x_, {d}, dt);
    check_like("causal_conv", "packed_info", get(info), x_, {n_rays, 2}, at::kLong);
    check_like("causal_conv", "initial_state", get(init), x_, {n_rays, width - 1, d}, dt);
    const Tensor x = flat_rows(x_);
    Guard g(device_of(x));
    const RowMap m(info, x, n_rays);
    const OptTensor b2 = some(get(b)), init2 = some(get(init));
    Tensor out;
    OptTensor last;
    if (records_grad("causal_conv", x, {x_, w, b, init})) {
        auto res = CausalConvFn::apply(x, w, b2, init2, m.info, m.ray, m.pos, n_rays, act, want_final);
        out = res[0];
        if (want_final) last = res[1];
    } else {
        std::tie(out, last) = causal_conv_fwd(x, w, b2, init2, m.info, m.ray, m.pos, n_rays, act, want_final);
    }
    return {x_.dim() == 2 ? out : out.view(x_.sizes()), last};
}

// whether two tensors share memory, by the spans between their first and last element
bool overlaps(const Tensor &s, const Tensor &t) {
    if (s.numel() == 0 || t.numel() == 0) return false;
    auto span = [](const Tensor &x) {
        int64_t reach = 1;
        for (int64_t i = 0; i < x.dim(); ++i) reach += (x.size(i) - 1) * x.stride(i);
        const char *at = (const char *)x.data_ptr();
        return std::pair<const char *, const char *>(at, at + reach * x.element_size());
    };
    const auto a = span(s), b = span(t);
    return a.first < b.second && b.first < a.second;
}
// where a step leaves its new state: `state` itself, or a buffer that shares no memory with it; nor with what the step reads beside it, in
// whatever order its workgroups run
Tensor state_buffer(const char *op, const Tensor &state, const OptTensor &to_, std::initializer_list<std::pair<const char *, OptTensor>> inputs) {
    const Tensor to = get(to_);
    if (!to.defined()) return at::empty(state.sizes(), state.options());
    TORCH_CHECK_VALUE(to.is_contiguous(), op, ": out_state must be contiguous");
    if (!(to.data_ptr() == state.data_ptr() && state.is_contiguous()))
        TORCH_CHECK_VALUE(!overlaps(state, to), op, ": out_state overlaps state; pass state itself to update it in place");
    for (auto &p : inputs) TORCH_CHECK_VALUE(!(p.second && p.second->defined() && overlaps(*p.second, to)), op, ": out_state overlaps ", p.first);
    return to;
}
void refuse_grad(const char *op, const char *other, std::initializer_list<OptTensor> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (auto &t : tensors)
        TORCH_CHECK(!(t && t->defined() && t->requires_grad()), op, " is not differentiable: call it under torch.no_grad(), or use ", other,
                    " with initial_state");
}
void written(const OptTensor &to) {
    if (to && to->defined() && !to->is_inference()) to->unsafeGetTensorImpl()->bump_version();
}

std::tuple<Tensor, Tensor> causal_conv_one(const Tensor &x, const Tensor &state, const Tensor &w, const OptTensor &b, int64_t act, const OptTensor &to_) {
    refuse_forward("causal_conv_step", {x, state, w, b, to_});
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0, "causal_conv_step: inputs must be (n_rays, channels)");
    const int64_t r = x.size(0), d = x.size(1), width = check_width("causal_conv_step", w, d);
    check_channels("causal_conv_step", d);
    check_native("causal_conv_step", x);
    const auto dt = x.scalar_type();
    check_like("causal_conv_step", "state", state, x, {r, width - 1, d}, dt);
    check_like("causal_conv_step", "weight", w, x, {d, width}, dt);
    check_like("causal_conv_step", "bias", get(b), x, {d}, dt);
    check_like("causal_conv_step", "out_state", get(to_), x, {r, width - 1, d}, dt);
    refuse_grad("causal_conv_step", "causal_conv", {x, state, w, b, to_});
    const Tensor to = state_buffer("causal_conv_step", state, to_, {{"inputs", x}, {"weight", w}, {"bias", b}});
    const Tensor out = causal_conv_step(x, state, w, some(get(b)), act, to);
    written(to_);
    return {out, to};
}

struct SelectiveScanFn : torch::autograd::Function<SelectiveScanFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &dt, const Tensor &B, const Tensor &C, const Tensor &A, const OptTensor &z,
                                 const OptTensor &D, const OptTensor &bias, const OptTensor &init, const OptTensor &info, const OptTensor &ray,
                                 const OptTensor &pos, const OptTensor &order, int64_t n_rays, bool softplus, bool want_final) {
        ctx->set_materialize_grads(false);
        auto res = selective_scan_fwd(u, dt, z, B, C, A, D, bias, init, info, ray, pos, order, n_rays, softplus, want_final, true);
        ctx->save_for_backward({u, dt, B, C, A, get(z), get(D), get(bias), get(init), get(info), get(ray), get(pos), get(std::get<2>(res)), get(order)});
        ctx->saved_data["n_rays"] = n_rays;
        ctx->saved_data["softplus"] = softplus;
        if (!want_final) return {std::get<0>(res)};
        return {std::get<0>(res), *std::get<1>(res)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const Tensor gy = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
        const auto g = selective_scan_bwd(gy, grads.size() > 1 ? some(grads[1]) : std::nullopt, s[0], s[1], some(s[5]), s[2], s[3], s[4], some(s[6]), some(s[7]),
                                          some(s[8]), s[12], some(s[9]), some(s[10]), some(s[11]), some(s[13]), ctx->saved_data["n_rays"].toInt(),
                                          ctx->saved_data["softplus"].toBool());
        // forward's order: u, dt, B, C, A, z, D, bias, init; needs_input_grad counts the tensors that were given
        static constexpr int from[9] = {0, 1, 3, 4, 5, 2, 6, 7, 8};
        variable_list out(16);
        int given = 0;
        for (int i = 0; i < 9; ++i) {
            if (!s[i].defined()) continue;
            if (ctx->needs_input_grad(given++)) out[i] = get(g[from[i]]);
        }
        // outputs are linear in u, B, C, D and the initial state, each by itself
        bool any[9] = {};
        for (int i = 0; i < 9; ++i)
            for (int j = 0; j < 9; ++j) any[i] |= s[j].defined() && s[j].requires_grad() && (j != i || i == 1 || i == 4 || i == 5 || i == 7);
        return once(out, grads, {any[0], any[1], any[2], any[3], any[4], any[5], any[6], any[7], any[8]});
    }
};

void check_scan(const char *op, const Tensor &x, at::IntArrayRef rows, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const OptTensor &D,
                const OptTensor &z, const OptTensor &bias) {
    TORCH_CHECK_VALUE(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= NFA_SCAN_MAX_STATES, op, ": A must be (channels, states) with 1 to ", NFA_SCAN_MAX_STATES,
                      " states, got ", A.sizes());
    check_native(op, x);
    const int64_t d = x.size(-1), s = A.size(1);
    at::DimVector wide(rows.begin(), rows.end()), narrow(wide);
    wide.push_back(d);
    narrow.push_back(s);
    const auto t = x.scalar_type();
    check_like(op, "delta", dt, x, wide, t);
    check_like(op, "A", A, x, {d, s}, at::kFloat);
    check_like(op, "B", B, x, narrow, t);
    check_like(op, "C", C, x, narrow, t);
    check_like(op, "D", get(D), x, {d}, at::kFloat);
    check_like(op, "gate", get(z), x, wide, t);
    check_like(op, "delta_bias", get(bias), x, {d}, at::kFloat);
}

std::tuple<Tensor, OptTensor> selective_scan(const Tensor &x_, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const OptTensor &D,
                                             const OptTensor &z, const OptTensor &bias, bool softplus, const OptTensor &info, const OptTensor &init,
                                             bool want_final) {
    refuse_forward("selective_scan", {x_, dt, A, B, C, D, z, bias, init});
    const int64_t n_rays = sequences_of("selective_scan", x_, info);
    check_scan("selective_scan", x_, x_.sizes().slice(0, x_.dim() - 1), dt, A, B, C, D, z, bias);
    check_like("selective_scan", "packed_info", get(info), x_, {n_rays, 2}, at::kLong);
    check_like("selective_scan", "initial_state", get(init), x_, {n_rays, x_.size(-1), A.size(1)}, at::kFloat);
    Guard g(device_of(x_));
    const Tensor x = flat_rows(x_);
    const RowMap m(info, x, n_rays);
    const OptTensor order = m.order(n_rays, x.size(0));
    const OptTensor z2 = some(flat_rows(get(z))), D2 = some(get(D)), bias2 = some(get(bias)), init2 = some(get(init));
    Tensor out;
    OptTensor last;
    if (records_grad("selective_scan", x, {x_, dt, A, B, C, D, z, bias, init})) {
        auto res = SelectiveScanFn::apply(x, flat_rows(dt), flat_rows(B), flat_rows(C), A, z2, D2, bias2, init2, m.info, m.ray, m.pos, order, n_rays, softplus, want_final);
        out = res[0];
        if (want_final) last = res[1];
    } else {
        OptTensor kept;
        std::tie(out, last, kept) = selective_scan_fwd(x, flat_rows(dt), z2, flat_rows(B), flat_rows(C), A, D2, bias2, init2, m.info, m.ray, m.pos, order, n_rays, softplus,
                                                       want_final, false);
    }
    return {x_.dim() == 2 ? out : out.view(x_.sizes()), last};
}

std::tuple<Tensor, Tensor> selective_scan_one(const Tensor &x, const Tensor &dt, const Tensor &A, const Tensor &B, const Tensor &C, const Tensor &state,
                                              const OptTensor &D, const OptTensor &z, const OptTensor &bias, bool softplus, const OptTensor &to_) {
    refuse_forward("selective_scan_step", {x, dt, A, B, C, D, z, bias, state, to_});
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) > 0, "selective_scan_step: inputs must be (n_rays, channels)");
    check_channels("selective_scan_step", x.size(1));
    check_scan("selective_scan_step", x, x.sizes().slice(0, 1), dt, A, B, C, D, z, bias);
    const int64_t r = x.size(0), d = x.size(1), s = A.size(1);
    check_like("selective_scan_step", "state", state, x, {r, d, s}, at::kFloat);
    check_like("selective_scan_step", "out_state", get(to_), x, {r, d, s}, at::kFloat);
    refuse_grad("selective_scan_step", "selective_scan", {x, dt, A, B, C, D, z, bias, state, to_});
    const Tensor to = state_buffer("selective_scan_step", state, to_,
                                   {{"inputs", x}, {"delta", dt}, {"A", A}, {"B", B}, {"C", C}, {"D", D}, {"gate", z}, {"delta_bias", bias}});
    const Tensor out = selective_scan_step(x, dt, some(get(z)), B, C, A, some(get(D)), some(get(bias)), state, softplus, to);
    written(to_);
    return {out, to};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "nerfacc_amd._hip: torch C++ extension over the C ABI of libnerfacc_hip.so (MI355X / gfx950)";
    m.def("version", []() { return std::string(nfa_version()); });

    py::class_<RaySegmentsSpec>(m, "RaySegmentsSpec")
        .def(py::init<>())
        .def_readwrite("vals", &RaySegmentsSpec::vals)
        .def_readwrite("is_left", &RaySegmentsSpec::is_left)
        .def_readwrite("is_right", &RaySegmentsSpec::is_right)
        .def_readwrite("is_valid", &RaySegmentsSpec::is_valid)
        .def_readwrite("chunk_starts", &RaySegmentsSpec::chunk_starts)
        .def_readwrite("chunk_cnts", &RaySegmentsSpec::chunk_cnts)
        .def_readwrite("ray_indices", &RaySegmentsSpec::ray_indices)
        .def("check", &RaySegmentsSpec::check);

    using namespace pybind11::literals;
    // ---- the reference boundary (nerfacc.cpp:126-163), same names and argument order
    m.def("is_cub_available", []() { return true; });     // scan-by-key is native (scan.hip): the keyed path is always there
    m.def("ray_aabb_intersect", &ray_aabb_intersect);
    m.def("traverse_grids", &traverse_grids);
    m.def("inclusive_sum", [](const Tensor &s, const Tensor &c, const Tensor &x, bool normalize, bool backward) {
        return scan_packed(s, c, x, NFA_OP_SUM, true, backward, normalize); });
    m.def("exclusive_sum", [](const Tensor &s, const Tensor &c, const Tensor &x, bool normalize, bool backward) {
        return scan_packed(s, c, x, NFA_OP_SUM, false, backward, normalize); });
    m.def("inclusive_prod_forward", [](const Tensor &s, const Tensor &c, const Tensor &x) { return scan_packed(s, c, x, NFA_OP_PROD, true, false, false); });
    m.def("exclusive_prod_forward", [](const Tensor &s, const Tensor &c, const Tensor &x) { return scan_packed(s, c, x, NFA_OP_PROD, false, false, false); });
    m.def("inclusive_prod_backward", [](const Tensor &s, const Tensor &c, const Tensor &x, const Tensor &y, const Tensor &gy) {
        return prod_bwd(std::nullopt, s, c, x, y, gy, true); });
    m.def("exclusive_prod_backward", [](const Tensor &s, const Tensor &c, const Tensor &x, const Tensor &y, const Tensor &gy) {
        return prod_bwd(std::nullopt, s, c, x, y, gy, false); });
    m.def("inclusive_sum_cub", [](const Tensor &k, const Tensor &x, bool backward) { return scan_keyed(k, x, NFA_OP_SUM, true, backward); });
    m.def("exclusive_sum_cub", [](const Tensor &k, const Tensor &x, bool backward) { return scan_keyed(k, x, NFA_OP_SUM, false, backward); });
    m.def("inclusive_prod_cub_forward", [](const Tensor &k, const Tensor &x) { return scan_keyed(k, x, NFA_OP_PROD, true, false); });
    m.def("exclusive_prod_cub_forward", [](const Tensor &k, const Tensor &x) { return scan_keyed(k, x, NFA_OP_PROD, false, false); });
    m.def("inclusive_prod_cub_backward", [](const Tensor &k, const Tensor &x, const Tensor &y, const Tensor &gy) {
        return prod_bwd(k, std::nullopt, std::nullopt, x, y, gy, true); });
    m.def("exclusive_prod_cub_backward", [](const Tensor &k, const Tensor &x, const Tensor &y, const Tensor &gy) {
        return prod_bwd(k, std::nullopt, std::nullopt, x, y, gy, false); });
    // the generic forms behind the 14 scan names (op, inclusive, reverse[, normalize]); tests drive every combination
    m.def("_packed", &scan_packed);
    m.def("_keyed", &scan_keyed);
    m.def("importance_sampling", &importance_sampling);
    m.def("searchsorted", &searchsorted);
    m.def("transform_stot", &transform_stot, "s_vals"_a, "t_min"_a, "t_max"_a, "lindisp"_a);
    m.def("edge_cdfs_fwd", &edge_cdfs_fwd, "t_edges"_a, "sigmas"_a, "want_trans"_a);
    m.def("edge_cdfs_bwd", &edge_cdfs_bwd, "t_edges"_a, "trans"_a, "g_cdfs"_a);
    m.def("pdf_loss_fwd", &pdf_loss_fwd, "query_vals"_a, "cdfs_query"_a, "key_vals"_a, "cdfs_key"_a, "eps"_a, "want_grad"_a);
    m.def("pdf_loss_bwd", &pdf_loss_bwd, "g_loss"_a, "ids_left"_a, "ids_right"_a, "coef"_a, "n_key"_a);
    m.def("opencv_lens_undistortion", [](py::args, py::kwargs) {
        raise_not_implemented("camera undistortion (camera.cu) is outside the OccGrid hot path and not built"); });
    m.def("opencv_lens_undistortion_fisheye", [](py::args, py::kwargs) {
        raise_not_implemented("camera undistortion (camera.cu) is outside the OccGrid hot path and not built"); });

    // ---- fused entry points of this implementation
    m.def("release_workspace", &release_workspace,
          "free this host thread's retained traversal workspace (<= 64 MB per device and stream) and any count pass launched ahead");
    m.def("sample_occgrid", &sample_occgrid, "rays_o"_a, "rays_d"_a, "binaries"_a, "aabbs"_a, "near_planes"_a, "far_planes"_a, "step_size"_a,
          "cone_angle"_a, "rays_mask"_a = py::none(), "traverse_steps_limit"_a = -1, "with_terminate_planes"_a = false, "near_plane"_a = 0.0,
          "far_plane"_a = std::numeric_limits<double>::infinity(), "t_min"_a = py::none(), "t_max"_a = py::none(), "jitter"_a = py::none(),
          "jitter_scale"_a = 0.0);
    m.def("pack_info", &pack_info, "ray_indices"_a, "n_rays"_a);
    m.def("unpack_info", &unpack_info, "chunk_starts"_a, "chunk_cnts"_a, "n"_a);
    m.def("render_weight_from_density_fwd", &render_weight_from_density_fwd, "ray_indices"_a, "t_starts"_a, "t_ends"_a, "sigmas"_a,
          "prefix_trans"_a = py::none());
    m.def("render_weight_from_density_bwd", &render_weight_from_density_bwd);
    m.def("sample_positions", &sample_positions, "rays_o"_a, "rays_d"_a, "ray_indices"_a, "t_starts"_a, "t_ends"_a, "with_dirs"_a = false);
    m.def("visibility_compact", &visibility_compact, "ray_indices"_a, "t_starts"_a, "t_ends"_a, "dens"_a, "from_alpha"_a, "early_stop_eps"_a,
          "alpha_thre"_a, "want_mask"_a = false);
    m.def("accumulate_along_rays", &accumulate_along_rays, "ray_indices"_a, "weights"_a, "values"_a, "n_rays"_a, "outputs"_a = py::none());
    m.def("accumulate_along_rays_bwd", &accumulate_along_rays_bwd);
    m.def("rendering_fwd", &rendering_fwd);
    m.def("rendering_bwd", &rendering_bwd, "ray_indices"_a, "t_starts"_a, "t_ends"_a, "sigmas"_a, "rgbs"_a, "weights"_a, "trans"_a, "alphas"_a,
          "opacities"_a, "depths"_a, "n_rays"_a, "bkgd"_a, "expected_depths"_a, "g_colors"_a, "g_opac"_a, "g_depth"_a, "g_w"_a, "g_T"_a, "g_a"_a,
          "need_sigma"_a = true, "need_rgb"_a = true);
    m.def("rendering", &rendering_autograd, "ray_indices"_a, "t_starts"_a, "t_ends"_a, "sigmas"_a, "rgbs"_a, "n_rays"_a, "render_bkgd"_a,
          "expected_depths"_a);
    m.def("grid_cell_points", &grid_cell_points);
    m.def("grid_ema_update", &grid_ema_update);
    m.def("grid_threshold", &grid_threshold, "occs"_a, "occ_thre"_a, "shape"_a = py::none());
    m.def("grid_mark_invisible", &grid_mark_invisible);
    m.def("packed_bricks", &packed_bricks);
    m.def("grid_occupied_counts", &grid_occupied_counts);
    m.def("grid_occupied_cells", &grid_occupied_cells);
    m.def("set_timing", &set_timing, "names"_a = py::none());
    m.def("timing_summary", &timing_summary);
    m.def("linear", &linear);
    m.def("causal_conv", &causal_conv);
    m.def("causal_conv_one", &causal_conv_one);
    m.def("selective_scan", &selective_scan);
    m.def("selective_scan_one", &selective_scan_one);
    m.def("foreign_nodes", &foreign_nodes);
    m.def("linear_fwd", &linear_fwd);
    m.def("linear_bwd", &linear_bwd);
    m.def("row_map", &row_map);
    m.def("ray_order", &ray_order);
    m.def("causal_conv_fwd", &causal_conv_fwd);
    m.def("causal_conv_bwd", &causal_conv_bwd);
    m.def("causal_conv_step", &causal_conv_step);
    m.def("selective_scan_fwd", &selective_scan_fwd);
    m.def("selective_scan_bwd", &selective_scan_bwd);
    m.def("selective_scan_step", &selective_scan_step);
}
