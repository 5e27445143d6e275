// The C ABI of the products over 16-bit weights (include/mlxs_moe.h): argument checks and dense strides.
#include <cmath>

#include "common.cuh"
#include "handle.h"

static constexpr uint32_t MAX_DIM = 262144, MAX_ROWS = 1u << 22, MAX_GROUPS = 1024, MAX_RANK = 256;

// the caller's current device comes back on every way out
struct DeviceGuard {
    int before = -1;
    cudaError_t enter(int device) {
        cudaError_t e = cudaGetDevice(&before);
        if (e != cudaSuccess) { before = -1; return e; }
        return before == device ? cudaSuccess : cudaSetDevice(device);
    }
    ~DeviceGuard() {
        int now = -1;
        if (before >= 0 && cudaGetDevice(&now) == cudaSuccess && now != before) cudaSetDevice(before);
    }
};

static int check_types(const char* who, uint32_t dtype, uint32_t out_dtype) {
    if (dtype != MLXS_DTYPE_BF16 && dtype != MLXS_DTYPE_F16) return mlxs_fail(MLXS_E_CONFIG, "%s: dtype %u is neither bf16 nor f16", who, dtype);
    if (out_dtype != dtype && out_dtype != MLXS_DTYPE_F32)
        return mlxs_fail(MLXS_E_CONFIG, "%s: out_dtype %u is neither dtype nor f32", who, out_dtype);
    return 0;
}
static int check_dim(const char* who, const char* what, uint32_t v) {
    if (v == 0 || v % 8 || v > MAX_DIM) return mlxs_fail(MLXS_E_CONFIG, "%s: %s %u is not a multiple of 8 in 8..%u", who, what, v, MAX_DIM);
    return 0;
}
// a dense stride for 0; otherwise a multiple of 8 elements that holds what it steps over
static int take_stride(const char* who, const char* what, uint64_t given, uint64_t dense, uint64_t least, size_t* out) {
    *out = (size_t)(given ? given : dense);
    if (*out % 8 || *out < least || *out > (1ull << 38))
        return mlxs_fail(MLXS_E_ARG, "%s: %s %llu is not a multiple of 8 in %llu..2^38", who, what, (unsigned long long)*out, (unsigned long long)least);
    return 0;
}
static int check_ptr(const char* who, const char* what, const void* p, uintptr_t align) {
    if (!p) return mlxs_fail(MLXS_E_ARG, "%s: %s is null", who, what);
    if (reinterpret_cast<uintptr_t>(p) % align) return mlxs_fail(MLXS_E_ARG, "%s: %s must be %u-byte aligned", who, what, (unsigned)align);
    return 0;
}

// the bounds of the kernels' waits (mlxs_moe_debug_wait)
template <class Args>
static void set_waits(Args& a, const mlxs_moe* h) {
    if (h->dbg_poll_limit) a.poll_limit = h->dbg_poll_limit;
    a.withhold = h->dbg_withhold;
}

extern "C" int mlxs_moe_grouped(mlxs_moe* h, const mlxs_grouped_desc* d, const void* x_dev, const void* w_dev, const uint32_t* offsets_dev,
                                const uint32_t* order_dev, void* y_dev, void* stream) {
    const char* who = "grouped";
    if (!d) return mlxs_fail(MLXS_E_ARG, "grouped: null descriptor");
    if (d->struct_size != sizeof *d) return mlxs_fail(MLXS_E_CONFIG, "grouped: struct_size %u, this library has %zu", d->struct_size, sizeof *d);
    int rc;
    if ((rc = check_types(who, d->dtype, d->out_dtype)) || (rc = check_dim(who, "n_in", d->n_in)) || (rc = check_dim(who, "n_out", d->n_out))) return rc;
    if (d->layout > MLXS_LAYOUT_IN_OUT) return mlxs_fail(MLXS_E_CONFIG, "grouped: layout %u unknown", d->layout);
    if (d->act > MLXS_GROUPED_SWIGLU) return mlxs_fail(MLXS_E_CONFIG, "grouped: act %u unknown", d->act);
    if (!(d->act_limit >= 0.f) || std::isinf(d->act_limit)) return mlxs_fail(MLXS_E_CONFIG, "grouped: act_limit is negative or not finite");
    if (d->act_limit > 0.f && d->act != MLXS_GROUPED_SWIGLU) return mlxs_fail(MLXS_E_CONFIG, "grouped: act_limit without an activation");
    if (d->n_groups == 0 || d->n_groups > MAX_GROUPS) return mlxs_fail(MLXS_E_CONFIG, "grouped: n_groups %u outside 1..%u", d->n_groups, MAX_GROUPS);
    if (d->row_flags & ~(uint32_t)(MLXS_ROWS_GATHER | MLXS_ROWS_SCATTER)) return mlxs_fail(MLXS_E_CONFIG, "grouped: row_flags %u unknown", d->row_flags);
    if (d->rows > MAX_ROWS || d->x_rows > MAX_ROWS || d->y_rows > MAX_ROWS)
        return mlxs_fail(MLXS_E_TOO_MANY_TOKENS, "grouped: rows %u, x_rows %u, y_rows %u: at most %u", d->rows, d->x_rows, d->y_rows, MAX_ROWS);
    GroupedArgs a{};
    a.gather = d->row_flags & MLXS_ROWS_GATHER; a.scatter = d->row_flags & MLXS_ROWS_SCATTER;
    if (!a.gather && d->x_rows < d->rows) return mlxs_fail(MLXS_E_ARG, "grouped: x_rows %u under rows %u without a gather", d->x_rows, d->rows);
    if (!a.scatter && d->y_rows < d->rows) return mlxs_fail(MLXS_E_ARG, "grouped: y_rows %u under rows %u without a scatter", d->y_rows, d->rows);
    if (a.gather && d->x_div == 0) return mlxs_fail(MLXS_E_ARG, "grouped: x_div is 0");
    a.G = d->n_groups; a.K = d->n_in; a.N = d->n_out; a.rows = d->rows;
    a.x_div = a.gather ? d->x_div : 1; a.x_rows = d->x_rows; a.y_rows = d->y_rows;
    a.in_out = d->layout == MLXS_LAYOUT_IN_OUT; a.swiglu = d->act == MLXS_GROUPED_SWIGLU; a.limit = d->act_limit;
    a.dtype = (int)d->dtype; a.out_dtype = (int)d->out_dtype;
    const uint64_t inner = a.in_out ? a.n_w() : a.K, outer = a.in_out ? a.K : a.n_w();
    if ((rc = take_stride(who, "ld_x", d->ld_x, a.K, a.K, &a.ld_x)) || (rc = take_stride(who, "ld_y", d->ld_y, a.N, a.N, &a.ld_y)) ||
        (rc = take_stride(who, "ld_w", d->ld_w, inner, inner, &a.ld_w)) ||
        (rc = take_stride(who, "w_stride", d->w_stride, outer * a.ld_w, (outer - 1) * a.ld_w + inner, &a.w_stride)))
        return rc;
    if (!h && d->rows == 0) return mlxs_fail(MLXS_E_ARG, "grouped: null handle");
    if (d->rows == 0) return MLXS_OK;
    if (!a.gather && !a.scatter) order_dev = nullptr;
    else if ((rc = check_ptr(who, "order_dev", order_dev, 4))) return rc;
    if ((rc = check_ptr(who, "x_dev", x_dev, 16)) || (rc = check_ptr(who, "w_dev", w_dev, 16)) || (rc = check_ptr(who, "y_dev", y_dev, 16)) ||
        ((offsets_dev || a.G != 1) && (rc = check_ptr(who, "offsets_dev", offsets_dev, 4))))
        return rc;
    if (a.x_rows == 0 || a.y_rows == 0) return mlxs_fail(MLXS_E_ARG, "grouped: x_rows %u, y_rows %u with %u rows", a.x_rows, a.y_rows, a.rows);
    if (!h) return mlxs_fail(MLXS_E_ARG, "grouped: null handle");
    a.x = x_dev; a.w = w_dev; a.y = y_dev; a.offsets = offsets_dev; a.order = order_dev;
    a.status = h->status; a.sm_count = h->sm_count;
    set_waits(a, h);
    DeviceGuard dev;
    cudaError_t e = dev.enter(h->cfg.device);
    if (e == cudaSuccess) e = launch_grouped(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return mlxs_fail(MLXS_E_CUDA, "grouped: %s", cudaGetErrorString(e));
    return MLXS_OK;
}

extern "C" int mlxs_moe_adapters(mlxs_moe* h, const mlxs_adapters_desc* d, const void* x_dev, const void* a_dev, const void* b_dev,
                                 const int32_t* ids_dev, const float* scales_dev, const int32_t* ranks_dev, const void* base_dev, void* y_dev,
                                 void* stream) {
    const char* who = "adapters";
    if (!d) return mlxs_fail(MLXS_E_ARG, "adapters: null descriptor");
    if (d->struct_size != sizeof *d) return mlxs_fail(MLXS_E_CONFIG, "adapters: struct_size %u, this library has %zu", d->struct_size, sizeof *d);
    int rc;
    if ((rc = check_types(who, d->dtype, d->out_dtype)) || (rc = check_dim(who, "n_in", d->n_in)) || (rc = check_dim(who, "n_out", d->n_out))) return rc;
    if (d->rank == 0 || d->rank % 8 || d->rank > MAX_RANK) return mlxs_fail(MLXS_E_CONFIG, "adapters: rank %u is not a multiple of 8 in 8..%u", d->rank, MAX_RANK);
    if (d->n_adapters == 0 || d->n_adapters > MAX_ROWS) return mlxs_fail(MLXS_E_CONFIG, "adapters: n_adapters %u outside 1..%u", d->n_adapters, MAX_ROWS);
    if (d->tokens > MAX_ROWS) return mlxs_fail(MLXS_E_TOO_MANY_TOKENS, "adapters: %u tokens, at most %u", d->tokens, MAX_ROWS);
    AdaptersArgs a{};
    a.K = d->n_in; a.N = d->n_out; a.R = d->rank; a.n_adapters = d->n_adapters; a.T = d->tokens;
    a.dtype = (int)d->dtype; a.out_dtype = (int)d->out_dtype;
    const uint64_t an = (uint64_t)a.R * a.K, bn = (uint64_t)a.N * a.R;
    if ((rc = take_stride(who, "ld_x", d->ld_x, a.K, a.K, &a.ld_x)) || (rc = take_stride(who, "ld_base", d->ld_base, a.N, a.N, &a.ld_base)) ||
        (rc = take_stride(who, "ld_y", d->ld_y, a.N, a.N, &a.ld_y)) || (rc = take_stride(who, "a_stride", d->a_stride, an, an, &a.a_stride)) ||
        (rc = take_stride(who, "b_stride", d->b_stride, bn, bn, &a.b_stride)))
        return rc;
    if (!h && d->tokens == 0) return mlxs_fail(MLXS_E_ARG, "adapters: null handle");
    if (d->tokens == 0) return MLXS_OK;
    if ((rc = check_ptr(who, "x_dev", x_dev, 16)) || (rc = check_ptr(who, "a_dev", a_dev, 16)) || (rc = check_ptr(who, "b_dev", b_dev, 16)) ||
        (rc = check_ptr(who, "ids_dev", ids_dev, 4)) || (rc = check_ptr(who, "y_dev", y_dev, 16)) ||
        (scales_dev && (rc = check_ptr(who, "scales_dev", scales_dev, 4))) || (ranks_dev && (rc = check_ptr(who, "ranks_dev", ranks_dev, 4))) ||
        (base_dev && (rc = check_ptr(who, "base_dev", base_dev, 16))))
        return rc;
    if (base_dev == y_dev && a.ld_base != a.ld_y) return mlxs_fail(MLXS_E_ARG, "adapters: in place with ld_base %zu and ld_y %zu", a.ld_base, a.ld_y);
    if (!h) return mlxs_fail(MLXS_E_ARG, "adapters: null handle");
    a.x = x_dev; a.a = a_dev; a.b = b_dev; a.base = base_dev; a.y = y_dev; a.ids = ids_dev; a.scales = scales_dev; a.ranks = ranks_dev;
    a.status = h->status; a.sm_count = h->sm_count;
    set_waits(a, h);
    DeviceGuard dev;
    cudaError_t e = dev.enter(h->cfg.device);
    if (e == cudaSuccess) e = launch_adapters(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return mlxs_fail(MLXS_E_CUDA, "adapters: %s", cudaGetErrorString(e));
    return MLXS_OK;
}

extern "C" int mlxs_moe_reserve_adapters(mlxs_moe* h) {
    if (!h) return mlxs_fail(MLXS_E_ARG, "reserve_adapters: null handle");
    if (!h->cfg.shared_expert) return mlxs_fail(MLXS_E_CONFIG, "reserve_adapters: the handle was created without a shared expert");
    if (h->sh_gate_up) return MLXS_OK;
    DeviceGuard dev;
    const cudaError_t e = dev.enter(h->cfg.device);
    if (e != cudaSuccess) return mlxs_fail(MLXS_E_CUDA, "reserve_adapters: %s", cudaGetErrorString(e));
    return h->alloc(&h->sh_gate_up, (size_t)h->cfg.max_tokens * 2 * h->cfg.inter * 4);
}

// what mlxs_moe_experts_adapted is given, before any device is touched
int mlxs_check_shared_adapters(const mlxs_shared_adapters* d, const int32_t* adapter_ids_dev) {
    const char* who = "experts_adapted";
    if (!d) return mlxs_fail(MLXS_E_ARG, "experts_adapted: null descriptor");
    if (d->struct_size != sizeof *d) return mlxs_fail(MLXS_E_CONFIG, "experts_adapted: struct_size %u, this library has %zu", d->struct_size, sizeof *d);
    if (d->rank == 0 || d->rank % 8 || d->rank > MAX_RANK) return mlxs_fail(MLXS_E_CONFIG, "experts_adapted: rank %u is not a multiple of 8 in 8..%u", d->rank, MAX_RANK);
    if (d->n_adapters == 0 || d->n_adapters > MAX_ROWS) return mlxs_fail(MLXS_E_CONFIG, "experts_adapted: n_adapters %u outside 1..%u", d->n_adapters, MAX_ROWS);
    const void* const pairs[3][2] = {{d->a1_dev, d->b1_dev}, {d->a3_dev, d->b3_dev}, {d->a2_dev, d->b2_dev}};
    const char* const names[3] = {"a1_dev / b1_dev", "a3_dev / b3_dev", "a2_dev / b2_dev"};
    int rc;
    for (int i = 0; i < 3; ++i) {
        if (!pairs[i][0] != !pairs[i][1]) return mlxs_fail(MLXS_E_ARG, "experts_adapted: one of %s is null", names[i]);
        for (int k = 0; k < 2; ++k)
            if (pairs[i][k] && (rc = check_ptr(who, names[i], pairs[i][k], 16))) return rc;
    }
    if ((rc = check_ptr(who, "adapter_ids_dev", adapter_ids_dev, 4)) || (d->scales_dev && (rc = check_ptr(who, "scales_dev", d->scales_dev, 4))) ||
        (d->ranks_dev && (rc = check_ptr(who, "ranks_dev", d->ranks_dev, 4))))
        return rc;
    return 0;
}

// The shared expert with adapters on its three linears: f32 gate and up rows, adapters on both, the activation, the down product, its adapters.
cudaError_t mlxs_run_shared_adapted(mlxs_moe* h, const LayerBank& L, const void* x_dev, uint32_t T, const mlxs_shared_adapters& d,
                                    const int32_t* adapter_ids_dev, float* out, cudaStream_t st) {
    const uint32_t H = h->cfg.hidden, I = h->cfg.inter;
    cudaError_t e;
    auto product = [&](const void* x, const void* w, uint32_t K, uint32_t N, float* y, size_t ld_y) {
        GroupedArgs a{};
        a.x = x; a.w = w; a.y = y; a.G = 1; a.K = K; a.N = N; a.rows = a.x_rows = a.y_rows = T; a.x_div = 1;
        a.dtype = DT_BF16; a.out_dtype = DT_F32; a.ld_x = a.ld_w = K; a.ld_y = ld_y; a.w_stride = (size_t)N * K;
        a.status = h->status; a.sm_count = h->sm_count;
        set_waits(a, h);
        return launch_grouped(a, st);
    };
    auto adapt = [&](const void* x, const void* A, const void* B, uint32_t K, uint32_t N, float* y, size_t ld_y) {
        if (!A) return cudaSuccess;
        AdaptersArgs a{};
        a.x = x; a.a = A; a.b = B; a.base = a.y = y; a.ids = adapter_ids_dev; a.scales = d.scales_dev; a.ranks = d.ranks_dev;
        a.K = K; a.N = N; a.R = d.rank; a.n_adapters = d.n_adapters; a.T = T; a.dtype = DT_BF16; a.out_dtype = DT_F32;
        a.ld_x = K; a.ld_base = a.ld_y = ld_y; a.a_stride = (size_t)d.rank * K; a.b_stride = (size_t)N * d.rank;
        a.status = h->status; a.sm_count = h->sm_count;
        set_waits(a, h);
        return launch_adapters(a, st);
    };
    const float limit = h->cfg.act == MLXS_ACT_SWIGLU_CLAMPED ? h->cfg.act_limit : 0.f;
    float* const gu = h->sh_gate_up;
    if ((e = product(x_dev, L.sh_w1, H, I, gu, 2 * (size_t)I)) != cudaSuccess || (e = product(x_dev, L.sh_w3, H, I, gu + I, 2 * (size_t)I)) != cudaSuccess ||
        (e = adapt(x_dev, d.a1_dev, d.b1_dev, H, I, gu, 2 * (size_t)I)) != cudaSuccess || (e = adapt(x_dev, d.a3_dev, d.b3_dev, H, I, gu + I, 2 * (size_t)I)) != cudaSuccess ||
        (e = launch_gate_up_act(gu, T, I, limit, h->sh_h, st)) != cudaSuccess || (e = product(h->sh_h, L.sh_w2, I, H, out, H)) != cudaSuccess)
        return e;
    return adapt(h->sh_h, d.a2_dev, d.b2_dev, I, H, out, H);
}
