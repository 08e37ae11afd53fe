// ll_moe_forward: argument checks, workspace layout and dispatch (kernels: moe_kernels.cuh).
#include <algorithm>

#include "moe_kernels.cuh"

using namespace llk;

namespace {

int check_desc(const char *op, const ll_moe_desc *d)
{
    if (!d) {
        llh::set_error("%s: null description", op);
        return LL_ERR_INVALID_ARG;
    }
    if (d->hidden < 1 || d->hidden > LL_MOE_MAX_DIM || d->inter < 1 || d->inter > LL_MOE_MAX_DIM) {
        llh::set_error("%s: hidden %d and inter %d must be in [1, %d]", op, d->hidden, d->inter, LL_MOE_MAX_DIM);
        return LL_ERR_BAD_DESC;
    }
    if (d->n_experts < 1 || d->n_experts > LL_MOE_MAX_EXPERTS || d->top_k < 1 || d->top_k > LL_MOE_MAX_TOPK ||
        d->top_k > d->n_experts) {
        llh::set_error("%s: n_experts %d must be in [1, %d] and top_k %d in [1, min(%d, n_experts)]", op, d->n_experts,
                       LL_MOE_MAX_EXPERTS, d->top_k, LL_MOE_MAX_TOPK);
        return LL_ERR_BAD_DESC;
    }
    if (d->act < LL_ACT_IDENTITY || d->act > LL_ACT_SILU || (d->gated != 0 && d->gated != 1) ||
        (d->renormalize != 0 && d->renormalize != 1)) {
        llh::set_error("%s: unknown activation %d, or gated / renormalize not 0 or 1", op, d->act);
        return LL_ERR_BAD_DESC;
    }
    if (d->wtype != LL_W_BF16 && d->wtype != LL_W_I8 && d->wtype != LL_W_F8) {
        llh::set_error("%s: expert weights must be bf16, int8 or e4m3 (type %d)", op, d->wtype);
        return LL_ERR_BAD_DESC;
    }
    if ((d->x_type != LL_T_F32 && d->x_type != LL_T_BF16 && d->x_type != LL_T_F16) ||
        (d->router_type != LL_T_F32 && d->router_type != LL_T_BF16)) {
        llh::set_error("%s: x must be fp32, bf16 or fp16 (type %d), the router fp32 or bf16 (type %d)", op, d->x_type,
                       d->router_type);
        return LL_ERR_BAD_DESC;
    }
    return LL_OK;
}

struct WorkLayout {
    size_t probs, hid, bytes;
    long long plane;
    int ld;
};

WorkLayout work_layout(const ll_moe_desc *d, int rows)
{
    WorkLayout w;
    const size_t n = (size_t)rows * d->top_k;
    w.probs = llh::round_up(4 * n, 256);
    w.hid = w.probs + llh::round_up(4 * n, 256);
    w.ld = moe_cols(d->inter, d->wtype == LL_W_BF16 ? 2 : 1);
    w.plane = (long long)(n * (size_t)w.ld);
    w.bytes = w.hid + (size_t)w.plane * 2 * (d->x_type == LL_T_F32 ? 3 : 2);
    return w;
}

}  // namespace

extern "C" {

int ll_moe_workspace_bytes(const ll_moe_desc *desc, int rows, size_t *bytes)
{
    static const char op[] = "ll_moe_workspace_bytes";
    LL_TRY(check_desc(op, desc));
    if (rows < 0 || rows > LL_MOE_MAX_ROWS || !bytes) {
        llh::set_error("%s: rows must be in [0, %d] (rows=%d) and bytes not null", op, LL_MOE_MAX_ROWS, rows);
        return LL_ERR_INVALID_ARG;
    }
    *bytes = std::max<size_t>(256, work_layout(desc, rows).bytes);
    return LL_OK;
}

int ll_moe_forward(const ll_moe_desc *d, const ll_moe_weights *w, const void *d_x, int64_t ldx, void *d_y, int64_t ldy,
                   int rows, int32_t *d_ids, float *d_probs, void *d_work, size_t work_bytes, void *stream)
{
    static const char op[] = "ll_moe_forward";
    LL_TRY(check_desc(op, d));
    if (ldx == 0)
        ldx = d->hidden;
    if (ldy == 0)
        ldy = d->hidden;
    if (rows < 0 || rows > LL_MOE_MAX_ROWS || ldx < d->hidden || ldy < d->hidden) {
        llh::set_error("%s: rows must be in [0, %d] and the strides at least hidden (rows=%d ldx=%lld ldy=%lld)", op,
                       LL_MOE_MAX_ROWS, rows, (long long)ldx, (long long)ldy);
        return LL_ERR_INVALID_ARG;
    }
    if (rows == 0)
        return LL_OK;
    const bool scaled = d->wtype != LL_W_BF16;
    if (!w || !d_x || !d_y || !d_work || !w->router || !w->gate || !w->down || (d->gated && !w->up) ||
        (scaled && (!w->gate_scale || !w->down_scale || (d->gated && !w->up_scale)))) {
        llh::set_error("%s: null pointer (a gated layer needs up, int8 and e4m3 experts their scales)", op);
        return LL_ERR_INVALID_ARG;
    }
    const WorkLayout wl = work_layout(d, rows);
    if (work_bytes < wl.bytes) {
        llh::set_error("%s: the workspace has %zu bytes, %zu are needed (ll_moe_workspace_bytes)", op, work_bytes,
                       wl.bytes);
        return LL_ERR_INVALID_ARG;
    }
    int dev = 0;
    unsigned *status = nullptr;
    LL_TRY(llh::ops_status_words(&dev, &status));
    const size_t xa = (size_t)type_bytes(d->x_type), wa = d->wtype == LL_W_BF16 ? 2 : 1;
    LL_TRY(llh::check_device_ptr(op, "x", d_x, dev, xa));
    LL_TRY(llh::check_device_ptr(op, "y", d_y, dev, xa));
    LL_TRY(llh::check_device_ptr(op, "the workspace", d_work, dev, 256));
    LL_TRY(llh::check_device_ptr(op, "router", w->router, dev, (size_t)type_bytes(d->router_type)));
    LL_TRY(llh::check_device_ptr(op, "gate", w->gate, dev, wa));
    LL_TRY(llh::check_device_ptr(op, "down", w->down, dev, wa));
    if (d->gated)
        LL_TRY(llh::check_device_ptr(op, "up", w->up, dev, wa));
    if (scaled) {
        LL_TRY(llh::check_device_ptr(op, "gate_scale", w->gate_scale, dev, 4));
        LL_TRY(llh::check_device_ptr(op, "down_scale", w->down_scale, dev, 4));
        if (d->gated)
            LL_TRY(llh::check_device_ptr(op, "up_scale", w->up_scale, dev, 4));
    }
    if (d_ids)
        LL_TRY(llh::check_device_ptr(op, "ids", d_ids, dev, 4));
    if (d_probs)
        LL_TRY(llh::check_device_ptr(op, "probs", d_probs, dev, 4));

    auto on16 = [](const void *p, long long row_bytes) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row_bytes % 16 == 0;
    };
    MoeParams p = {};
    p.x = d_x;
    p.ldx = ldx;
    p.y = d_y;
    p.ldy = ldy;
    p.rows = rows;
    p.hidden = d->hidden;
    p.inter = d->inter;
    p.experts = d->n_experts;
    p.top_k = d->top_k;
    p.act = d->act;
    p.gated = d->gated;
    p.renorm = d->renormalize;
    p.x_type = d->x_type;
    p.router = w->router;
    p.router_f32 = d->router_type == LL_T_F32;
    p.router_vec = on16(w->router, (long long)d->hidden * type_bytes(d->router_type));
    p.x_vec = on16(d_x, ldx * (long long)xa);
    p.wg = static_cast<const uint8_t *>(w->gate);
    p.wu = static_cast<const uint8_t *>(w->up);
    p.wd = static_cast<const uint8_t *>(w->down);
    p.sg = w->gate_scale;
    p.su = w->up_scale;
    p.sd = w->down_scale;
    // The widest copy that every weight row allows.
    auto grain = [](uintptr_t bits) { return (int)std::min<uintptr_t>(16, bits & (~bits + 1)); };
    p.up_grain = grain(reinterpret_cast<uintptr_t>(p.wg) | (d->gated ? reinterpret_cast<uintptr_t>(p.wu) : 0) |
                       (uintptr_t)d->hidden * wa);
    p.down_grain = grain(reinterpret_cast<uintptr_t>(p.wd) | (uintptr_t)d->inter * wa);
    uint8_t *work = static_cast<uint8_t *>(d_work);
    p.ids = reinterpret_cast<int *>(work);
    p.probs = reinterpret_cast<float *>(work + wl.probs);
    p.hid = reinterpret_cast<__nv_bfloat16 *>(work + wl.hid);
    p.hid_plane = wl.plane;
    p.hid_ld = wl.ld;
    p.user_ids = d_ids;
    p.user_probs = d_probs;
    p.status = status;
    p.wait_ns = llh::ops_wait_ns();
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return d->wtype == LL_W_BF16 ? launch_moe_bf16(p, dev, st)
           : d->wtype == LL_W_I8 ? launch_moe_i8(p, dev, st)
                                 : launch_moe_f8(p, dev, st);
}

}  // extern "C"
