// layer.cpp -- the entry points of the layer operators (helix_layer.h): checks,
// choice of the kernel, launches. As in dispatch.cpp every check comes before the
// first launch, and nothing is allocated, synchronized or waited for.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>
#include <utility>
#include <vector>

#include "helix/helix_layer.h"
#include "helix_internal.h"
#include "../kernels/layer_params.h"

using helix::rt::set_error;

namespace {

const char* const kTags[] = {"f32", "f16", "bf16"};   // by helix_dtype
const size_t kBytes[] = {4, 2, 2};

bool dtype_ok(int32_t t) { return t == HELIX_F32 || t == HELIX_F16 || t == HELIX_BF16; }

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Bad {
    helix_status st;
    std::string why;
};

void need(bool ok, const char* why, helix_status st = HELIX_ERR_INVALID_ARG) {
    if (!ok) throw Bad{st, why};
}

// A matrix of `rows` rows of `dim` elements of `es` bytes, `ld` apart: present,
// aligned to its elements, and with rows that do not overlap where it is written.
void matrix(const char* name, const void* p, long long rows, long long dim, long long ld, size_t es, bool written) {
    const std::string n = name;
    if (!p) throw Bad{HELIX_ERR_INVALID_ARG, n + " is NULL"};
    if (!aligned(p, es)) throw Bad{HELIX_ERR_INVALID_ARG, n + " is not aligned to its elements"};
    if (ld < 0 || (written && rows > 1 && ld < dim))
        throw Bad{HELIX_ERR_INVALID_ARG, n + (written ? ": rows overlap" : ": negative stride")};
}

// The current device is the context's while it lives.
class OnDevice {
public:
    explicit OnDevice(int device) : device_(device) {
        (void)hipGetDevice(&prev_);
        if (prev_ != device_ && hipSetDevice(device_) != hipSuccess) {
            (void)hipGetLastError();
            throw Bad{HELIX_ERR_NO_DEVICE, "hipSetDevice failed"};
        }
    }
    ~OnDevice() {
        if (prev_ >= 0 && prev_ != device_) (void)hipSetDevice(prev_);
    }

private:
    int device_, prev_ = -1;
};

hipFunction_t kernel(const helix_ctx* ctx, const std::string& name) {
    need(ctx->module != nullptr, "context has no device (host-only context)", HELIX_ERR_NO_DEVICE);
    const auto it = ctx->kernels.find(name);
    if (it == ctx->kernels.end()) throw Bad{HELIX_ERR_PIPELINE, "kernel " + name + " is not in the code object"};
    return it->second;
}

void launch_args(hipFunction_t f, void* stream, unsigned gx, unsigned gy, unsigned threads, void** args) {
    const hipError_t e = hipModuleLaunchKernel(f, gx, gy, 1, threads, 1, 1, 0, static_cast<hipStream_t>(stream), args,
                                               nullptr);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        throw Bad{HELIX_ERR_PIPELINE, std::string("kernel launch failed: ") + hipGetErrorString(e)};
    }
}

template <typename P>
void launch(hipFunction_t f, void* stream, unsigned gx, unsigned gy, unsigned threads, P& params) {
    void* args[] = {&params};
    launch_args(f, stream, gx, gy, threads, args);
}

// A launch counts its threads along x in 32 bits, and one of more begins with as few as the lowest 32 bits say, without
// an error: what may be more is launched in slices.
constexpr long long most_groups(int threads) { return ((1LL << 32) - 1) / threads; }

unsigned grid(long long n, int threads) {
    need(n <= most_groups(threads), "launch grid exceeds 2^32 threads");
    return (unsigned)n;
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// p, if there is one, `elements` of `size` bytes on.
template <typename T>
void advance(T*& p, long long elements, size_t size) {
    if (p) p = (T*)((uintptr_t)p + elements * (long long)size);
}

// Runs an entry point's body: no exception leaves it.
template <typename F>
helix_status entry(helix_ctx* ctx, F&& body) {
    try {
        body();
        return HELIX_OK;
    } catch (const Bad& b) {
        set_error(ctx, b.why);
        return b.st;
    } catch (const std::exception& e) {
        set_error(ctx, e.what());
        return HELIX_ERR_PIPELINE;
    }
}

constexpr int kNormThreads = 256;

// Kernel of rows of dim channels that are read once: "_w" + the chunks of 512 a wave holds, where `wave`, or "_g" + those of
// 2048 a workgroup does; empty: the forms that read a row twice.
std::string norm_form(long long dim, bool wave) {
    const long long chunks = ceil_div(dim, wave ? 512 : 2048);
    for (const int n : {1, 2, 3, 4, 6, 8})
        if (chunks <= n) return (wave ? "_w" : "_g") + std::to_string(n);
    return "";
}

void norm(helix_ctx* ctx, void* stream, const helix_norm_args* a, bool quantize) {
    need(ctx && a, "NULL context or arguments");
    need(a->rows >= 0 && a->dim >= 1 && a->dim <= HELIX_LAYER_MAX_DIM, "rows or dim out of range",
         HELIX_ERR_UNSUPPORTED_SHAPE);
    need(dtype_ok(a->io_dtype), "io_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
    if (a->rows == 0) return;   // an empty tensor may have no address
    if (quantize) {
        need(!a->weight && !a->rstd && !a->y, "quantisation takes no weight, rstd or y");
        need(a->q != nullptr, "q is NULL");
    } else {
        need(a->weight_dtype == HELIX_F32 || a->weight_dtype == a->io_dtype,
             "weight_dtype is neither HELIX_F32 nor io_dtype");
        need(!a->y != !a->q, "exactly one of y and q is wanted");
        need(std::isfinite(a->eps) && a->eps >= 0, "eps is negative or not finite");
    }
    const size_t es = kBytes[a->io_dtype];
    const long long blocks = ceil_div(a->dim, HELIX_FP8_BLOCK);
    matrix("x", a->x, a->rows, a->dim, a->ld_x, es, false);
    if (a->residual) matrix("residual", a->residual, a->rows, a->dim, a->ld_residual, es, false);
    if (!quantize) matrix("weight", a->weight, 1, a->dim, 0, kBytes[a->weight_dtype], false);
    if (a->h) matrix("h", a->h, a->rows, a->dim, a->ld_h, es, true);
    if (a->y) matrix("y", a->y, a->rows, a->dim, a->ld_y, es, true);
    if (a->q) {
        matrix("q", a->q, a->rows, a->dim, a->ld_q, 1, true);
        matrix("scale", a->scale, a->rows, blocks, a->ld_scale, 1, true);
    }
    need(aligned(a->rstd, 4), "rstd is not aligned to its elements");

    HelixNormParams p{};
    p.x = a->x;
    p.residual = a->residual;
    p.weight = a->weight;
    p.h = a->h;
    p.y = a->y;
    p.q = static_cast<uint8_t*>(a->q);
    p.scale = static_cast<uint8_t*>(a->scale);
    p.rstd = a->rstd;
    p.ld_x = a->ld_x;
    p.ld_residual = a->ld_residual;
    p.ld_h = a->ld_h;
    p.ld_y = a->ld_y;
    p.ld_q = a->ld_q;
    p.ld_scale = a->ld_scale;
    p.rows = a->rows;
    p.dim = a->dim;
    p.w_f32 = a->weight_dtype == HELIX_F32;
    p.eps = a->eps;
    // A wave each (four to a workgroup) where they give every CU four: 8192 rows of 512 and of 1024 6.8 and 10.9 us, as
    // workgroups 12.3 and 13.8; 128 and 512 rows of 2048 4.0 and 4.3 us, as workgroups 3.4 and 3.9.
    const std::string form = norm_form(a->dim, a->dim <= 4 * 512 && a->rows >= 4 * 256);
    const int each = form[0] && form[1] == 'w' ? 4 : 1;   // rows of a workgroup
    need(ceil_div(a->rows, each) <= 0x7fffffffLL, "launch grid exceeds 2^31 workgroups");
    const hipFunction_t f = kernel(ctx, std::string("helix_norm_") + kTags[a->io_dtype] + form);
    const OnDevice on(ctx->device);
    const long long most = each * most_groups(kNormThreads);
    for (long long left = a->rows; left > 0; left -= most) {
        p.rows = std::min(left, most);
        launch(f, stream, grid(ceil_div(p.rows, each), kNormThreads), 1, kNormThreads, p);
        if (left <= most) break;
        advance(p.x, most * p.ld_x, es);
        advance(p.residual, most * p.ld_residual, es);
        advance(p.h, most * p.ld_h, es);
        advance(p.y, most * p.ld_y, es);
        advance(p.q, most * p.ld_q, 1);
        advance(p.scale, most * p.ld_scale, 1);
        advance(p.rstd, most, sizeof(float));
    }
}

// Whether the backward pass gives a row to a wave: up to two chunks of 512, more would not fit in its registers with their
// sums (512 rows of 1024 8.0 us, as workgroups 16.6; 32768 of them 53 and 78).
bool norm_waves(long long dim) { return dim <= 2 * 512; }

// Parts that dweight's rows are summed in, a workgroup's each: two for every CU, of four steps at least.
long long norm_parts(long long rows, long long dim) {
    return std::max(1LL, std::min(2 * 256LL, rows / (norm_waves(dim) ? 16 : 4)));
}

}  // namespace

extern "C" helix_status helix_norm_encode(helix_ctx* ctx, void* stream, const helix_norm_args* args) {
    return entry(ctx, [&] { norm(ctx, stream, args, false); });
}

extern "C" helix_status helix_quantize_fp8_encode(helix_ctx* ctx, void* stream, const helix_norm_args* args) {
    return entry(ctx, [&] { norm(ctx, stream, args, true); });
}

extern "C" size_t helix_norm_backward_scratch_size(const helix_norm_backward_args* a) {
    if (!a || !a->dweight || a->rows <= 0 || a->dim <= 0) return 0;
    return (size_t)norm_parts(a->rows, a->dim) * a->dim * sizeof(float);
}

extern "C" helix_status helix_norm_backward_encode(helix_ctx* ctx, void* stream, const helix_norm_backward_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        need(a->rows >= 0 && a->dim >= 1 && a->dim <= HELIX_LAYER_MAX_DIM, "rows or dim out of range",
             HELIX_ERR_UNSUPPORTED_SHAPE);
        need(dtype_ok(a->io_dtype), "io_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
        need(a->weight_dtype == HELIX_F32 || a->weight_dtype == a->io_dtype,
             "weight_dtype is neither HELIX_F32 nor io_dtype");
        need(a->reserved == 0, "reserved is not 0");
        need(aligned(a->dweight, 4), "dweight is not aligned to its elements");
        const size_t es = kBytes[a->io_dtype];
        if (a->rows) {
            matrix("dy", a->dy, a->rows, a->dim, a->ld_dy, es, false);
            matrix("h", a->h, a->rows, a->dim, a->ld_h, es, false);
            matrix("weight", a->weight, 1, a->dim, 0, kBytes[a->weight_dtype], false);
            matrix("rstd", a->rstd, 1, a->rows, 0, 4, false);
            if (a->dh) matrix("dh", a->dh, a->rows, a->dim, a->ld_dh, es, false);
            matrix("dx", a->dx, a->rows, a->dim, a->ld_dx, es, true);
            const size_t want = helix_norm_backward_scratch_size(a);
            need(want == 0 || (a->scratch && a->scratch_bytes >= want),
                 "scratch smaller than helix_norm_backward_scratch_size()", HELIX_ERR_SCRATCH_TOO_SMALL);
            need(aligned(a->scratch, 16), "scratch is not 16-byte aligned");
        } else if (!a->dweight) {
            return;
        }
        HelixNormBwdParams p{};
        p.dy = a->dy;
        p.h = a->h;
        p.weight = a->weight;
        p.rstd = a->rstd;
        p.dh = a->dh;
        p.dx = a->dx;
        p.dweight = a->dweight;
        p.part = static_cast<float*>(a->scratch);
        p.ld_dy = a->ld_dy;
        p.ld_h = a->ld_h;
        p.ld_dh = a->ld_dh;
        p.ld_dx = a->ld_dx;
        p.rows = a->rows;
        p.dim = a->dim;
        p.w_f32 = a->weight_dtype == HELIX_F32;
        p.parts = a->rows ? (int)norm_parts(a->rows, a->dim) : 0;   // no rows: dweight is 0
        p.part_rows = p.parts ? ceil_div(a->rows, p.parts) : 0;
        const std::string tag = kTags[a->io_dtype];
        const std::string form = norm_form(a->dim, norm_waves(a->dim));
        const unsigned gx = a->rows && form.empty() ? grid(a->rows, kNormThreads) : (unsigned)p.parts;
        const unsigned gc = (unsigned)ceil_div(a->dim, kNormThreads), gd = (unsigned)ceil_div(a->dim, 32);
        const hipFunction_t dx = kernel(ctx, "helix_norm_bwd_" + tag + form), part = kernel(ctx, "helix_norm_dw_part_" + tag),
                            dw = kernel(ctx, "helix_norm_dw");
        const OnDevice on(ctx->device);
        if (a->rows && form.empty()) {   // dweight first: dx may be dy
            if (p.dweight) launch(part, stream, gc, (unsigned)p.parts, kNormThreads, p);
            launch(dx, stream, gx, 1, kNormThreads, p);
        } else if (a->rows) {
            launch(dx, stream, gx, 1, kNormThreads, p);
        }
        if (p.dweight) launch(dw, stream, gd, 1, 1024, p);
    });
}

namespace {

// Lanes and vectors of eight of a group of `width` channels (kernels/group_norm.hip): the least that hold it. 8192 rows of 4096
// channels with a gate in bf16, us with these | the next ones, forward and backward: groups of 64 39 | 71, 78 | 105; of 1024
// (two vectors a lane, or a workgroup) 35 | 64, 93 | 103; of 2048 (a workgroup) 38 | 59, 77 | 131.
struct GroupForm {
    int lanes = 256, vectors = 4;
    std::string name() const { return "_l" + std::to_string(lanes) + "_" + std::to_string(vectors); }
};
const GroupForm kGroupForms[] = {{4, 1}, {8, 1}, {16, 1}, {32, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {256, 4}};
GroupForm group_form(int width) {
    for (const GroupForm& f : kGroupForms)
        if (width <= 8 * f.lanes * f.vectors) return f;
    return {};
}

bool group_shape(long long rows, int dim, int groups, int io, int weight, int act) {
    need(rows >= 0 && dim >= 1 && dim <= HELIX_LAYER_MAX_DIM, "rows or dim out of range", HELIX_ERR_UNSUPPORTED_SHAPE);
    need(groups >= 1 && dim % groups == 0 && dim / groups <= HELIX_GROUP_NORM_MAX_GROUP,
         "groups does not divide dim, or its groups are too wide", HELIX_ERR_UNSUPPORTED_SHAPE);
    need(dtype_ok(io), "io_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
    need(weight == HELIX_F32 || weight == io, "weight_dtype is neither HELIX_F32 nor io_dtype");
    need(act == HELIX_ACT_NONE || act == HELIX_ACT_SILU || act == HELIX_ACT_SIGMOID, "activation is no helix_activation");
    return rows > 0;
}

// How the backward pass of a group norm is spread.
struct GroupBwdPlan {
    GroupForm form;
    int group_slots = 1, row_slots = 1;
    long long gx = 0, parts = 0;   // workgroups along the groups and along the rows
};
// A workgroup has as many groups side by side as there are, up to its room, and rows in what is left of it. Along the
// rows four workgroups a CU in all (32768 rows of 80 groups of 64, with a gate, bf16: two 448 us, four 370, eight 372), of two
// rows a slot at least (256 rows of 64 groups of 64: of one 12.4 us, of two 11.2, of four 13.0).
GroupBwdPlan group_bwd_plan(long long rows, int dim, int groups) {
    GroupBwdPlan p;
    p.form = group_form(dim / groups);
    const int room = kNormThreads / p.form.lanes;
    while (p.group_slots < room && p.group_slots < groups) p.group_slots *= 2;
    p.row_slots = room / p.group_slots;
    p.gx = ceil_div(groups, p.group_slots);
    p.parts = std::max(1LL, std::min(ceil_div(4 * 256, p.gx), rows / (2 * p.row_slots)));
    return p;
}

}  // namespace

extern "C" helix_status helix_group_norm_encode(helix_ctx* ctx, void* stream, const helix_group_norm_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        if (!group_shape(a->rows, a->dim, a->groups, a->io_dtype, a->weight_dtype, a->activation)) return;
        need(!a->y != !a->q, "exactly one of y and q is wanted");
        need(std::isfinite(a->eps) && a->eps >= 0, "eps is negative or not finite");
        const int width = a->dim / a->groups;
        const bool line_up = width % 128 == 0 || ((width == 32 || width == 64) && a->dim % 128 == 0);
        need(!a->q || line_up || a->dim <= HELIX_GROUP_NORM_MAX_ROW, "dim too large for 8 bits in these groups",
             HELIX_ERR_UNSUPPORTED_SHAPE);
        const size_t es = kBytes[a->io_dtype], ws = kBytes[a->weight_dtype];
        matrix("x", a->x, a->rows, a->dim, a->ld_x, es, false);
        matrix("weight", a->weight, 1, a->dim, 0, ws, false);
        if (a->bias) matrix("bias", a->bias, 1, a->dim, 0, ws, false);
        if (a->gate) matrix("gate", a->gate, a->rows, a->dim, a->ld_gate, es, false);
        if (a->y) matrix("y", a->y, a->rows, a->dim, a->ld_y, es, true);
        if (a->q) {
            matrix("q", a->q, a->rows, a->dim, a->ld_q, 1, true);
            matrix("scale", a->scale, a->rows, ceil_div(a->dim, HELIX_FP8_BLOCK), a->ld_scale, 1, true);
        }
        need(aligned(a->mean, 4) && aligned(a->rstd, 4), "mean or rstd is not aligned to its elements");
        HelixGroupNormParams p{};
        p.x = a->x;
        p.weight = a->weight;
        p.bias = a->bias;
        p.gate = a->gate;
        p.y = a->y;
        p.q = static_cast<uint8_t*>(a->q);
        p.scale = static_cast<uint8_t*>(a->scale);
        p.mean = a->mean;
        p.rstd = a->rstd;
        p.ld_x = a->ld_x;
        p.ld_gate = a->ld_gate;
        p.ld_y = a->ld_y;
        p.ld_q = a->ld_q;
        p.ld_scale = a->ld_scale;
        p.dim = a->dim;
        p.groups = a->groups;
        p.width = width;
        p.w_f32 = a->weight_dtype == HELIX_F32;
        p.act = a->activation;
        p.eps = a->eps;
        const GroupForm form = group_form(width);
        const bool any = a->q && !line_up;
        const hipFunction_t f = kernel(ctx, std::string(a->q ? "helix_group_norm_fp8_" : "helix_group_norm_") +
                                                kTags[a->io_dtype] + (any ? "_any" : form.name()));
        const int units = kNormThreads / form.lanes;   // of a workgroup
        // Units of a launch stay below 2^31 and its threads below 2^32.
        const long long groups = any ? 1 : a->groups, each = any ? 1 : units;
        const long long most = std::min((1LL << 31) - each, each * most_groups(kNormThreads)) / groups;
        const OnDevice on(ctx->device);
        for (long long left = a->rows; left > 0; left -= most) {
            p.rows = std::min(left, most);
            launch(f, stream, grid(ceil_div(p.rows * groups, each), kNormThreads), 1, kNormThreads, p);
            if (left <= most) break;
            advance(p.x, most * p.ld_x, es);
            advance(p.gate, most * p.ld_gate, es);
            advance(p.y, most * p.ld_y, es);
            advance(p.q, most * p.ld_q, 1);
            advance(p.scale, most * p.ld_scale, 1);
            advance(p.mean, most * p.groups, sizeof(float));
            advance(p.rstd, most * p.groups, sizeof(float));
        }
    });
}

extern "C" size_t helix_group_norm_backward_scratch_size(const helix_group_norm_backward_args* a) {
    if (!a || (!a->dweight && !a->dbias) || a->rows <= 0 || a->dim <= 0 || a->groups <= 0 || a->dim % a->groups) return 0;
    const GroupBwdPlan plan = group_bwd_plan(a->rows, a->dim, a->groups);
    return (size_t)plan.parts * plan.row_slots * 2 * a->dim * sizeof(float);
}

extern "C" helix_status helix_group_norm_backward_encode(helix_ctx* ctx, void* stream,
                                                         const helix_group_norm_backward_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        const bool some = group_shape(a->rows, a->dim, a->groups, a->io_dtype, a->weight_dtype, a->activation);
        need(a->reserved == 0, "reserved is not 0");
        need(aligned(a->dweight, 4) && aligned(a->dbias, 4), "dweight or dbias is not aligned to its elements");
        const bool sums = a->dweight || a->dbias;
        if (!some && !sums) return;
        const size_t es = kBytes[a->io_dtype], ws = kBytes[a->weight_dtype];
        if (some) {
            matrix("dy", a->dy, a->rows, a->dim, a->ld_dy, es, false);
            matrix("x", a->x, a->rows, a->dim, a->ld_x, es, false);
            matrix("weight", a->weight, 1, a->dim, 0, ws, false);
            if (a->bias) matrix("bias", a->bias, 1, a->dim, 0, ws, false);
            if (a->gate) matrix("gate", a->gate, a->rows, a->dim, a->ld_gate, es, false);
            need(!a->gate == !a->dgate, "dgate is wanted where there is a gate, and there alone");
            matrix("mean", a->mean, a->rows, a->groups, a->groups, 4, false);
            matrix("rstd", a->rstd, a->rows, a->groups, a->groups, 4, false);
            matrix("dx", a->dx, a->rows, a->dim, a->ld_dx, es, true);
            if (a->dgate) matrix("dgate", a->dgate, a->rows, a->dim, a->ld_dgate, es, true);
            const size_t want = helix_group_norm_backward_scratch_size(a);
            need(want == 0 || (a->scratch && a->scratch_bytes >= want),
                 "scratch smaller than helix_group_norm_backward_scratch_size()", HELIX_ERR_SCRATCH_TOO_SMALL);
            need(aligned(a->scratch, 16), "scratch is not 16-byte aligned");
        }
        const GroupBwdPlan plan = group_bwd_plan(a->rows, a->dim, a->groups);
        HelixGroupNormBwdParams p{};
        p.dy = a->dy;
        p.x = a->x;
        p.weight = a->weight;
        p.bias = a->bias;
        p.gate = a->gate;
        p.mean = a->mean;
        p.rstd = a->rstd;
        p.dx = a->dx;
        p.dgate = a->dgate;
        p.dweight = a->dweight;
        p.dbias = a->dbias;
        p.part = sums ? static_cast<float*>(a->scratch) : nullptr;
        p.ld_dy = a->ld_dy;
        p.ld_x = a->ld_x;
        p.ld_gate = a->ld_gate;
        p.ld_dx = a->ld_dx;
        p.ld_dgate = a->ld_dgate;
        p.rows = a->rows;
        p.part_rows = some ? ceil_div(a->rows, plan.parts) : 0;
        p.dim = a->dim;
        p.groups = a->groups;
        p.width = a->dim / a->groups;
        p.w_f32 = a->weight_dtype == HELIX_F32;
        p.act = a->activation;
        p.group_slots = plan.group_slots;
        p.parts = some ? (int)(plan.parts * plan.row_slots) : 0;   // no rows: the sums are 0
        const hipFunction_t f = kernel(ctx, std::string("helix_group_norm_bwd_") + kTags[a->io_dtype] + plan.form.name()),
                            dw = kernel(ctx, "helix_group_norm_dw");
        const unsigned gd = (unsigned)ceil_div(2LL * a->dim, 32);
        const OnDevice on(ctx->device);
        if (some) launch(f, stream, grid(plan.gx, kNormThreads), (unsigned)plan.parts, kNormThreads, p);
        if (sums) launch(dw, stream, gd, 1, 1024, p);
    });
}

namespace {

// How a product is computed (kernels/matmul_fp8.hip).
struct MatmulPlan {
    std::string kernel = "_blocks";
    int rows = 0, waves = 8;                      // > 0: rows of a that a workgroup takes at once, and its waves
    int bm = 0, bn = 0, per_cu = 1;               // > 0: tiles
    int parts = 1, part_blocks = 0;               // of the sum, of which each tile has a workgroup each
    size_t pitch = 0, a_bytes = 0, b_bytes = 0;   // copies of the scales, in scratch
    size_t part_bytes = 0;                        // and the parts, after them
    size_t bytes() const { return a_bytes + b_bytes + part_bytes; }
};

struct Tiling {
    const char* kernel;
    int bm, bn, per_cu;
    double step, tile;   // us of a step of 128 and of the rest of a tile, with every CU at work
};
// Fitted to 8192 x 8192 x 8192, 8192 x 10304 x 2048 and 32768 x 2560 x 5120: the large tiles take 20e-6 us per element
// and step, the small ones up to 33e-6, but waste less of a last round. Of one or two rounds it says too little (2871 x
// 5183 x 2560: 36 us, measured 48).
const Tiling kTilings[] = {
    {"_t88", 256, 256, 1, 1.38, 6.4}, {"_t86", 192, 256, 1, 1.04, 6.4}, {"_t84", 128, 256, 1, 0.93, 2.2},
    {"_t44", 128, 128, 2, 1.10, 1.5}, {"_t42", 64, 128, 2, 0.75, 1.2},
};
// A step of a workgroup that has a CU to itself: the way of a load, which goes one and a half steps ahead. And a launch.
constexpr double kLoneStep = 0.36, kLaunch = 2.5;

MatmulPlan matmul_plan(const helix_matmul_fp8_args& a) {
    MatmulPlan p;
    const long long m = a.m, n = a.n, k = a.k, blocks = ceil_div(k, HELIX_FP8_BLOCK);
    double best = 1e30;
    // Rows: 4 us and 8 TB/s of what workgroups read, b once for each 64 rows of a and a for each 16 of b (17, 33 and 67 rows
    // of 2048 x 4096: 7.5, 9.8, 11.6 us; of 10304 x 2048: 9.6, 13.0, 23.0).
    if (m <= 128) {
        const long long tiles = ceil_div(m, 16), ny = ceil_div(tiles, 4), each = ceil_div(tiles, ny);
        p.rows = (int)(16 * each);
        p.kernel = "_r" + std::to_string(each);
        // Four waves where workgroups are many: eight and four for one row of 2048 x 8192, 16384 and 32768 5.6 and 5.4, 9.5
        // and 8.3, 16.8 and 13.2 us, of 1024 x 10304 5.2 and 4.5, of 4096 x 10304 11.4 and 11.3 (16 rows 15.2 and 15.7); below
        // within 0.2 us of each other (2048 x 4096: 3.9 and 3.9; 4096 x 4096: 6.0 and 6.2).
        if (each == 1 && n >= 8192) p.kernel = "_r1w4", p.waves = 4;
        best = 4 + (double)ceil_div(n, 16) * k * 16 * (ny + tiles) / 8e6;
        if (m <= 16) return p;
    }
    // The tiles' loads and stores reach a tile's rows by 32-bit offsets, and their loop is four steps long at least. fp32
    // results do not come from its instruction.
    const long long reach = (1LL << 31) / 256 / 2;
    if (a.out_dtype == HELIX_F32 || blocks < 4 || a.ld_a >= reach || a.ld_b >= reach || a.ld_c >= reach / 2 ||
        a.ld_a_scale >= reach || a.ld_b_scale >= reach || n >= reach / 4)
        return p;
    const MatmulPlan rows = p;
    for (const Tiling& t : kTilings) {
        const long long tiles = ceil_div(m, t.bm) * ceil_div(n, t.bn), slots = 256 * t.per_cu;
        // The sum in parts (groups of four blocks) where small tiles leave CUs without work: another launch adds them up
        // (67 and 256 rows of 2048 x 4096 in eight parts 12.5 and 21.5 us, in one 13.0 and 15.1; 67 of 2560 x 5120 in six
        // 15.0, in one 17.6).
        const long long most = t.bn > 128 ? 1 : std::max(1LL, slots / tiles);
        for (long long each = blocks; each >= 4; each = each == blocks ? (blocks - 1) / 4 * 4 : each - 4) {
            const long long rest = blocks % each, s = blocks / each + (rest >= 4), steps = rest && rest < 4 ? each + rest : each;
            if (s > most) break;
            const double busy = std::min(1.0, (double)tiles * s / slots);
            double us = kLaunch + ceil_div(tiles, slots) * (steps * std::max(t.step * busy, kLoneStep) + t.tile);
            if (s > 1) us += 5 + 4.0 * m * n * (s + 1) / 2e6;
            if (us >= best) continue;
            best = us;
            p = MatmulPlan{};
            p.kernel = std::string(t.kernel) + (s > 1 ? "p" : "");
            p.bm = t.bm;
            p.bn = t.bn;
            p.per_cu = t.per_cu;
            p.parts = (int)s;
            p.part_blocks = s > 1 ? (int)each : (int)blocks;
        }
    }
    if (!p.bm) return rows;
    auto up = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    p.pitch = (size_t)ceil_div(blocks, 4) * 4;
    // Scales are loaded as words of four.
    if (a.ld_a_scale % 4 || !aligned(a.a_scale, 4)) p.a_bytes = up((size_t)m * p.pitch);
    if (a.ld_b_scale % 4 || !aligned(a.b_scale, 4)) p.b_bytes = up((size_t)n * p.pitch);
    if (p.parts > 1) p.part_bytes = (size_t)p.parts * m * ((n + 3) & ~3LL) * 4;
    return p;
}

// 2^32 / d + 1: the high word of its product with x is x / d while x d is below 2^32 (d above 1).
unsigned reciprocal(unsigned d) { return d > 1 ? (unsigned)((1ULL << 32) / d + 1) : 0; }

}  // namespace

extern "C" size_t helix_matmul_fp8_scratch_size(const helix_matmul_fp8_args* a) {
    if (!a || a->m <= 0 || a->n <= 0 || a->k <= 0) return 0;
    const MatmulPlan p = matmul_plan(*a);
    return p.bytes();
}

extern "C" helix_status helix_matmul_fp8_encode(helix_ctx* ctx, void* stream, const helix_matmul_fp8_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        need(a->m >= 0 && a->n >= 0 && a->k >= 1 && a->k <= HELIX_LAYER_MAX_DIM, "m, n or k out of range",
             HELIX_ERR_UNSUPPORTED_SHAPE);
        need(dtype_ok(a->out_dtype), "out_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
        if (a->m == 0 || a->n == 0) return;
        const long long blocks = ceil_div(a->k, HELIX_FP8_BLOCK);
        matrix("a", a->a, a->m, a->k, a->ld_a, 16, false);
        matrix("b", a->b, a->n, a->k, a->ld_b, 16, false);
        matrix("a_scale", a->a_scale, a->m, blocks, a->ld_a_scale, 1, false);
        matrix("b_scale", a->b_scale, a->n, blocks, a->ld_b_scale, 1, false);
        matrix("c", a->c, a->m, a->n, a->ld_c, kBytes[a->out_dtype], true);
        need((a->m == 1 || a->ld_a % 16 == 0) && (a->n == 1 || a->ld_b % 16 == 0),
             "ld_a and ld_b have to be multiples of 16");
        const MatmulPlan plan = matmul_plan(*a);
        need(a->scratch_bytes >= plan.bytes() && (a->scratch || !plan.bytes()),
             "scratch smaller than helix_matmul_fp8_scratch_size()", HELIX_ERR_SCRATCH_TOO_SMALL);
        need(aligned(a->scratch, 16), "scratch is not 16-byte aligned");
        HelixMatmulParams p{};
        p.a = static_cast<const uint8_t*>(a->a);
        p.a_scale = static_cast<const uint8_t*>(a->a_scale);
        p.b = static_cast<const uint8_t*>(a->b);
        p.b_scale = static_cast<const uint8_t*>(a->b_scale);
        p.c = a->c;
        p.ld_a = a->ld_a;
        p.ld_a_scale = a->ld_a_scale;
        p.ld_b = a->n == 1 ? ceil_div(a->k, 16) * 16 : a->ld_b;   // a single row's may be anything
        p.ld_b_scale = a->ld_b_scale;
        p.ld_c = a->ld_c;
        p.m = a->m;
        p.n = a->n;
        p.k = a->k;
        const hipFunction_t f =
            kernel(ctx, plan.bm ? std::string("helix_matmul_fp8") + plan.kernel
                                : std::string("helix_matmul_fp8_") + kTags[a->out_dtype] + plan.kernel);
        if (plan.rows) {
            const unsigned gy = (unsigned)ceil_div(a->m, plan.rows);
            const OnDevice on(ctx->device);
            const int threads = 64 * plan.waves, most = (int)(16 * most_groups(threads));
            for (long long left = a->n; left > 0; left -= most) {
                p.n = (int)std::min<long long>(left, most);
                launch(f, stream, grid(ceil_div(p.n, 16), threads), gy, threads, p);
                if (left <= most) break;
                advance(p.b, most * p.ld_b, 1);
                advance(p.b_scale, most * p.ld_b_scale, 1);
                advance(p.c, most, kBytes[a->out_dtype]);
            }
            return;
        }
        if (!plan.bm) {
            const unsigned gx = grid(ceil_div(a->m, 64) * ceil_div(a->n, 128), 256);
            const OnDevice on(ctx->device);
            launch(f, stream, gx, 1, 256, p);
            return;
        }
        const long long mt = ceil_div(a->m, plan.bm), nt = ceil_div(a->n, plan.bn), tiles = mt * nt;
        need(tiles <= 0x7fffffffLL, "launch grid exceeds 2^31 workgroups");
        // Bands of 2048 rows, or of one row of tiles where c is so large that a band's number would not come out exactly.
        p.gm = std::max(1, 2048 / plan.bm);
        if (tiles * p.gm * nt >= (1LL << 32)) p.gm = 1;
        need(tiles * p.gm * nt < (1LL << 32), "m and n are too large", HELIX_ERR_UNSUPPORTED_SHAPE);
        p.band = (unsigned)(p.gm * nt);
        p.inv_band = reciprocal(p.band);
        p.inv_gm = reciprocal(p.gm);
        p.inv_rest = reciprocal((unsigned)(mt % p.gm));
        p.stride = (int)std::min<long long>(tiles, 256LL * plan.per_cu);
        p.f16 = a->out_dtype == HELIX_F16;
        const unsigned ga = grid(plan.a_bytes ? ceil_div((long long)a->m * plan.pitch, 256) : 0, 256),
                       gb = grid(plan.b_bytes ? ceil_div((long long)a->n * plan.pitch, 256) : 0, 256),
                       gj = grid(plan.parts > 1 ? ceil_div((long long)a->m * ceil_div(a->n, 4), 256) : 0, 256);
        const hipFunction_t copy = kernel(ctx, "helix_fp8_scales"),
                            join = kernel(ctx, std::string("helix_matmul_fp8_join_") + kTags[a->out_dtype]);
        const OnDevice on(ctx->device);
        auto repack = [&](const uint8_t*& scale, long long& ld, long long rows, uint8_t* to, unsigned gx) {
            int nb = (int)blocks, pitch = (int)plan.pitch;
            void* args[] = {&scale, &to, &ld, &rows, &nb, &pitch};
            launch_args(copy, stream, gx, 1, 256, args);
            scale = to;
            ld = pitch;
        };
        if (plan.a_bytes) repack(p.a_scale, p.ld_a_scale, a->m, static_cast<uint8_t*>(a->scratch), ga);
        if (plan.b_bytes) repack(p.b_scale, p.ld_b_scale, a->n, static_cast<uint8_t*>(a->scratch) + plan.a_bytes, gb);
        p.parts = plan.parts;
        p.part_blocks = plan.part_blocks;
        p.part = plan.parts > 1 ? reinterpret_cast<float*>(static_cast<uint8_t*>(a->scratch) + plan.a_bytes + plan.b_bytes) : nullptr;
        launch(f, stream, (unsigned)p.stride, (unsigned)plan.parts, 256, p);
        if (plan.parts == 1) return;
        launch(join, stream, gj, 1, 256, p);
    });
}

namespace {

constexpr int kScanThreads = 256;

// How the recurrence of a shape is cut (kernels/gated_scan.hip).
struct ScanPlan {
    int waves = 0;               // of a workgroup; 0: one thread walks all tokens of four channels
    int n_slab = 0, n_chunk = 1, n_group = 0;
    long long streams = 0;
    size_t part_at = 0, left_at = 0, bytes = 0;   // scratch: the ticket, then these
};

// run: tokens of a thread's run. As few tokens as one thread walks quickly, and
// rows so far apart that a wave's reach past 32-bit offsets, go token by token. Four
// waves where they hold the whole sequence, else eight: over 8192 tokens of 4096
// channels (bf16) chunks of 4, 8 and 16 waves took 67, 52 and 54 us, backward over 8 x
// 4096 tokens of 5120 channels 534, 419 and 422.
ScanPlan scan_plan(long long n_seq, long long n_tok, long long n_chan, int run, bool far) {
    ScanPlan p;
    if (n_seq <= 0 || n_tok < 0 || n_chan <= 0) return p;
    p.n_slab = (int)ceil_div(n_chan, 64);
    p.streams = n_seq * p.n_slab;
    if (n_tok <= HELIX_GS_STEPS || far) return p;
    p.waves = n_tok <= 4LL * run * 4 ? 4 : 8;
    p.n_chunk = (int)ceil_div(n_tok, 4LL * run * p.waves);
    p.n_group = (int)ceil_div(p.n_chunk, HELIX_GS_GROUP);
    if (p.n_chunk > 1) {
        p.part_at = 256;
        p.left_at = p.part_at + (size_t)p.streams * p.n_chunk * 64 * 8;
        p.bytes = p.left_at + (size_t)p.streams * p.n_group * 64 * 4;
    }
    return p;
}

// Whether a wave's rows (4 runs of 8 tokens at most, and one before them) reach
// beyond 2^29 bytes.
bool far_rows(long long tok, size_t es) { return tok >= (1LL << 29) / 33 / (long long)es; }

// Fills in a plan, and runs it: P is HelixGatedScanParams or its backward form, ahead(p, n) takes p n sequences on.
template <typename A, typename P, typename F>
void run_scan(helix_ctx* ctx, void* stream, const A& a, P& p, const char* name, int run, bool far, F&& ahead) {
    const ScanPlan plan = scan_plan(a.n_seq, a.n_tok, a.n_chan, run, far);
    need(plan.bytes == 0 || (a.scratch && a.scratch_bytes >= plan.bytes), "scratch smaller than its _scratch_size()",
         HELIX_ERR_SCRATCH_TOO_SMALL);
    need(aligned(a.scratch, 16), "scratch is not 16-byte aligned");
    p.n_tok = a.n_tok;
    p.n_chan = a.n_chan;
    p.n_slab = plan.n_slab;
    p.join = HelixGatedScanJoin{};
    p.join.n_chunk = plan.n_chunk;
    p.join.n_group = plan.n_group;
    const std::string base = std::string(name) + kTags[a.io_dtype] + (a.n_chan % 4 ? "_s" : "_v");   // (channels that come in fours, or not)
    const int threads = plan.waves ? 64 * plan.waves : kScanThreads;
    // Sequences of a launch.
    const long long most = plan.waves ? most_groups(threads) / ((long long)plan.n_slab * plan.n_chunk)
                                      : most_groups(threads) * threads / ceil_div(a.n_chan, 4);
    need(most > 0, "launch grid exceeds 2^32 threads");
    const hipFunction_t f = kernel(ctx, plan.waves ? base + "_w" + std::to_string(plan.waves) : base + "_steps");
    const hipFunction_t ff = plan.bytes ? kernel(ctx, "helix_gated_scan_fill") : nullptr;
    char* sc = static_cast<char*>(a.scratch);
    const OnDevice on(ctx->device);
    for (long long left = a.n_seq; left > 0; left -= most) {
        p.n_seq = (int)std::min(left, most);
        const ScanPlan slice = scan_plan(p.n_seq, a.n_tok, a.n_chan, run, far);
        if (slice.bytes) {
            p.join.ticket = reinterpret_cast<unsigned*>(sc);
            p.join.part = reinterpret_cast<unsigned long long*>(sc + slice.part_at);
            p.join.left = reinterpret_cast<unsigned*>(sc + slice.left_at);
            long long n = (long long)(slice.bytes / 16);
            void* args[] = {&sc, &n};
            launch_args(ff, stream, grid(ceil_div(n, kScanThreads), kScanThreads), 1, kScanThreads, args);
        }
        const long long groups = plan.waves ? slice.streams * plan.n_chunk : ceil_div(p.n_seq * ceil_div(a.n_chan, 4), kScanThreads);
        launch(f, stream, grid(groups, threads), 1, threads, p);
        if (left > most) ahead(p, most);
    }
}

template <typename A>
bool scan_shape(const A& a) {
    need(a.n_seq >= 0 && a.n_tok >= 0 && a.n_chan >= 0, "n_seq, n_tok or n_chan is negative",
         HELIX_ERR_UNSUPPORTED_SHAPE);
    need(dtype_ok(a.io_dtype), "io_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
    return a.n_seq && a.n_chan;
}

// A tensor (n_seq, n_tok, n_chan) with contiguous channels.
template <typename A>
void tokens(const char* name, const A& a, const void* p, long long seq, long long tok, bool written) {
    if (!a.n_tok) return;
    matrix(name, p, a.n_tok, a.n_chan, tok, kBytes[a.io_dtype], written);
    need(seq >= 0 && (!written || a.n_seq == 1 || seq >= a.n_chan), "sequences overlap or have a negative stride");
}

}  // namespace

extern "C" size_t helix_gated_scan_scratch_size(const helix_gated_scan_args* a) {
    return a ? scan_plan(a->n_seq, a->n_tok, a->n_chan, HELIX_GS_RUN, false).bytes : 0;
}

extern "C" helix_status helix_gated_scan_encode(helix_ctx* ctx, void* stream, const helix_gated_scan_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        if (!scan_shape(*a)) return;
        tokens("g", *a, a->g, a->seq_g, a->tok_g, false);
        tokens("v", *a, a->v, a->seq_v, a->tok_v, false);
        tokens("h", *a, a->h, a->seq_h, a->tok_h, true);
        need(aligned(a->h0, 4) && aligned(a->last, 4), "h0 or last is not aligned to its elements");
        HelixGatedScanParams p{};
        p.g = a->g;
        p.v = a->v;
        p.h0 = a->h0;
        p.h = a->h;
        p.last = a->last;
        p.seq_g = a->seq_g;
        p.tok_g = a->tok_g;
        p.seq_v = a->seq_v;
        p.tok_v = a->tok_v;
        p.seq_h = a->seq_h;
        p.tok_h = a->tok_h;
        const size_t es = kBytes[a->io_dtype];
        bool far = false;
        for (const long long tok : {(long long)a->tok_g, (long long)a->tok_v, (long long)a->tok_h}) far |= far_rows(tok, es);
        run_scan(ctx, stream, *a, p, "helix_gated_scan_", HELIX_GS_RUN, far, [&](HelixGatedScanParams& q, long long n) {
            advance(q.g, n * q.seq_g, es);
            advance(q.v, n * q.seq_v, es);
            advance(q.h, n * q.seq_h, es);
            advance(q.h0, n * a->n_chan, sizeof(float));
            advance(q.last, n * a->n_chan, sizeof(float));
        });
    });
}

extern "C" size_t helix_gated_scan_backward_scratch_size(const helix_gated_scan_backward_args* a) {
    return a ? scan_plan(a->n_seq, a->n_tok, a->n_chan, HELIX_GS_RUN_BWD, false).bytes : 0;
}

extern "C" helix_status helix_gated_scan_backward_encode(helix_ctx* ctx, void* stream,
                                                         const helix_gated_scan_backward_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        if (!scan_shape(*a)) return;
        tokens("dh", *a, a->dh, a->seq_dh, a->tok_dh, false);
        tokens("g", *a, a->g, a->seq_g, a->tok_g, false);
        tokens("v", *a, a->v, a->seq_v, a->tok_v, false);
        tokens("h", *a, a->h, a->seq_h, a->tok_h, false);
        tokens("dg", *a, a->dg, a->seq_dg, a->tok_dg, true);
        tokens("dv", *a, a->dv, a->seq_dv, a->tok_dv, true);
        need(aligned(a->h0, 4) && aligned(a->dh_last, 4) && aligned(a->dh0, 4),
             "h0, dh_last or dh0 is not aligned to its elements");
        HelixGatedScanBwdParams p{};
        p.dh = a->dh;
        p.g = a->g;
        p.v = a->v;
        p.h = a->h;
        p.h0 = a->h0;
        p.dh_last = a->dh_last;
        p.dg = a->dg;
        p.dv = a->dv;
        p.dh0 = a->dh0;
        p.seq_dh = a->seq_dh;
        p.tok_dh = a->tok_dh;
        p.seq_g = a->seq_g;
        p.tok_g = a->tok_g;
        p.seq_v = a->seq_v;
        p.tok_v = a->tok_v;
        p.seq_h = a->seq_h;
        p.tok_h = a->tok_h;
        p.seq_dg = a->seq_dg;
        p.tok_dg = a->tok_dg;
        p.seq_dv = a->seq_dv;
        p.tok_dv = a->tok_dv;
        const size_t es = kBytes[a->io_dtype];
        bool far = false;
        for (const long long tok : {(long long)a->tok_dh, (long long)a->tok_g, (long long)a->tok_v, (long long)a->tok_h, (long long)a->tok_dg, (long long)a->tok_dv}) far |= far_rows(tok, es);
        run_scan(ctx, stream, *a, p, "helix_gated_scan_bwd_", HELIX_GS_RUN_BWD, far, [&](HelixGatedScanBwdParams& q, long long n) {
            advance(q.dh, n * q.seq_dh, es);
            advance(q.g, n * q.seq_g, es);
            advance(q.v, n * q.seq_v, es);
            advance(q.h, n * q.seq_h, es);
            advance(q.dg, n * q.seq_dg, es);
            advance(q.dv, n * q.seq_dv, es);
            advance(q.h0, n * a->n_chan, sizeof(float));
            advance(q.dh_last, n * a->n_chan, sizeof(float));
            advance(q.dh0, n * a->n_chan, sizeof(float));
        });
    });
}

namespace {

constexpr int kDeltaThreads = 256, kDeltaPairThreads = 640;

// Elements of strides that do not overlap: each dimension's stride reaches past what the ones below it span.
bool disjoint(std::initializer_list<std::pair<long long, long long>> dims) {   // (size, stride)
    std::vector<std::pair<long long, long long>> d;   // (stride, size)
    for (const auto& x : dims)
        if (x.first > 1) d.push_back({x.second, x.first});
    std::sort(d.begin(), d.end());
    long long span = 1;
    for (const auto& x : d) {
        if (x.first < span) return false;
        span = x.first * (x.second - 1) + span;
    }
    return true;
}

// Gates (n_seq, n_tok, heads), fp32 with dense heads, at any distance of their tokens: the kernels' offsets in them are 64 bits.
void gates(const char* name, const float* p, long long n_tok, long long seq, long long tok) {
    if (!n_tok) return;
    const std::string n = name;
    if (!p) throw Bad{HELIX_ERR_INVALID_ARG, n + " is NULL"};
    if (!aligned(p, 4)) throw Bad{HELIX_ERR_INVALID_ARG, n + " is not aligned to its elements"};
    if (seq < 0 || tok < 0) throw Bad{HELIX_ERR_INVALID_ARG, n + ": negative stride"};
}

// A tensor (n_seq, n_tok, heads, width) with contiguous last dimension: present, aligned, and within the kernels' reach.
void heads(const char* name, const void* p, long long n_seq, long long n_tok, long long n_head, long long width, long long seq,
           long long tok, long long head, size_t es, bool written) {
    if (!n_tok) return;
    const std::string n = name;
    if (!p) throw Bad{HELIX_ERR_INVALID_ARG, n + " is NULL"};
    if (!aligned(p, es)) throw Bad{HELIX_ERR_INVALID_ARG, n + " is not aligned to its elements"};
    if (seq < 0 || tok < 0 || head < 0) throw Bad{HELIX_ERR_INVALID_ARG, n + ": negative stride"};
    if (n_tok > 1 && tok >= (1LL << 31) / 64 / (long long)es)
        throw Bad{HELIX_ERR_UNSUPPORTED_SHAPE, n + ": 64 tokens span 2^31 bytes or more"};
    if (written && !disjoint({{n_seq, seq}, {n_tok, tok}, {n_head, head}, {width, 1}}))
        throw Bad{HELIX_ERR_INVALID_ARG, n + ": elements overlap"};
}

// Checks of what both passes have; whether there is anything to do.
template <typename A>
bool delta_shape(const A& a) {
    need(a.n_seq >= 0 && a.n_tok >= 0 && a.n_qk_head >= 0 && a.n_head >= 0, "n_seq, n_tok, n_qk_head or n_head is negative",
         HELIX_ERR_UNSUPPORTED_SHAPE);
    need(a.n_key >= 1 && a.n_key <= HELIX_DELTA_MAX_KEY && a.n_val >= 1 && a.n_val <= HELIX_DELTA_MAX_VAL,
         "n_key or n_val out of range", HELIX_ERR_UNSUPPORTED_SHAPE);
    need(dtype_ok(a.io_dtype), "io_dtype is none of HELIX_F32, HELIX_F16 and HELIX_BF16");
    need(std::isfinite(a.scale), "scale is not finite");
    if (!a.n_seq || !a.n_head) return false;
    need((long long)a.n_seq * a.n_head < 1LL << 31, "n_seq * n_head out of range", HELIX_ERR_UNSUPPORTED_SHAPE);
    need(a.n_qk_head >= 1 && a.n_head % a.n_qk_head == 0, "n_qk_head does not divide n_head", HELIX_ERR_UNSUPPORTED_SHAPE);
    return true;
}

// Whether sizes are such as a call takes, of some heads (those that it refuses may be any here).
template <typename A>
bool delta_heads(const A& a) {
    return a.n_seq > 0 && a.n_head > 0 && a.n_tok >= 0 && a.n_key > 0 && a.n_key <= HELIX_DELTA_MAX_KEY && a.n_val > 0 &&
           a.n_val <= HELIX_DELTA_MAX_VAL && (long long)a.n_seq * a.n_head < 1LL << 31 && a.n_qk_head > 0 &&
           a.n_head % a.n_qk_head == 0;
}

int delta_keys(int n_key) { return n_key <= 64 ? 64 : 128; }   // of the kernels
// Type and keys of a kernel; "_s": for rows of 16 bits and an odd width (the steps go element by element anyway).
template <typename A>
std::string delta_form(const A& a, bool steps = false) {
    const bool odd = !steps && a.io_dtype != HELIX_F32 && ((a.n_key | a.n_val) & 1);
    return std::string(kTags[a.io_dtype]) + "_" + std::to_string(delta_keys(a.n_key)) + (odd ? "_s" : "");
}

// Columns of the state that a workgroup of the walks has: 32 where that still gives every CU a workgroup.
// (2048 tokens, bf16, 128 keys x 64, us with 16 | 32, forward and backward: 64 heads 96 | 108, 306 | 344; 128 heads
// 134 | 125, 550 | 498; 256 heads 322 | 259, 1070 | 923. fp32, 64 keys x 128: 32 heads 92 | 106, 279 | 311; 64 heads
// 140 | 123, 539 | 447.)
int delta_columns(long long heads, int n_val) { return n_val > 16 && heads * ceil_div(n_val, 32) >= 256 ? 32 : 16; }

// The most tokens that go one by one, by the workgroups that their kernel has. One by one a token costs 1.1 to 1.4 us where
// all of them run at once; a chunk costs about the same for 1 token as for 64, and more in fp32. Measured, us one by one | as a
// chunk, 128 keys: bf16, 64 workgroups, 4 tokens 9 | 14, 8 tokens 15 | 14; 256, 8 tokens 16 | 23, 12 tokens 22 | 23; 384,
// 16 tokens 29 | 31; 4096, 16 tokens 173 | 223, 24 tokens 247 | 226. fp32, 64 workgroups, 12 tokens 17 | 19, 16 tokens
// 22 | 19; 384, 32 tokens 46 | 43; 1024, 32 tokens 73 | 87, 64 tokens 132 | 98.
int delta_steps(long long heads, int n_val, int io) {
    const long long groups = heads * ceil_div(n_val, 64);
    return (io == HELIX_F32 ? 2 : 1) * (groups < 256 ? 6 : groups < 384 ? 10 : 16);
}

// Whether a long call goes in segments, and the walk of each takes along the kernel that forms the next one's operands: where
// walks leave CUs room for it (16 bits, at most three workgroups of 16 columns for two CUs) and there is less to form than to
// walk. Segments of 2048 chunks of heads at least, whose operands take as long as some launches. Measured, us in one piece |
// in segments, bf16: 8192 tokens of 64 heads of 128 x 64 349 | 317; of 96 heads 546 | 490; 32768 tokens of 32 heads of
// 128 x 128 1181 | 1045. f16: 486 | 476, 699 | 684, 1646 | 1470. Past the bounds: 104 heads of 128 x 64 bf16 572 | 536, f16
// 721 | 729; 112 heads 595 | 587, 747 | 773; 120 heads 616 | 620, 770 | 816; 128 heads of 128 x 32 547 | 530, 659 | 731; 192 of
// them 704 | 745, 919 | 983; 256 of 128 x 16 748 | 754, 930 | 1085: one bound for both types.
bool delta_ahead(long long heads, int columns, const helix_delta_rule_args& a) {
    return columns == 16 && a.io_dtype != HELIX_F32 && heads <= 96 && heads * ceil_div(a.n_val, 16) <= 384;
}

// Heads of a call that go together, part after part through the same scratch: those of `seqs` sequences or, where `heads` are
// fewer than there are, so many of one sequence's. A part's heads do not meet another's.
struct DeltaParts {
    int seqs = 0, heads = 0;
    long long all() const { return (long long)seqs * heads; }
};
// Parts of at most `most` heads, as alike as may be. Heads that share one of the queries' stay together unless `split`.
DeltaParts delta_parts(long long n_seq, long long n_qk, long long share, long long most, bool split = false) {
    const long long n_head = n_qk * share;
    DeltaParts p{1, (int)n_head};
    if (most >= n_head) p.seqs = (int)ceil_div(n_seq, ceil_div(n_seq, most / n_head));
    else if (split && most < share) p.heads = (int)ceil_div(share, ceil_div(share, most));
    else p.heads = (int)(share * ceil_div(n_qk, ceil_div(n_qk, std::max(1LL, most / share))));
    return p;
}

// What is the whole call's in p, for the part that begins at a sequence and a head (a call's last parts may be smaller).
HelixDeltaParams delta_part(HelixDeltaParams p, const DeltaParts& part, long long seq, long long head, size_t es) {
    const long long qk = head / p.share, state = (seq * p.n_head + head) * p.n_key * p.n_val;
    advance(p.q, seq * p.seq_q + qk * p.head_q, es);
    advance(p.k, seq * p.seq_k + qk * p.head_k, es);
    advance(p.v, seq * p.seq_v + head * p.head_v, es);
    advance(p.g, seq * p.seq_g + head, 4);
    advance(p.beta, seq * p.seq_b + head, 4);
    advance(p.o, seq * p.seq_o + head * p.head_o, es);
    advance(p.d_o, seq * p.seq_o + head * p.head_o, es);
    for (const float** s : {&p.s0, &p.d_s}) advance(*s, state, 4);
    for (float** s : {&p.s, &p.ds0}) advance(*s, state, 4);
    const long long row = seq * p.n_tok;   // dense ones
    advance(p.dq, (row * p.n_qk + qk) * p.n_key, es);
    advance(p.dk, (row * p.n_qk + qk) * p.n_key, es);
    advance(p.dv, (row * p.n_head + head) * p.n_val, es);
    advance(p.dg, row * p.n_head + head, 4);
    advance(p.dbeta, row * p.n_head + head, 4);
    p.n_seq = (int)std::min<long long>(part.seqs, p.n_seq - seq);
    p.n_head = (int)std::min<long long>(part.heads, p.n_head - head);
    if (part.heads < p.share) p.n_head = (int)std::min<long long>(p.n_head, p.share - head % p.share);
    p.share = std::min(p.share, p.n_head);
    p.n_qk = p.n_head / p.share;
    return p;
}
// f(parameters) for every part of a call.
template <typename F>
void each_part(const HelixDeltaParams& call, const DeltaParts& part, size_t es, F&& f) {
    for (long long seq = 0; seq < call.n_seq; seq += part.seqs)
        for (long long head = 0; head < call.n_head;) {
            const HelixDeltaParams p = delta_part(call, part, seq, head, es);
            head += p.n_head;
            f(p);
        }
}

// How the rule is cut: parts, and segments of `chunks` chunks of them, whose operands scratch holds at a time.
struct DeltaPlan {
    DeltaParts part;
    int n_chunk = 0, chunks = 0, columns = 0, sets = 1;   // sets: of a segment's operands
    size_t x_at = 0, p_at = 0, decay_at = 0, set = 0, bytes = 0;
};
// Scratch: up to a gigabyte.
constexpr size_t kDeltaScratch = (size_t)1 << 30;

DeltaPlan delta_plan(const helix_delta_rule_args& a) {
    DeltaPlan p;
    if (!delta_heads(a)) return p;
    const long long all = (long long)a.n_seq * a.n_head, share = a.n_head / a.n_qk_head;
    if (a.n_tok <= delta_steps(all, a.n_val, a.io_dtype)) {
        p.part = delta_parts(a.n_seq, a.n_qk_head, share, most_groups(kDeltaThreads) / ceil_div(a.n_val, 64), true);
        return p;
    }
    const size_t x = 6 * 3 * HELIX_DR_FRAG, each = 2 * x + HELIX_DR_DECAY;   // of a chunk of a head
    p.part = delta_parts(a.n_seq, a.n_qk_head, share, std::min<long long>(kDeltaScratch / each, most_groups(2 * kDeltaThreads) / ceil_div(a.n_val, 16)), true);
    const size_t sh = p.part.all();
    p.n_chunk = (int)ceil_div(a.n_tok, HELIX_DR_CHUNK);
    p.chunks = (int)std::min<size_t>(p.n_chunk, kDeltaScratch / (sh * each));
    p.columns = delta_columns((long long)sh, a.n_val);
    if (delta_ahead((long long)sh, p.columns, a)) {
        const int least = (int)std::max<size_t>(32, 2048 / sh), n = std::max<int>(p.n_chunk / least, (int)ceil_div(2 * p.n_chunk, p.chunks));
        if (n > 2) {
            p.chunks = (int)ceil_div(p.n_chunk, n);
            p.sets = 2;
        }
    }
    p.p_at = p.x_at + sh * p.chunks * x;
    p.decay_at = p.p_at + sh * p.chunks * x;
    p.set = p.decay_at + sh * p.chunks * HELIX_DR_DECAY;
    p.bytes = p.sets * p.set;
    return p;
}

// What both passes' arguments have alike.
template <typename A>
HelixDeltaParams delta_params(const A& a) {
    HelixDeltaParams p{};
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.g = a.g;
    p.beta = a.beta;
    p.s0 = a.s0;
    p.seq_q = a.seq_q;
    p.tok_q = a.tok_q;
    p.head_q = a.head_q;
    p.seq_k = a.seq_k;
    p.tok_k = a.tok_k;
    p.head_k = a.head_k;
    p.seq_v = a.seq_v;
    p.tok_v = a.tok_v;
    p.head_v = a.head_v;
    p.seq_g = a.seq_g;
    p.tok_g = a.tok_g;
    p.seq_b = a.seq_beta;
    p.tok_b = a.tok_beta;
    p.n_seq = a.n_seq;
    p.n_tok = a.n_tok;
    p.n_qk = a.n_qk_head;
    p.n_head = a.n_head;
    p.share = a.n_head / a.n_qk_head;
    p.row_qk = a.n_qk_head;
    p.row_head = a.n_head;
    p.n_key = a.n_key;
    p.n_val = a.n_val;
    p.scale = a.scale;
    return p;
}
template <typename A>
void delta_inputs(const A& a, size_t es) {
    heads("q", a.q, a.n_seq, a.n_tok, a.n_qk_head, a.n_key, a.seq_q, a.tok_q, a.head_q, es, false);
    heads("k", a.k, a.n_seq, a.n_tok, a.n_qk_head, a.n_key, a.seq_k, a.tok_k, a.head_k, es, false);
    heads("v", a.v, a.n_seq, a.n_tok, a.n_head, a.n_val, a.seq_v, a.tok_v, a.head_v, es, false);
    gates("g", a.g, a.n_tok, a.seq_g, a.tok_g);
    gates("beta", a.beta, a.n_tok, a.seq_beta, a.tok_beta);
    need(aligned(a.s0, 4), "s0 is not aligned to its elements");
}

}  // namespace

extern "C" size_t helix_delta_rule_scratch_size(const helix_delta_rule_args* a) { return a ? delta_plan(*a).bytes : 0; }

extern "C" helix_status helix_delta_rule_encode(helix_ctx* ctx, void* stream, const helix_delta_rule_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        if (!delta_shape(*a)) return;
        const size_t es = kBytes[a->io_dtype];
        delta_inputs(*a, es);
        heads("o", a->o, a->n_seq, a->n_tok, a->n_head, a->n_val, a->seq_o, a->tok_o, a->head_o, es, true);
        need(a->s != nullptr && aligned(a->s, 4), "s is NULL or not aligned to its elements");
        const DeltaPlan plan = delta_plan(*a);
        need(plan.bytes == 0 || (a->scratch && a->scratch_bytes >= plan.bytes),
             "scratch smaller than helix_delta_rule_scratch_size()", HELIX_ERR_SCRATCH_TOO_SMALL);
        need(aligned(a->scratch, 16), "scratch is not 16-byte aligned");
        HelixDeltaParams call = delta_params(*a);
        call.o = a->o;
        call.s = a->s;
        call.seq_o = a->seq_o;
        call.tok_o = a->tok_o;
        call.head_o = a->head_o;
        const std::string form = delta_form(*a, !plan.bytes);
        if (!plan.bytes) {
            const hipFunction_t f = kernel(ctx, "helix_delta_steps_" + form);
            const long long slices = ceil_div(a->n_val, 64);
            const OnDevice on(ctx->device);
            each_part(call, plan.part, es, [&](HelixDeltaParams p) {
                launch(f, stream, (unsigned)((long long)p.n_seq * p.n_head * slices), 1, kDeltaThreads, p);
            });
            return;
        }
        const hipFunction_t prep = kernel(ctx, "helix_delta_prep_" + form),
                            walk = kernel(ctx, "helix_delta_walk_" + form + "_c" + std::to_string(plan.columns));
        call.n_slice = (int)ceil_div(a->n_val, plan.columns);
        char* sc = static_cast<char*>(a->scratch);
        const OnDevice on(ctx->device);
        each_part(call, plan.part, es, [&](HelixDeltaParams p) {
            const long long sh = (long long)p.n_seq * p.n_head;
            p.n_walk = (unsigned)(sh * p.n_slice);
            for (int first = 0, set = 0; first < plan.n_chunk; first += plan.chunks, set ^= plan.sets - 1) {
                auto at = [&](int i, size_t off) { return sc + i * plan.set + off; };
                const int other = set ^ (plan.sets - 1), next = first + plan.chunks;
                p.x = at(set, plan.x_at);
                p.p = at(set, plan.p_at);
                p.decay = reinterpret_cast<float*>(at(set, plan.decay_at));
                p.chunk0 = first;
                p.n_chunk = std::min(plan.chunks, plan.n_chunk - first);
                if (!first || plan.sets == 1) launch(prep, stream, (unsigned)(sh * p.n_chunk), 1, kDeltaThreads, p);
                p.n_next = plan.sets == 2 ? std::max(0, std::min(plan.chunks, plan.n_chunk - next)) : 0;
                p.next_x = at(other, plan.x_at);
                p.next_p = at(other, plan.p_at);
                p.next_decay = reinterpret_cast<float*>(at(other, plan.decay_at));
                launch(walk, stream, p.n_walk + (unsigned)(sh * p.n_next), 1, 2 * kDeltaThreads, p);
                p.s0 = p.s;   // the next segment starts where this one ends
            }
        });
    });
}

namespace {

// The backward pass: its parts, what a segment's chunks leave for its kernels, and the states that the segments start from.
struct DeltaBwdPlan {
    DeltaParts part;
    int n_chunk = 0, chunks = 0, n_seg = 0, columns = 0;
    size_t x_at = 0, tt_at = 0, pt_at = 0, decay_at = 0, s_at = 0, e_at = 0, d_at = 0, z_at = 0, pg_at = 0, pb_at = 0, tri_at = 0, start_at = 0, state = 0, bytes = 0;
};
// Scratch of a segment: up to two gigabytes, and up to one for the states that a part's segments start from. Where a call wants
// more it goes in parts: heads with all their tokens, if those that fit give every CU a workgroup of 32 columns, else as many as
// do that, in segments, whose states are formed twice. bf16, heads of 128 x 64, ms with parts of whole tokens | with all heads
// in segments: 32 x 4096 tokens of 64 heads 16.4 | 19.9, 1000 x 256 of 16 heads 6.4 | 9.4. Segments, with workgroups for half
// the CUs | for each | two for each: 2 x 65536 tokens of 64 heads 23.8 | 20.8 | 20.8, 4 x 32768 23.9 | 20.2 | 19.7. (The heads
// of one query head may take more than two gigabytes for a chunk, or than one for the states.)
constexpr size_t kDeltaBwdScratch = (size_t)2 << 30, kDeltaBwdStates = (size_t)1 << 30;

DeltaBwdPlan delta_bwd_plan(const helix_delta_rule_backward_args& a) {
    DeltaBwdPlan p;
    if (!delta_heads(a)) return p;
    const long long launch_heads = most_groups(kDeltaPairThreads) / ceil_div(a.n_val, 16);
    if (!a.n_tok) {   // ds0 = d_s
        p.part = delta_parts(a.n_seq, a.n_qk_head, a.n_head / a.n_qk_head, launch_heads);
        p.columns = 16;
        return p;
    }
    const size_t x = 6 * 3 * HELIX_DR_FRAG, tri = 2 * 10 * 256 * 4, share = a.n_head / a.n_qk_head, sh = (size_t)a.n_seq * a.n_head;
    auto up = [](size_t bytes) { return (bytes + 255) & ~(size_t)255; };
    const size_t state = (size_t)a.n_key * a.n_val * 4, rows = (size_t)HELIX_DR_CHUNK * a.n_val * 4;
    const size_t each = 3 * x + HELIX_DR_DECAY + 2 * state + 2 * rows + 12 * HELIX_DR_CHUNK + tri / share + 1;   // of a chunk of a head
    p.n_chunk = (int)ceil_div(a.n_tok, HELIX_DR_CHUNK);
    auto chunks = [&](size_t heads) { return (int)std::min<size_t>(p.n_chunk, std::max<size_t>(1, kDeltaBwdScratch / (heads * each))); };
    size_t most = sh;
    if (chunks(sh) < p.n_chunk || sh * each > kDeltaBwdScratch) {
        most = std::max<size_t>(kDeltaBwdScratch / (p.n_chunk * each), ceil_div(256, ceil_div(a.n_val, 32)));
        while (most > share && (most * each > kDeltaBwdScratch || (ceil_div(p.n_chunk, chunks(most)) - 1) * most * state > kDeltaBwdStates)) most /= 2;
    }
    p.part = delta_parts(a.n_seq, a.n_qk_head, share, std::min((long long)most, launch_heads));
    const size_t heads = p.part.all(), qk = heads / share;
    p.chunks = chunks(heads);
    p.n_seg = (int)ceil_div(p.n_chunk, p.chunks);
    // (fp32 of 128 keys and 32 columns would not fit in LDS.)
    p.columns = a.io_dtype == HELIX_F32 && a.n_key > 64 ? 16 : delta_columns((long long)heads, a.n_val);
    const size_t of = heads * p.chunks;
    p.tt_at = p.x_at + of * x;
    p.pt_at = p.tt_at + of * x;
    p.decay_at = p.pt_at + of * x;
    p.s_at = p.decay_at + up(of * HELIX_DR_DECAY);
    p.e_at = p.s_at + up(of * state);
    p.d_at = p.e_at + up(of * state);
    p.z_at = p.d_at + up(of * rows);
    p.pg_at = p.z_at + up(of * rows);
    p.pb_at = p.pg_at + of * HELIX_DR_CHUNK * 8;
    p.tri_at = p.pb_at + of * HELIX_DR_CHUNK * 4;
    p.start_at = p.tri_at + qk * p.chunks * tri;
    p.state = up(heads * state);
    p.bytes = p.start_at + (size_t)(p.n_seg - 1) * p.state;
    return p;
}

}  // namespace

extern "C" size_t helix_delta_rule_backward_scratch_size(const helix_delta_rule_backward_args* a) {
    return a ? delta_bwd_plan(*a).bytes : 0;
}

extern "C" helix_status helix_delta_rule_backward_encode(helix_ctx* ctx, void* stream,
                                                         const helix_delta_rule_backward_args* a) {
    return entry(ctx, [&] {
        need(ctx && a, "NULL context or arguments");
        if (!delta_shape(*a)) return;
        const size_t es = kBytes[a->io_dtype];
        delta_inputs(*a, es);
        heads("d_o", a->d_o, a->n_seq, a->n_tok, a->n_head, a->n_val, a->seq_do, a->tok_do, a->head_do, es, false);
        for (const void* o : {(const void*)a->dq, (const void*)a->dk, (const void*)a->dv})
            need(!a->n_tok || (o && aligned(o, es)), "dq, dk or dv is NULL or not aligned to its elements");
        for (const float* o : {a->dg, a->dbeta})
            need(!a->n_tok || (o && aligned(o, 4)), "dg or dbeta is NULL or not aligned to its elements");
        need(a->ds0 != nullptr && aligned(a->ds0, 4) && aligned(a->d_s, 4),
             "ds0 is NULL, or it or d_s not aligned to its elements");
        need((long long)a->n_head * a->n_val < (1LL << 31) / 64 / (long long)es && (long long)a->n_qk_head * a->n_key < (1LL << 31) / 64 / (long long)es,
             "64 tokens of dq, dk or dv span 2^31 bytes or more", HELIX_ERR_UNSUPPORTED_SHAPE);
        const DeltaBwdPlan plan = delta_bwd_plan(*a);
        need(plan.part.all() * std::max<long long>(plan.chunks, ceil_div(a->n_val, plan.columns)) <= most_groups(kDeltaPairThreads),
             "the heads that share a query head exceed a launch", HELIX_ERR_UNSUPPORTED_SHAPE);
        need(plan.bytes == 0 || (a->scratch && a->scratch_bytes >= plan.bytes),
             "scratch smaller than helix_delta_rule_backward_scratch_size()", HELIX_ERR_SCRATCH_TOO_SMALL);
        need(aligned(a->scratch, 16), "scratch is not 16-byte aligned");
        HelixDeltaParams call = delta_params(*a);
        call.d_o = a->d_o;
        call.d_s = a->d_s;
        call.seq_o = a->seq_do;
        call.tok_o = a->tok_do;
        call.head_o = a->head_do;
        call.dq = a->dq;
        call.dk = a->dk;
        call.dv = a->dv;
        call.dg = a->dg;
        call.dbeta = a->dbeta;
        call.ds0 = a->ds0;
        char* sc = static_cast<char*>(a->scratch);
        call.x = sc + plan.x_at;
        call.tt = sc + plan.tt_at;
        call.pt = sc + plan.pt_at;
        call.decay = reinterpret_cast<float*>(sc + plan.decay_at);
        call.keep_s = reinterpret_cast<float*>(sc + plan.s_at);
        call.keep_e = reinterpret_cast<float*>(sc + plan.e_at);
        call.keep_d = reinterpret_cast<float*>(sc + plan.d_at);
        call.keep_z = reinterpret_cast<float*>(sc + plan.z_at);
        call.pair_g = reinterpret_cast<double*>(sc + plan.pg_at);
        call.pair_b = reinterpret_cast<float*>(sc + plan.pb_at);
        call.tri = reinterpret_cast<float*>(sc + plan.tri_at);
        call.n_slice = (int)ceil_div(a->n_val, plan.columns);
        const std::string form = delta_form(*a), wide = form + "_c" + std::to_string(plan.columns);
        const hipFunction_t prep = kernel(ctx, "helix_delta_prep_bwd_" + form), keep = kernel(ctx, "helix_delta_keep_" + wide),
                            back = kernel(ctx, "helix_delta_back_" + wide), pairs = kernel(ctx, "helix_delta_pairs_" + form),
                            grad = kernel(ctx, "helix_delta_grad_" + form);
        const OnDevice on(ctx->device);
        // A part: the states that its segments start from (that of segment i > 0 at i - 1), then its segments from the last on.
        auto run = [&](HelixDeltaParams p) {
            const long long sh = (long long)p.n_seq * p.n_head, sk = (long long)p.n_seq * p.n_qk;
            const unsigned gw = (unsigned)(sh * p.n_slice);
            p.n_walk = gw;
            const float* const s0 = p.s0;
            auto start = [&](int i) { return reinterpret_cast<float*>(sc + plan.start_at + (size_t)(i - 1) * plan.state); };
            auto states = [&](int i) {
                p.chunk0 = i * plan.chunks;
                p.n_chunk = std::min(plan.chunks, plan.n_chunk - p.chunk0);
                p.s0 = i ? start(i) : s0;
                launch(prep, stream, (unsigned)(sh * p.n_chunk), 1, kDeltaThreads, p);
                launch(keep, stream, gw, 1, 2 * kDeltaThreads, p);
            };
            for (int i = 0; i + 1 < plan.n_seg; ++i) {
                p.s = start(i + 1);
                states(i);
            }
            p.s = nullptr;
            for (int i = plan.n_seg - 1; i >= 0; --i) {
                states(i);
                launch(back, stream, gw, 1, 2 * kDeltaThreads, p);
                launch(pairs, stream, (unsigned)(sk * p.n_chunk), 1, kDeltaPairThreads, p);
                launch(grad, stream, (unsigned)(sk * p.n_chunk), 1, 2 * kDeltaThreads, p);
                p.d_s = p.ds0;   // the segment before goes on from here
            }
            if (!plan.n_seg) launch(back, stream, gw, 1, 2 * kDeltaThreads, p);   // no tokens: ds0 = d_s
        };
        each_part(call, plan.part, es, run);
    });
}

namespace helix::rt {

const std::vector<std::string>& layer_kernel_names() {
    static const std::vector<std::string> names = [] {
        std::vector<std::string> v{"helix_norm_dw", "helix_fp8_scales", "helix_matmul_fp8_join_f16",
                                   "helix_matmul_fp8_join_bf16", "helix_gated_scan_fill"};
        for (const char* t : kTags)
            for (const char* k : {"helix_norm_", "helix_norm_bwd_", "helix_norm_dw_part_"})
                v.push_back(std::string(k) + t);
        for (const char* tag : kTags)
            for (const char* n : {"1", "2", "3", "4", "6", "8"}) {
                for (const char* k : {"helix_norm_", "helix_norm_bwd_"}) v.push_back(std::string(k) + tag + "_g" + n);
                if (n[0] <= '4') v.push_back(std::string("helix_norm_") + tag + "_w" + n);
                if (n[0] <= '2') v.push_back(std::string("helix_norm_bwd_") + tag + "_w" + n);
            }
        for (const char* tag : kTags)
            for (const char* n : {"_64", "_128"}) {
                v.push_back(std::string("helix_delta_steps_") + tag + n);
                for (const char* s : {"", "_s"}) {
                    if (*s && tag == kTags[HELIX_F32]) continue;
                    for (const char* k : {"prep_", "prep_bwd_", "pairs_", "grad_"}) v.push_back(std::string("helix_delta_") + k + tag + n + s);
                    for (const char* k : {"walk_", "keep_", "back_"})
                        for (const char* c : {"_c16", "_c32"})
                            if (std::string(k) + tag + n + c != "back_f32_128_c32") v.push_back(std::string("helix_delta_") + k + tag + n + s + c);
                }
            }
        v.push_back("helix_group_norm_dw");
        for (const char* tag : kTags) {
            v.push_back(std::string("helix_group_norm_fp8_") + tag + "_any");
            for (const GroupForm& f : kGroupForms)
                for (const char* k : {"helix_group_norm_", "helix_group_norm_bwd_", "helix_group_norm_fp8_"})
                    v.push_back(k + (tag + f.name()));
        }
        for (const char* tag : kTags)
            for (const char* k : {"_blocks", "_r1", "_r1w4", "_r2", "_r3", "_r4"})
                v.push_back(std::string("helix_matmul_fp8_") + tag + k);
        for (const Tiling& t : kTilings) v.push_back(std::string("helix_matmul_fp8") + t.kernel);
        for (const char* k : {"_t44p", "_t42p"}) v.push_back(std::string("helix_matmul_fp8") + k);
        for (const char* t : kTags)
            for (const char* k : {"helix_gated_scan_", "helix_gated_scan_bwd_"})
                for (const char* x : {"_v_", "_s_"})
                    for (const char* w : {"steps", "w4", "w8"}) v.push_back(std::string(k) + t + x + w);
        return v;
    }();
    return names;
}

}  // namespace helix::rt
