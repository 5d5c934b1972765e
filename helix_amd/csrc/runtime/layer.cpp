// layer.cpp -- the entry points of the layer operators (helix_layer.h): checks,
// choice of the kernel, launches. As in dispatch.cpp every check comes before the
// first launch, and nothing is allocated, synchronized or waited for.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <string>

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
