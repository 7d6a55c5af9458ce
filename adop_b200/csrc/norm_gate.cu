// Host side of the group normalisation with an activation and of the gate of a gated convolution: argument checks, which
// kernel and launch shape a call takes, and the C ABI. The kernels are in norm_gate.cuh, compiled once per image type.
#include "common.cuh"
#include "norm_gate.h"
#include "per_device.h"

namespace adop {

namespace {

int64_t gcd64(int64_t a, int64_t b)
{
    while (b) { const int64_t r = a % b; a = b; b = r; }
    return a;
}

adop_status refuse(adop_status s, const char* why)
{
    snprintf(last_error_buffer(), 512, "%s", why);
    return s;
}

int element_size(int type) { return type == ADOP_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

adop_status check_params(const adop_norm_params* p, bool norm)
{
    if (!p) return refuse(ADOP_ERR_INVALID_ARGUMENT, "no parameters");
    if (p->batch < 0 || p->pixels < 0 || p->channels <= 0) return refuse(ADOP_ERR_INVALID_ARGUMENT, "batch, pixels or channels");
    if (p->type != ADOP_TYPE_F32 && p->type != ADOP_TYPE_F16 && p->type != ADOP_TYPE_BF16)
        return refuse(ADOP_ERR_INVALID_ARGUMENT, "type is not ADOP_TYPE_*");
    if (p->activation < ADOP_ACTIVATION_NONE || p->activation > ADOP_ACTIVATION_SILU)
        return refuse(ADOP_ERR_INVALID_ARGUMENT, "activation is not ADOP_ACTIVATION_*");
    if (p->channels > ADOP_NORM_MAX_CHANNELS) return refuse(ADOP_ERR_SIZE_LIMIT, "more than ADOP_NORM_MAX_CHANNELS channels");
    if (p->batch > 65535 || p->pixels > 0x7F000000)  // rows are counted with 32-bit ints
        return refuse(ADOP_ERR_SIZE_LIMIT, "more than 65535 images, or 0x7F000000 pixels in one");
    if (norm)
    {
        if (p->num_groups <= 0 || p->channels % p->num_groups != 0)
            return refuse(ADOP_ERR_INVALID_ARGUMENT, "num_groups does not divide the channels");
        if (p->param_type != ADOP_TYPE_F32 && p->param_type != p->type)
            return refuse(ADOP_ERR_INVALID_ARGUMENT, "param_type is neither ADOP_TYPE_F32 nor the images' type");
        const size_t size = p->param_type == ADOP_TYPE_F32 ? 4 : 2;
        if (!aligned(p->weight, size) || !aligned(p->bias, size)) return refuse(ADOP_ERR_INVALID_ARGUMENT, "weight or bias is not aligned to its type");
        if (!(p->eps >= 0.f) || p->eps > 3.0e38f) return refuse(ADOP_ERR_INVALID_ARGUMENT, "eps is negative or not finite");
    }
    return ADOP_OK;
}

constexpr int64_t kExtent = (int64_t)1 << 56;  // elements from the first image to the last, and of an image

adop_status check_image(const adop_norm_params* p, const adop_norm_image& im, bool output, const char* what)
{
    if (!im.data || !aligned(im.data, (size_t)element_size(p->type))) return refuse(ADOP_ERR_INVALID_ARGUMENT, what);
    if (im.image_stride < 0 || im.pixel_stride < 0 || im.image_stride > kExtent / p->batch || im.pixel_stride > kExtent / p->pixels)
        return refuse(ADOP_ERR_INVALID_ARGUMENT, what);
    if (output)
    {
        if (p->pixels > 1 && im.pixel_stride < p->channels) return refuse(ADOP_ERR_INVALID_ARGUMENT, what);
        if (p->batch > 1 && im.image_stride < (p->pixels - 1) * im.pixel_stride + p->channels) return refuse(ADOP_ERR_INVALID_ARGUMENT, what);
    }
    return ADOP_OK;
}

constexpr size_t kMostShared = 220 * 1024;  // of a block

// Vector and row of a call. The widest vector that every tensor's address and strides allow: 16, 8 or 4 bytes or one element.
// A vector either lies within a pixel's channels, or all tensors are dense and a row of lcm(channels, vector) elements holds
// whole pixels, an even number of times per image.
struct Shape
{
    int vec, V, P, ppr;
};
Shape choose_shape(const adop_norm_params* p, const adop_norm_image* const* images, int n, int from = kVec16)
{
    const int es = element_size(p->type);
    for (int vec = from; vec < kVec1; ++vec)
    {
        const int V = (16 >> vec) / es;
        if (V < 2) break;
        bool ok = true, dense = true;
        for (int i = 0; i < n; ++i)
        {
            const adop_norm_image& im = *images[i];
            ok = ok && aligned(im.data, (size_t)V * es) && (p->batch == 1 || im.image_stride % V == 0);
            dense = dense && (p->pixels == 1 || im.pixel_stride == p->channels);
        }
        if (!ok) continue;
        bool within = p->channels % V == 0;
        for (int i = 0; i < n; ++i) within = within && (p->pixels == 1 || images[i]->pixel_stride % V == 0);
        if (within) return {vec, V, p->channels / V, 1};
        const int common = (int)gcd64(p->channels, V), ppr = V / common;
        if (dense && p->pixels % ppr == 0 && (int64_t)p->channels * ppr <= ADOP_NORM_MAX_CHANNELS) return {vec, V, p->channels / common, ppr};
    }
    return {kVec1, 1, p->channels, 1};
}

// Blocks and threads of a launch over rows of P vectors: as many whole rows as `most` threads hold.
void threads_of(int P, int most, int* R, int* threads)
{
    *R = P > most ? 1 : most / P;
    *threads = P > most ? most : (*R * P + 31) / 32 * 32;
}

// The last launch of a backward pass shares the SMs with no other: it gets two blocks an SM where they have something to do (four images
// of 33 MB of inputs 65.1 -> 62.2 us, sixteen 249 -> 232 us, 254 us with the others' launches doubled too; parts of 35 KB 17.7 -> 19.6 us).
constexpr int64_t kAlonePart = 64 << 10;  // bytes of one tensor

// Images are taken in groups, a launch for the sums and one for what follows each, which costs 5 us of waits and tails a group. Where the
// second read is bound by memory, forward without a gate, groups that the L2 holds pay (sixteen images of 17 MB, four at a time 135 us,
// all at once 141 us). With a gate the arithmetic hides the second read (sixteen of 33 MB two at a time 252 us, all at once 231 us). Backward,
// in between (sixteen of 50 MB two at a time 372 us, four at a time 346 us, all at once 352 us).
constexpr int64_t kForwardGroup = 70ll << 20, kBackwardGroup = 210ll << 20, kGroupCost = 20ll << 20;
constexpr int64_t kMinChunk = 16 << 10;  // bytes of one tensor that a block is worth

// How the streaming kernels share out a batch: images of a launch and blocks of an image. By the sizes alone, so that the
// workspace is known without the tensors.
struct Share
{
    int images, chunks;
};
int param_blocks_of(const adop_norm_params* p) { return (p->channels + kParamChannels - 1) / kParamChannels; }
Share share_of(const adop_norm_params* p, bool gated, bool backward)
{
    const int64_t tensor = p->pixels * p->channels * element_size(p->type);
    const int64_t read = tensor * (1 + (gated ? 1 : 0) + (backward ? 1 : 0));
    int64_t most = backward ? kBackwardGroup / read : gated ? p->batch : kForwardGroup / read;
    if (most > p->batch) most = p->batch;
    if (most < 1) most = 1;
    // groups of one size, the last one too where a few images are a group: its blocks have as much to do as the others'
    const int64_t launches = (p->batch + most - 1) / most;
    most = (p->batch + launches - 1) / launches;
    int64_t images = most, least = -1;
    for (int64_t n = most; n >= 1 && 2 * n >= most && n > most - 16; --n)
    {
        const int64_t cost = (p->batch + n - 1) / n * (kGroupCost + n * read);
        if (least < 0 || cost < least) { least = cost; images = n; }
    }
    // A block for each SM, as many for every image, rounded down: up to sixteen images leave few SMs without one. Larger batches may leave half
    // of them: a gated forward pass over 75 images of 128 x 128 x 32 in bfloat16 takes 126 us, 69 us over 74, and 243 us over 150, 132 us over 148
    // (backward, taken in groups of images, 116 and 118, 245 and 236 us).
    // Backward, the few blocks that add up the parameters' gradients are among them: with one more than SMs, two blocks of the
    // launch that starts early share one (four 256 x 256 images of 32 channels in fp32, backward: 29.1 us, so 26.3 us).
    const int64_t params = backward && param_blocks_of(p) <= 4 ? param_blocks_of(p) : 0, wave = sm_count() > 8 ? sm_count() - params : sm_count();
    int64_t chunks = wave / images, worth = (tensor + kMinChunk - 1) / kMinChunk;
    if (chunks > worth) chunks = worth;
    return {(int)images, (int)(chunks < 1 ? 1 : chunks)};
}

// A thread adds up kChain vectors at most in 32 bits before its sums go on in 64, or in a second chain: n terms of one sign are off by n 2^-25 of
// their sum at worst, as each addition rounds by 2^-24 of what there is by then. Where a block's share of an image is longer (2 MB of 16-byte
// vectors; no image in memory where there is a second chain of as many), the sums take several launches, each over the next piece of every share.
// Two values in turn, the worst of their kind (the same term rounds the same way), came out off by 2e-4 in float32 for 14000 vectors in one
// chain, by 3e-6 so. The launches cost nothing where they overlap (a 4K image of 64 channels in bfloat16: 553 us forward with four as with one, 903
// backward with five for 963) and 1 to 2 % where they cannot; second chains of wide vectors would spill, 2 % for all sizes backward.
int sum_launches(int64_t rows, int V, int R, int chunks)
{
    const int64_t share = (rows + chunks - 1) / chunks, most = (int64_t)R * kChain * (second_chain(V) ? kChain : 1);
    return (int)((share + most - 1) / most);
}
// of the vectors that the tensors may turn out to allow, the ones that take most
int most_sum_launches(const adop_norm_params* p, int chunks, bool backward)
{
    int most = 1;
    for (int V = 16 / element_size(p->type); V >= 1; V >>= 1)
    {
        const int common = (int)gcd64(p->channels, V);
        int R, threads;
        threads_of(p->channels / common, backward ? kNormGradThreads : kNormThreads, &R, &threads);
        const int launches = sum_launches(p->pixels / (V / common), V, R, chunks);
        if (launches > most) most = launches;
    }
    return most;
}

constexpr size_t align16(size_t v) { return (v + 15) / 16 * 16; }
size_t group_part_bytes(const adop_norm_params* p, int64_t parts) { return align16(sizeof(float2) * p->batch * (size_t)parts * p->num_groups); }
size_t channel_part_bytes(const adop_norm_params* p, int64_t parts) { return align16(sizeof(float2) * p->batch * (size_t)parts * p->channels); }

constexpr size_t kWarpScratch = sizeof(double2) * (kNormThreads / 32);  // group_sums'
// the block's sums, as the kernels lay them out: block_moments' with the counts, block_sums'
size_t sum_rows(const Shape& sh, int R, int threads) { return (size_t)(32 % sh.P == 0 ? threads / 32 : R) * sh.P; }
size_t moments_scratch(const Shape& sh, int m, int R, int threads) { return sizeof(float) * (2 * (sh.V / m) + 1) * sum_rows(sh, R, threads); }
size_t sums_scratch(const Shape& sh, int R, int threads) { return sizeof(float) * 2 * sh.V * sum_rows(sh, R, threads); }

// ---- images that stay in a block's shared memory ----------------------------------------------------------------------------
// A block takes one of 2^slices channel ranges of an image, whole groups of at least kSliceBytes side by side. One launch in place of two
// and no workspace: on the host 6 us in place of 10. On the device a block of 15 KB takes 5.1 us and one of 32 KB 6.2 us, two launches over
// the whole GPU 5.4 and 5.8 us, so 32 KB; where there is a block for every other SM, 96 KB (256 images of 16 KB: 7.4 against 8.7 us, sixteen
// of 1 MB 13.6 against 13.8 us).
constexpr int64_t kSliceBytes = 64;
constexpr int64_t kResidentBytes = 32 << 10;
constexpr int64_t kResidentManyBytes = 96 << 10;
struct Resident
{
    int slices, threads, R;  // slices: log2
    size_t fixed, smem;      // bytes in front of the vectors, and in all
};
bool resident_of(const adop_norm_params* p, const Shape& sh, bool gated, Resident* r)
{
    if (sh.vec == kVec1) return false;
    const int es = element_size(p->type), tensors = gated ? 2 : 1;
    const int64_t rows = p->pixels / sh.ppr;
    if (rows * sh.P * sh.V * es * tensors > kResidentManyBytes * p->num_groups) return false;
    // the fewest ranges that do
    for (int log2 = 0; log2 <= 12 && p->num_groups % (1 << log2) == 0; ++log2)
    {
        const int slices = 1 << log2, C = p->channels / slices, G = p->num_groups / slices;
        if (log2 > 0 && (sh.ppr != 1 || C % sh.V != 0 || (int64_t)C * es < kSliceBytes)) return false;
        Shape s = sh;
        s.P = sh.P / slices;
        if (s.P > kNormThreads) continue;
        Resident c{log2};
        threads_of(s.P, kNormThreads, &c.R, &c.threads);
        const int64_t vectors = (rows + c.R - 1) / c.R * c.threads * sh.V * es * tensors;
        const bool many = ((int64_t)p->batch << log2) * 2 >= sm_count();
        if (vectors > (many ? kResidentManyBytes : kResidentBytes)) continue;
        const int m = (int)gcd64(p->channels / p->num_groups, sh.V);
        c.fixed = align16(kWarpScratch + sizeof(float2) * G + sizeof(float) * 2 * (size_t)C + moments_scratch(s, m, c.R, c.threads));
        c.smem = c.fixed + (size_t)vectors;
        if (c.smem > kMostShared) continue;
        *r = c;
        return true;
    }
    return false;
}

// ---- launches -----------------------------------------------------------------------------------------------------------
struct Launch
{
    const char* name;
    int which, threads;
    dim3 grid;
    size_t smem;
    bool early;  // may start before the launch in front of it has ended (it waits by itself)
};

const void* kernel_of(int type, int which, int vec, bool gated, int act)
{
    if (type == ADOP_TYPE_F32) return norm_kernel_f32(which, vec, gated, act);
    return type == ADOP_TYPE_F16 ? norm_kernel_f16(which, vec, gated, act) : norm_kernel_bf16(which, vec, gated, act);
}

adop_status launch(const Launch& l, const adop_norm_params* p, const Shape& sh, bool gated, NormArgs& a, cudaStream_t st)
{
    const void* f = kernel_of(p->type, l.which, sh.vec, gated, p->activation);
    if (l.smem > 48 * 1024)
    {
        static OncePerDevice once[3][kNormKernels][kNormVectors][2][4];
        int device = 0;
        ADOP_CUDA_TRY(cudaGetDevice(&device));
        ADOP_CUDA_TRY(once[p->type][l.which][sh.vec][gated][p->activation].run(
            device, [&] { return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared); }));
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = l.grid;
    cfg.blockDim = dim3((unsigned)l.threads);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = st;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = l.early ? 1 : 0;
    void* args[] = {&a};
    cudaError_t e = cudaSuccess;
    ADOP_LAUNCH(l.name, st, (e = cudaLaunchKernelExC(&cfg, f, args)));
    if (e == cudaSuccess) return ADOP_OK;
    cudaGetLastError();  // the caller has it, the next call's checks are not to find it
    return record_cuda_error(e, l.name);
}

NormImage image_of(const adop_norm_image& im, const Shape& sh) { return {im.data, im.image_stride, im.pixel_stride * sh.ppr}; }

NormArgs args_of(const adop_norm_params* p, const Shape& sh, bool norm)
{
    NormArgs a{};
    a.C = p->channels;
    a.G = norm ? p->num_groups : 1;
    a.Cg = a.C / a.G;
    a.P = sh.P; a.ppr = sh.ppr;
    a.rows = (int)(p->pixels / sh.ppr);
    a.m = (int)gcd64(a.Cg, sh.V);
    a.act = p->activation;
    a.param_type = p->param_type;
    a.eps = p->eps;
    a.weight = p->weight; a.bias = p->bias;
    return a;
}
NormParts parts_of(int rows, int64_t count)
{
    if (count > rows) count = rows;
    return {(int)count, rows / (int)count, rows % (int)count};
}
// what follows from the sizes of a slice, the threads and the number of parts that an image's sums are taken in
void finish(NormArgs* a, int threads, int64_t chunks)
{
    auto log2_of = [](int64_t items) {
        int l = 0;
        while (l < 5 && (1 << l) < items) ++l;
        return l;
    };
    const int rows = 32 % a->P == 0 ? threads / 32 : a->R;
    a->row_lanes = log2_of(rows);
    const int slots = a->Cg / a->m * a->ppr;
    a->lanes = log2_of((int64_t)(1 << a->row_lanes) * slots);
    // few groups of many sums: more warps than one each
    a->warps = rows * slots > 64 && a->G * 2 <= threads / 32 ? threads / 32 / a->G : 1;
    a->sums = a->own = parts_of(a->rows, chunks);
    const double per_row = (double)a->ppr * a->Cg;
    a->inv_n = 1.0 / (a->rows * per_row);
    a->inv_short = 1.0 / (a->sums.rows * per_row);
    a->inv_long = 1.0 / ((a->sums.rows + 1) * per_row);
    a->inv_P = 1.f / a->P; a->inv_Cg = 1.f / a->Cg;
    a->gather = log2_of(chunks);
    while (a->gather > 0 && a->G << a->gather > threads) --a->gather;
}
size_t apply_smem(const NormArgs& a) { return sizeof(float2) * 2 * a.G + sizeof(float) * 2 * a.C; }

// the streaming kernels' vectors behind `fixed` bytes of shared memory; all in all
size_t stream_smem(size_t fixed, const Shape& sh, int es, int threads, bool gated, bool grad)
{
    const int tensors = 1 + (gated ? 1 : 0) + (grad ? 1 : 0);
    return align16(fixed) + (sh.vec == kVec1 ? 0 : (size_t)stream_depth(gated, grad) * tensors * threads * sh.V * es);
}

adop_status check_workspace(const adop_norm_params* p, const adop_norm_io* io, bool gated, bool backward)
{
    const size_t need = adop_group_norm_workspace_bytes(p, gated, backward);
    if (need == 0) return ADOP_OK;
    if (!io->workspace || io->workspace_bytes < need) return refuse(ADOP_ERR_WORKSPACE_TOO_SMALL, "workspace below adop_group_norm_workspace_bytes");
    if (!aligned(io->workspace, 16)) return refuse(ADOP_ERR_INVALID_ARGUMENT, "the workspace is not 16-byte aligned");
    return ADOP_OK;
}

#define ADOP_TRY(expr)                       \
    do {                                     \
        const adop_status _s = (expr);       \
        if (_s != ADOP_OK) return _s;        \
    } while (0)

}  // namespace
}  // namespace adop

using namespace adop;

extern "C" size_t adop_group_norm_workspace_bytes(const adop_norm_params* p, int32_t gated, int32_t backward)
{
    if (check_params(p, true) != ADOP_OK || p->batch == 0 || p->pixels == 0) return 0;
    const Share s = share_of(p, gated != 0, backward != 0);
    const int64_t parts = (int64_t)s.chunks * most_sum_launches(p, s.chunks, backward != 0);
    return group_part_bytes(p, parts) + (backward ? channel_part_bytes(p, parts) : 0);
}

extern "C" adop_status adop_group_norm_forward(const adop_norm_params* p, const adop_norm_io* io, void* stream)
{
    ADOP_TRY(check_params(p, true));
    if (!io) return refuse(ADOP_ERR_INVALID_ARGUMENT, "no tensors");
    if (!io->mean != !io->rstd || !aligned(io->mean, 4) || !aligned(io->rstd, 4))
        return refuse(ADOP_ERR_INVALID_ARGUMENT, "mean and rstd are given together or not at all, aligned to their type");
    if (p->batch == 0 || p->pixels == 0) return ADOP_OK;
    const bool gated = io->gate.data != nullptr;
    ADOP_TRY(check_image(p, io->x, false, "x"));
    if (gated) ADOP_TRY(check_image(p, io->gate, false, "gate"));
    ADOP_TRY(check_image(p, io->y, true, "y"));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const adop_norm_image* images[3] = {&io->x, &io->y, &io->gate};
    const Shape sh = choose_shape(p, images, gated ? 3 : 2);
    NormArgs a = args_of(p, sh, true);
    a.x = image_of(io->x, sh);
    a.gate = image_of(io->gate, sh);
    a.y = image_of(io->y, sh);
    a.mean = io->mean; a.rstd = io->rstd;
    a.group_part = static_cast<float2*>(io->workspace);
    Resident r;
    if (resident_of(p, sh, gated, &r))
    {
        a.slices = r.slices;
        a.C >>= r.slices; a.G >>= r.slices; a.P >>= r.slices;
        a.R = r.R;
        finish(&a, r.threads, 1);
        a.vectors = (int)r.fixed;
        return launch({"k_norm_resident", kNormResident, r.threads, dim3((unsigned)p->batch << r.slices), r.smem, false}, p, sh, gated, a, st);
    }
    ADOP_TRY(check_workspace(p, io, gated, false));
    int threads;
    threads_of(a.P, kNormThreads, &a.R, &threads);
    const Share share = share_of(p, gated, false);
    const NormParts shares = parts_of(a.rows, share.chunks);
    a.part_step = sum_launches(a.rows, sh.V, a.R, shares.count);
    finish(&a, threads, (int64_t)shares.count * a.part_step);
    const size_t smem_stats = kWarpScratch + moments_scratch(sh, a.m, a.R, threads);
    const size_t smem_apply = apply_smem(a);
    const int es = element_size(p->type);
    for (a.image0 = 0; a.image0 < p->batch; a.image0 += share.images)
    {
        const unsigned n = (unsigned)(p->batch - a.image0 < share.images ? p->batch - a.image0 : share.images);
        a.vectors = (int)align16(smem_stats);
        a.own = a.sums;
        // Behind a gate a block has its SM busy: blocks that start early on SMs which the launch in front leaves free gather there, and the results'
        // blocks after them (32 images of 960 x 540 x 16 in bfloat16, 128 blocks: 721 us, 503 us one launch after the other). With a block on every SM
        // they find one place each (a 4K image of 32 channels in float32: 826 us, 857 us one after the other).
        const bool early = !gated || (int64_t)shares.count * n >= sm_count();
        for (a.part0 = 0; a.part0 < a.part_step; ++a.part0)
            ADOP_TRY(launch({"k_norm_stats", kNormStats, threads, dim3((unsigned)shares.count, n), stream_smem(smem_stats, sh, es, threads, gated, false),
                             a.part0 == 0 ? a.image0 > 0 : early}, p, sh, gated, a, st));
        a.vectors = (int)align16(smem_apply);
        a.own = shares;
        ADOP_TRY(launch({"k_norm_apply", kNormApply, threads, dim3((unsigned)a.own.count, n), stream_smem(smem_apply, sh, es, threads, gated, false), true}, p, sh,
                        gated, a, st));
    }
    return ADOP_OK;
}

extern "C" adop_status adop_group_norm_backward(const adop_norm_params* p, const adop_norm_io* io, void* stream)
{
    ADOP_TRY(check_params(p, true));
    if (!io) return refuse(ADOP_ERR_INVALID_ARGUMENT, "no tensors");
    if (!aligned(io->grad_weight, (size_t)element_size(p->param_type)) || !aligned(io->grad_bias, (size_t)element_size(p->param_type)))
        return refuse(ADOP_ERR_INVALID_ARGUMENT, "grad_weight or grad_bias is not aligned to its type");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->batch == 0 || p->pixels == 0)
    {
        const size_t bytes = (size_t)p->channels * element_size(p->param_type);
        if (io->grad_weight) ADOP_CUDA_TRY(cudaMemsetAsync(io->grad_weight, 0, bytes, st));
        if (io->grad_bias) ADOP_CUDA_TRY(cudaMemsetAsync(io->grad_bias, 0, bytes, st));
        return ADOP_OK;
    }
    const bool gated = io->gate.data != nullptr;
    if (!io->mean || !io->rstd || !aligned(io->mean, 4) || !aligned(io->rstd, 4)) return refuse(ADOP_ERR_INVALID_ARGUMENT, "mean and rstd of the forward call");
    ADOP_TRY(check_image(p, io->x, false, "x"));
    ADOP_TRY(check_image(p, io->grad_y, false, "grad_y"));
    ADOP_TRY(check_image(p, io->grad_x, true, "grad_x"));
    if (gated)
    {
        ADOP_TRY(check_image(p, io->gate, false, "gate"));
        ADOP_TRY(check_image(p, io->grad_gate, true, "grad_gate"));
    }
    const adop_norm_image* images[5] = {&io->x, &io->grad_y, &io->grad_x, &io->gate, &io->grad_gate};
    const int es = element_size(p->type);
    Shape sh;
    NormArgs a;
    int threads;
    size_t smem_sums;
    // thousands of channels leave no room for wide vectors under way beside their sums
    for (int from = kVec16;; from = sh.vec + 1)
    {
        sh = choose_shape(p, images, gated ? 5 : 3, from);
        a = args_of(p, sh, true);
        threads_of(a.P, kNormGradThreads, &a.R, &threads);
        smem_sums = sizeof(float2) * a.G + sizeof(float) * 4 * (size_t)a.C + sums_scratch(sh, a.R, threads);
        if (sh.vec == kVec1 || stream_smem(smem_sums, sh, es, threads, gated, true) <= kMostShared) break;
    }
    a.x = image_of(io->x, sh);
    a.gate = image_of(io->gate, sh);
    a.dy = image_of(io->grad_y, sh);
    a.dx = image_of(io->grad_x, sh);
    a.dgate = image_of(io->grad_gate, sh);
    a.mean = io->mean; a.rstd = io->rstd;
    a.dweight = io->grad_weight; a.dbias = io->grad_bias;
    const bool params = io->grad_weight || io->grad_bias;
    ADOP_TRY(check_workspace(p, io, gated, true));
    const Share share = share_of(p, gated, true);
    const NormParts shares = parts_of(a.rows, share.chunks);
    a.part_step = sum_launches(a.rows, sh.V, a.R, shares.count);
    finish(&a, threads, (int64_t)shares.count * a.part_step);
    a.group_part = static_cast<float2*>(io->workspace);
    a.channel_part = params ? reinterpret_cast<float2*>(static_cast<char*>(io->workspace) + group_part_bytes(p, a.sums.count)) : nullptr;
    a.param_parts = p->batch * a.sums.count;
    size_t smem_apply = apply_smem(a);
    if (params && smem_apply < sizeof(double) * 2 * threads) smem_apply = sizeof(double) * 2 * threads;
    const int64_t part = (int64_t)shares.rows * a.P * sh.V * es;
    for (a.image0 = 0; a.image0 < p->batch; a.image0 += share.images)
    {
        const unsigned n = (unsigned)(p->batch - a.image0 < share.images ? p->batch - a.image0 : share.images);
        const bool last = a.image0 + share.images >= p->batch;
        // the parameters' gradients need the sums of all images: blocks of the last launch add them up
        a.param_blocks = params && last ? param_blocks_of(p) : 0;
        a.vectors = (int)align16(smem_sums);
        a.own = a.sums;
        for (a.part0 = 0; a.part0 < a.part_step; ++a.part0)
            ADOP_TRY(launch({"k_norm_grad_sums", kNormGradSums, threads, dim3((unsigned)shares.count, n), stream_smem(smem_sums, sh, es, threads, gated, true),
                             a.image0 + a.part0 > 0}, p, sh, gated, a, st));
        a.vectors = (int)align16(smem_apply);
        a.own = last && part >= kAlonePart ? parts_of(a.rows, (int64_t)shares.count * 2) : shares;
        ADOP_TRY(launch({"k_norm_grad_apply", kNormGradApply, threads, dim3((unsigned)(a.own.count + a.param_blocks), n),
                         stream_smem(smem_apply, sh, es, threads, gated, true), true}, p, sh, gated, a, st));
    }
    return ADOP_OK;
}

namespace {
adop_status gate_launch(const adop_norm_params* p, const Shape& sh, NormArgs& a, bool backward, cudaStream_t st)
{
    const int most = backward ? kNormGradThreads : kNormThreads;
    int threads;
    threads_of(a.P, most, &a.R, &threads);
    const int64_t worth = (p->pixels * p->channels * element_size(p->type) + kMinChunk - 1) / kMinChunk;
    int64_t chunks = ((int64_t)sm_count() * (backward ? kNormGradBlocks : kNormBlocks) + p->batch - 1) / p->batch;
    if (chunks > worth) chunks = worth;
    if (chunks > a.rows) chunks = a.rows;
    finish(&a, threads, (int)chunks);
    return launch({backward ? "k_gate_grad" : "k_gate", backward ? kGateGrad : kGate, threads, dim3((unsigned)chunks, (unsigned)p->batch),
                   stream_smem(0, sh, element_size(p->type), threads, true, backward), false}, p, sh,
                  true, a, st);
}
}  // namespace

extern "C" adop_status adop_gated_activation_forward(const adop_norm_params* p, const adop_norm_io* io, void* stream)
{
    ADOP_TRY(check_params(p, false));
    if (!io) return refuse(ADOP_ERR_INVALID_ARGUMENT, "no tensors");
    if (p->batch == 0 || p->pixels == 0) return ADOP_OK;
    ADOP_TRY(check_image(p, io->x, false, "x"));
    ADOP_TRY(check_image(p, io->gate, false, "gate"));
    ADOP_TRY(check_image(p, io->y, true, "y"));
    const adop_norm_image* images[3] = {&io->x, &io->gate, &io->y};
    const Shape sh = choose_shape(p, images, 3);
    NormArgs a = args_of(p, sh, false);
    a.x = image_of(io->x, sh);
    a.gate = image_of(io->gate, sh);
    a.y = image_of(io->y, sh);
    return gate_launch(p, sh, a, false, static_cast<cudaStream_t>(stream));
}

extern "C" adop_status adop_gated_activation_backward(const adop_norm_params* p, const adop_norm_io* io, void* stream)
{
    ADOP_TRY(check_params(p, false));
    if (!io) return refuse(ADOP_ERR_INVALID_ARGUMENT, "no tensors");
    if (p->batch == 0 || p->pixels == 0) return ADOP_OK;
    ADOP_TRY(check_image(p, io->x, false, "x"));
    ADOP_TRY(check_image(p, io->gate, false, "gate"));
    ADOP_TRY(check_image(p, io->grad_y, false, "grad_y"));
    ADOP_TRY(check_image(p, io->grad_x, true, "grad_x"));
    ADOP_TRY(check_image(p, io->grad_gate, true, "grad_gate"));
    const adop_norm_image* images[5] = {&io->x, &io->gate, &io->grad_y, &io->grad_x, &io->grad_gate};
    const Shape sh = choose_shape(p, images, 5);
    NormArgs a = args_of(p, sh, false);
    a.x = image_of(io->x, sh);
    a.gate = image_of(io->gate, sh);
    a.dy = image_of(io->grad_y, sh);
    a.dx = image_of(io->grad_x, sh);
    a.dgate = image_of(io->grad_gate, sh);
    return gate_launch(p, sh, a, true, static_cast<cudaStream_t>(stream));
}
