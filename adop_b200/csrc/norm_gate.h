// Group normalisation with an activation and the gate of a gated convolution on channels-last images: what the host side
// (norm_gate.cu) and the kernels (norm_gate.cuh, compiled once per image type) share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace adop {

enum NormKernel
{
    kNormStats,         // sums of u and u^2 per group
    kNormApply,         // y = act((u - mean) rstd w + b)
    kNormGradSums,      // per channel: sums of dz and dz uhat
    kNormGradApply,     // dx, and the parameters' gradients from the sums
    kNormResident,      // forward pass of images that fit a block's shared memory
    kGate,              // y = act(f) sigmoid(g)
    kGateGrad,          // df, dg
    kNormKernels
};
enum NormVector { kVec16, kVec8, kVec4, kVec1, kNormVectors };  // bytes of a thread's vector; kVec1 = one element (kVec4: of 16-bit images)

// One channels-last tensor: element (b, pixel, c) at p + b * image + pixel * (row / pixels per row) + c; strides in elements.
struct NormImage
{
    const void* p;
    int64_t image, row;
};

// An image's rows in parts: `rows` each, the first `more` of them one more.
struct NormParts
{
    int count, rows, more;
};

// An image is walked in rows of P vectors: P vectors of VEC elements are the smallest run that starts and ends with a pixel,
// so a thread that moves on by whole rows keeps its channels, and with them its coefficients and its sums, in registers.
// 352 bytes, no gaps: with 360 a small gate's call took 5.3 us on the host for 4.9.
struct NormArgs
{
    int C, G, Cg;     // channels and groups of a slice; channels of a group
    int slices;       // log2 of the independent channel ranges of an image (0 but in the resident kernel)
    int P, ppr;       // vectors and pixels of a row
    int R;            // rows that a block takes at once (1 when a row has more vectors than the block threads)
    int m;            // channels of a thread's vector that share a group: gcd(Cg, VEC)
    int lanes, row_lanes;  // log2 of the threads of a warp that add up one group's sums, and of those for one slot's rows
    int warps;        // warps that add up one group's sums
    int rows;         // rows of an image
    int image0;       // first image of the launch
    NormParts sums;   // parts of an image that have a partial sum each
    NormParts own;    // parts that the blocks of the launch take
    int part0;        // the sums' block k takes part part0 + k part_step (below)
    double inv_n, inv_short, inv_long;     // 1 / values of a group in the image, in a part, in one with a row more
    int gather;           // log2 of the threads that add up a group's partial sums
    float inv_P, inv_Cg;
    int param_blocks; // blocks of kNormGradApply that add up the parameters' gradients
    int param_parts;  // partial sums of a channel, over all images
    int vectors;      // bytes of shared memory in front of the vectors
    int act, param_type;
    float eps;
    int part_step;
    NormImage x, gate, y, dy, dx, dgate;
    const void *weight, *bias;
    void *dweight, *dbias;
    float *mean, *rstd;   // [B, G of all slices]
    float2* group_part;   // [B, G, chunks]
    float2* channel_part; // [B, chunks, C]
};

// Threads of a block and resident blocks of an SM that the kernels are compiled for: 64 registers forward and 80 backward, where a vector's
// eight channels have four coefficients each. 256 threads with 128 registers hold too few vectors back from memory. Forward nothing spills;
// backward some kernels of 16-byte vectors of 16-bit images spill 4 to 20 bytes (the last launch, gated or with SiLU, and the sums behind an
// activation without a gate), with 512 threads and 64 registers all of them, 20 to 120 bytes.
constexpr int kNormThreads = 512, kNormBlocks = 2;          // forward
constexpr int kNormGradThreads = 384, kNormGradBlocks = 2;  // backward
// vectors that the streaming kernels have under way for each thread: a power of two
__host__ __device__ constexpr int stream_depth(bool gated, bool grad) { return gated ? 4 : 8; }
// vectors in a row that a thread adds up in 32 bits; those of one or two elements go on in a second chain then, which takes four registers
constexpr int kChain = 256;
__host__ __device__ constexpr bool second_chain(int vec) { return vec <= 2; }
constexpr int kParamChannels = 32;  // channels whose parameters' gradients one block adds up

static_assert(sizeof(NormArgs) == 352, "the arguments' size is felt on the host");

const void* norm_kernel_f32(int which, int vec, bool gated, int act);
const void* norm_kernel_f16(int which, int vec, bool gated, int act);
const void* norm_kernel_bf16(int which, int vec, bool gated, int act);

}  // namespace adop
