// Launch API of the gfx950 optimizer kernels (implemented in
// adamw_kernels.hip). Pure HIP host interface, like gar_kernels.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace adamw {

// Element types of parameters and gradients.
enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// Elements that share one scale in an 8-bit state.
constexpr int kGroup = 32;
// Elements that one workgroup updates: few, so that its registers leave room
// for eight waves a SIMD and small tensors spread out. With 8-bit states, whose
// vector work is what the memory barely hides, two quads a thread share what a
// workgroup computes once, where there is enough to fill the card all the same
// (four workgroups a CU). Measured, 1024 / 2048 a workgroup: 8 bits 1.8M
// elements 8.3 / 8.5 us, 3.5M 15.9 / 14.1, 47M 141 / 128; 32 bits 80k 4.0 / 4.4,
// 26M 116 / 118.
constexpr long kChunkSmall = 1024, kChunkLarge = 2048;

inline long chunk_of(int bits, long elements) {
  return bits == 8 && elements >= 1024 * kChunkLarge ? kChunkLarge
                                                     : kChunkSmall;
}

// Tensors of one update launch: their gradients' addresses travel in the
// kernel's arguments, of which there are 4 KiB.
constexpr int kMaxTensors = 448;
// Spans of one norm launch: as many as 4 KiB of arguments hold. (ResNet-50's
// 161 gradients in separate memory: 24.3 us as one launch, 32.4 us as two, and
// where one is enough, up to 176 or up to 200 of them made no difference.) The
// workgroups of one such launch at most (three a CU), and the bytes that one of
// them reads at a time. Measured for VGG-16's bf16 gradient: 512, 768, 1024, 2048
// workgroups 52, 46.7, 47.7, 50.5 us; 8192, 16384, 32768 bytes 54, 47.7, 48.8 us.
constexpr int kMaxSpans = 200;
constexpr int kNormBlocks = 768;
constexpr int kNormChunkBytes = 16384;

// Workgroups of one launch: the threads of a grid's dimension are counted in 32
// bits.
constexpr long kMaxWork = (1l << 32) / 256 - 1;

// What one workgroup updates: `left` elements of a tensor from the element
// `start` on (a multiple of the chunk), where the pointers point. All that it
// needs is in one place, so that its first loads of data wait for one load only.
// 32-bit states: m and r point to floats (r to the mean square itself), ms and
// rs are null. 8-bit states: m and r point to e4m3 codes (r to those of the mean
// square's root), ms and rs to their groups' biased exponents.
struct Work {
  void* p;
  void* m;
  void* r;
  uint8_t* ms;
  uint8_t* rs;
  long start;
  int tensor;
  int left;
  uint32_t key;  // of the rounding's random bits
  int type;      // of p
};

// The gradients of a launch: null where a tensor has none (not where it has no
// elements), and two bits each for their types.
struct Grads {
  const void* g[kMaxTensors];
  uint32_t types[kMaxTensors / 16];
};

struct Hyper {
  double lr, beta1, beta2, eps, weight_decay;
  const float* norm;  // null: no clipping
  double max_norm;
};

// Whether update() has a form for parameters of type p and gradients of type g.
bool supported(int p, int g);

// Arrivals of a launch's workgroups: one counter for all, then kTicketLines for
// a part of them each, every one on a cache line of its own. Zero before the
// first launch; each launch leaves them so.
constexpr int kTicketLines = 32;
constexpr int kTicketInts = 32 * (kTicketLines + 1);

// One AdamW step of the tensors [first, first + count): steps[i] += 1 for those
// that have a gradient. work[0..nwork) is all that there is to do for them, in
// parts of at most `chunk`, and grads.g[i] belongs to tensor first + i.
void update(int bits, long chunk, const Work* work, long nwork, int first,
            int count, int* steps, unsigned* tickets, const Grads& grads,
            const Hyper& hyper, hipStream_t stream);

// Spans of elements that lie back to back in memory: n4t[i] is four times the
// number of elements of span i, and its type; start[i] is its first chunk (of
// kNormChunkBytes) within the launch, start[count] the number of chunks.
struct Spans {
  const void* ptr[kMaxSpans];
  long n4t[kMaxSpans];
  int start[kMaxSpans + 1];
  int count;
};

// Workgroups, and so partial sums, of a launch over these spans.
int norm_blocks(const Spans& spans);

// partials[b] = the b-th workgroup's sum of squares. With tickets (zero before,
// and again after; not shared with a launch that may run at the same time) the
// last workgroup to arrive goes on to out = sqrt(sum of partials).
void norm_partials(const Spans& spans, double* partials, unsigned* tickets,
                   float* out, hipStream_t stream);

// out = sqrt(sum of partials[0..count)).
void norm_finish(const double* partials, int count, float* out,
                 hipStream_t stream);

}  // namespace adamw
