// Beam drafting: selection over a sequence's beams and the vocabulary, and reordering of
// the beams' states (beam_kernels.cu).
#pragma once

#include "common.cuh"

namespace dels {

constexpr int kBeamMax = 64;         // beams of a sequence, read or selected
constexpr int kBeamGroup = 256;      // logits of a group, the unit a warp scans at a time
constexpr int kBeamMaxGroups = 2048; // groups of a row: at most 524288 logits
constexpr int kBeamThreads = 256;

// One (value, token) entry of a row's list of best candidates.
struct BeamEntry {
  float x;
  int token;
};

// Scratch of one selection.  A row is a beam of a sequence; its V logits are cut into
// `groups` groups of kBeamGroup logits, and its scan into `slices` CTAs.
struct BeamScratch {
  uint32_t* group_key;  // [rows][groups] ordered maxima
  float2* part;         // [rows][slices] running maximum and sum of a slice
  BeamEntry* best;      // [rows][select] the row's candidates, best first
  float2* stat;         // [rows] maximum, cum - log(sum)
};

struct BeamSelectArgs {
  const void* logits;        // [rows, V], row stride ld
  long long ld;
  const void* base;          // [n_seq, V] shared by a sequence's beams, or null
  long long ld_base;
  const float* prior;        // [V] or null
  const float* beta;         // [1], with prior
  const float* cum;          // [rows] accumulated scores
  const uint8_t* finished;   // [rows] or null
  int pad_token;
  int n_seq, beams, select, V;
  int groups, slices;
  int* parents;              // [n_seq, select]
  long long* tokens;         // [n_seq, select]
  float* scores;             // [n_seq, select]
  BeamScratch ws;
};

template <typename T, bool MIX, bool VEC>
__global__ void beam_scan_kernel(const BeamSelectArgs a);
template <typename T, bool MIX>
__global__ void beam_row_kernel(const BeamSelectArgs a);
__global__ void beam_merge_kernel(const BeamSelectArgs a);

// One state of the beams: rows x outer x inner contiguous bytes.
struct BeamState {
  const char* src;
  char* dst;
  long long src_row, dst_row, src_outer, dst_outer;  // strides in bytes
  long long inner;                                   // bytes
  int outer;
  int chunk;         // bytes of one tile's piece of `inner`
  int width;         // bytes moved at once: 16, 8, 4, 2 or 1
  int chunks;        // pieces of `inner`
  long long tile0;   // first tile of this state
};

constexpr int kBeamStatesPerLaunch = 32;

struct BeamReorderArgs {
  BeamState st[kBeamStatesPerLaunch];
  int n_states;
  const int* parents;  // [n_seq, select]
  int n_seq, beams, select;
  int* status;         // or null
  long long tiles;
};

constexpr int kBeamReorderSmem = 32768;

__global__ void beam_reorder_kernel(const __grid_constant__ BeamReorderArgs a);

}  // namespace dels
