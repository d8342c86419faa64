// Beam drafting: selection over a sequence's beams and the vocabulary, and reordering of
// the beams' states (beam_kernels.cu).
#pragma once

#include "common.cuh"

namespace dels {

constexpr int kBeamMax = 64;         // beams of a sequence, read or selected
constexpr int kBeamGroup = 512;      // logits of a group, the unit a warp scans at a time
constexpr int kBeamScanWarps = 4;    // most warps of a scanning CTA
constexpr int kBeamScanRows = 8;     // most rows a scanning CTA takes together
// Most scanning CTAs of an SM.  64 x 8 beams took 53 us when this was chosen (5: 60, 7 with a
// shorter ring: 53, 8: 54); compensated sums have made that 55.
constexpr int kBeamScanCtas = 6;
constexpr int kBeamFinishWarps = 16; // most warps of a sequence's finishing CTA
constexpr int kBeamFinishCap = 256;  // quarter groups or candidates it lists before it counts exactly
constexpr int kBeamListCap = 192;    // counting exactly: quarter groups or logits a warp lists
constexpr int kBeamFillTokens = 2048; // tokens it searches for logits equal to the bound
constexpr int kBeamRowScratch = kBeamListCap * 12 + 16;

// One (value, token) entry of a row's list of best candidates.
struct BeamEntry {
  float x;
  int token;
};

// Scratch of one selection.  A row is a beam of a sequence; its V logits are cut into
// `groups` groups of kBeamGroup; see beam_scan_kernel for the parts.
struct BeamScratch {
  float4* group_top;  // [rows][groups] maxima of a group's quarters
  float2* part;       // [rows][parts] running maximum and sum of a CTA's share of the row
};

// The scan's CTAs share out the units (all blocks' groups, in order) as evenly as they go: CTA
// c takes [first(c), first(c + 1)), per of them or one more.
struct ScanShare {
  int per, more;  // the first `more` CTAs take per + 1
  __host__ __device__ __forceinline__ int first(int c) const { return c * per + (c < more ? c : more); }
  // the CTA that takes unit u
  __host__ __device__ __forceinline__ int cta(int u) const {
    const int cut = more * (per + 1);
    return u < cut ? u / (per + 1) : more + (u - cut) / per;
  }
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
  int groups, parts;
  int run_rows;              // rows that blocks are cut from: a sequence's where they share logits, else all
  int scan_rows;             // rows of a block, scanned together
  int scan_ctas;
  ScanShare share;
  int finish_split;          // warps of the finishing CTA that share a beam; it has a multiple of them
  int finish_direct;         // the bound comes from the logits themselves, not from group maxima
  int finish_values;         // maxima a lane of them offers for it
  int slot_bytes;            // of its staging ring
  int* status;               // device error word
  int* parents;              // [n_seq, select]
  long long* tokens;         // [n_seq, select]
  float* scores;             // [n_seq, select]
  BeamScratch ws;
};

// Warps that scan a group together, two rows each, and teams of them in a CTA.
__host__ __device__ __forceinline__ int scan_pairs(int rows) { return (rows + 1) / 2; }
__host__ __device__ __forceinline__ int scan_teams(int rows) { return kBeamScanWarps / scan_pairs(rows); }

// The scan's staging rings, one for each team: groups in flight, as many as six CTAs of an SM
// have room for (one of bf16 less made no difference).
constexpr int beam_scan_depth(int elem) { return elem == 2 ? 3 : 2; }
// Bytes of a slot: `rows` rows of a group, and the draft logits and prior they share.
constexpr int beam_slot_bytes(int rows, int elem, bool shared) {
  return rows * kBeamGroup * elem + (shared ? kBeamGroup * (elem + 4) : 0);
}
// Dynamic shared memory of beam_scan_kernel with VEC.
inline int beam_scan_smem(int rows, int elem, bool shared) {
  return scan_teams(rows) * beam_scan_depth(elem) * beam_slot_bytes(rows, elem, shared);
}
constexpr int kBeamScanSmemMax = 65536;  // two rows of fp32: 4 teams x 2 slots x 8 KB

// Dynamic shared memory of beam_finish_kernel.
constexpr int beam_finish_smem(int beams, int select, int warps, int values) {
  const int listing = kBeamFinishCap * 24 + values * 4;
  const int exact = warps * kBeamRowScratch + beams * select * 12;
  return (beams * 8 + 15) / 16 * 16 + (listing > exact ? listing : exact);
}

// The kernels for bf16 or fp32 logits, with 16-byte loads (vec) or without.
using BeamKernel = void (*)(BeamSelectArgs);
BeamKernel beam_scan_kernel_for(bool bf16, bool vec);
BeamKernel beam_finish_kernel_for(bool bf16, bool vec);

// One state of the beams: rows x outer x inner contiguous bytes.
struct BeamState {
  const char* src;
  char* dst;
  long long src_row, dst_row, src_outer, dst_outer;  // strides in bytes
  long long inner;                                   // bytes
  int outer;
  int chunk;         // bytes of one tile's piece of `inner`
  int chunks;        // pieces of `inner`
  long long tile0;   // first tile of this state
};

// States of a launch.  Their 2.5 KB of arguments cost nothing that shows: a list of at most four
// took 3.4 us on the device and 3.7 us of the host's time for two states, as this one does.
constexpr int kBeamStatesPerLaunch = 32;
constexpr int kBeamThreads = 256;

struct BeamReorderArgs {
  const int* parents;  // [n_seq, select]
  int* status;         // or null
  long long tiles;
  int n_states;
  int n_seq, beams, select;
};
struct BeamStates {
  BeamState st[kBeamStatesPerLaunch];
};

// A tile's stage: each beam's piece, up to 15 bytes before it and a word after.
constexpr int kBeamReorderSmem = 33792;
constexpr int kBeamReorderCtas = 5;  // an SM holds: 597 MB of a cache in 98 us; a sixth would wait its turn (126 us)

__global__ void beam_reorder_kernel(const BeamReorderArgs a, const __grid_constant__ BeamStates states);

}  // namespace dels
