// Records of a plan for the attention of a step's rows over 8-bit pages (attend_plan.hip writes them, attend.hip reads them).
//
// A virtual row of a KV head is (row, query head of the group): row r of a request and head g are virtual row r G + g. A tile is
// a run of virtual rows that reads keys once for all of them: of one request over its own pages, or of all requests behind
// a shared prefix over the prefix's pages. A tile's pages are cut into units, one workgroup for each KV head; the units of
// a tile leave partial results (maximum, sum, accumulators) wherever there is more than one of them, or a shared prefix
// besides, and the join adds them up.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "internal.hpp"

namespace kvs {

constexpr int TILE_FEW = 16;    // virtual rows of a small tile
constexpr int TILE_MANY = 128;  // of a large one
constexpr int MAX_ATTEND_B = 2048, MAX_SHARED = 64, MAX_TILE_UNITS = 128;

struct alignas(16) AttendUnit {
  int kind;      // 1: a large tile; 2: over a shared prefix
  int row0;      // first row of the request; over a shared prefix first entry of its requests' rows
  int v0, nv;    // virtual rows [v0, v0 + nv)
  int p0;        // position of the request's first row
  int pre;       // keys before this position are seen by every row
  int table;     // row of the block table, or of the shared prefixes'
  int len;       // keys in the pages
  int base;      // position of the first of them
  int a1, b0;    // pages [0, a1), then from b0 on
  int i0, n;     // this unit's of that list
  int part;      // first row of the partial results, -1: the result itself
  int spare[2];
};
static_assert(sizeof(AttendUnit) == 64, "a unit is one line");

constexpr int JOIN_ROWS = 8;
struct alignas(16) AttendJoin {  // a run of virtual rows whose partial results are added up
  int row0, v0, n;               // first row of the request; virtual rows [v0, v0 + n)
  int part, ns, step;            // partial rows part + i + s step of row v0 + i, s < ns: over its own pages
  int more, more_ns, more_step;  // and over its shared prefix's
  int spare[3];
};

struct AttendRow {  // a row behind a shared prefix
  int row, pos, pre, spare;
};
struct alignas(16) AttendTile {  // scratch of the plan
  int who, v0, pages, part;
  int nv, ns, spare[2];
};

// Sizes of a plan and where its parts lie in the workspace (int32 elements).
struct AttendSizes {  // (host)
  bool large;        // large tiles occur
  int few, many;     // heights (many 0: small tiles only)
  int64_t tiles, joins, units, part_rows;
  int64_t at_units, at_joins, at_tiles, at_rows, total;
};

// The workspace's first elements: units, joins, the requests' first row and the one after their last.
constexpr int HEAD = 16;
enum { H_UNITS = 0, H_JOINS = 1, H_FIRST = 2, H_LAST = 3 };

AttendSizes attend_sizes(const kvskip_attend_plan_args& p);

hipError_t launch_attend_plan(const kvskip_attend_plan_args& p, const AttendSizes& z, hipStream_t s);
hipError_t launch_attend(const kvskip_attend_args& a, const AttendSizes& z, hipStream_t s);
hipError_t launch_norm_rope(const kvskip_rope_args& a, hipStream_t s);

}  // namespace kvs
