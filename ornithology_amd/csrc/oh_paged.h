// oh_paged.h - the paged key/value pool: its layout, and what the kernels of
// oh_kernels_paged.hip and oh_kernels_pattn*.hip and their host side share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// Element types of rows and of the pool (ggml numbers; OH_PT_Q8: int8 codes
// with one f32 scale per position and head)
enum { OH_PT_F32 = 0, OH_PT_F16 = 1, OH_PT_Q8 = 8, OH_PT_BF16 = 30 };
// what a kernel reports in the pool's fault word
enum { OH_PF_PAGE = 1, OH_PF_POSITION = 2, OH_PF_BATCH = 4 };

// A pool. One block of memory per (page, head): keys, values, and for 8-bit
// pools the keys' and the values' scales. Keys and values are kept in tiles of
// 32 positions, in the order in which a wave of the attention kernels loads
// them as matrix operands, 16 bytes a lane, so that they need no shuffle on
// the way in:
//   keys: units of 16 bytes of one position (8 values, or 16 codes), the 32
//     positions of a dim group side by side;
//   values: per position group g (of four) and dim, the 8 positions
//     4g..4g+3 and 16+4g..16+4g+3: those whose probabilities a lane of group
//     g holds after S^T = K Q^T.
struct oh_pool {
    uint8_t *mem;
    int32_t *fault;
    int32_t nkv, hd, type, page_sh, n_pages;    // page_sh: log2 of positions per page
    uint32_t v_off, ks_off, vs_off;             // in a (page, head) block
    uint32_t block;                             // bytes of one
    // rotation: (cos, sin) of 1024-position steps and of the positions within
    // one, in 64 bits, per frequency; their product's angle is the position's
    const double2 *rope_hi, *rope_lo;
    const uint8_t *rope_axis;
    int32_t rope_dim, max_pos;
};
constexpr int kRopeStep = 1024;

// rows [start[s], start[s + 1]) of sequence s sit at its positions ending at
// len[s] - 1; table[s]: its pages
struct oh_pbatch {
    const int32_t *start, *len, *table;
    int32_t n_seq, n_rows, max_pages, max_new;
};

// rows of heads: element (r, h, d) at p + r * rs + h * hs + d
struct oh_prows { void *p; int64_t rs, hs; };

struct oh_pappend {
    oh_pool pool;
    oh_pbatch b;
    oh_prows q, q_out, k, v;                    // q.p null: no queries
    const float *q_norm, *k_norm;               // null: none
    float eps;
    const int32_t *pos;                         // null: the cache position on every axis
    int64_t pos_stride;                         // between axes
    int32_t axes;                               // that the pool's frequencies name
    int32_t nh, type;                           // type of all rows
};

struct oh_pattn {
    oh_pool pool;
    oh_pbatch b;
    oh_prows q, out;
    float scale, sign;                          // |scale| times log2(e): scores are powers of two
    int32_t nh, G, type;
    // shared prefixes: group i: sequences [gfirst[i], gfirst[i + 1]), the
    // whole pages within its glen[i] positions
    const int32_t *gfirst, *glen;
    int32_t n_group;
    // Parts of the key axis, at most (short stretches have fewer), and positions
    // of one, at least: of the sequences that the kernel for few rows takes, of
    // those that the one for many takes, of the groups' prefixes
    int32_t parts, mparts, gparts;
    int32_t least, mleast, gleast;
    // sequences of up to `few` rows (times heads of a group) go to the one, of
    // more than `many` (-1: none) to the other; prefixes by gmany
    int32_t few, many, gmany;
    int32_t mrows, grows;                       // rows of a block of the latter: 128, or up to oh_pattn_many_rows
    // Partial results, not divided by the sum, [..][hd], and their running maximum
    // (log2) and sum: of row j of sequence s, head h and part c at ((s * few_rows +
    // j) * nh + h) * parts + c; of row r of one with many rows at (r * nh + h) *
    // mparts + c; of row r over its group's prefix at (r * nh + h) * gparts + c
    int32_t few_rows;
    float *po, *mpo, *gpo;
    float2 *pml, *mpml, *gpml;
};

// a launch of so many blocks of 256 threads is within the runtime's limits
constexpr int64_t kMaxBlocks = (1 << 24) - 1;

extern "C" {
hipError_t oh_launch_rope_tables(double2 *t, int steps, int half, double theta, hipStream_t st);
hipError_t oh_launch_paged_append(const oh_pappend *a, hipStream_t st);
hipError_t oh_launch_paged_read(const oh_pappend *a, hipStream_t st);
hipError_t oh_launch_pattn_few(const oh_pattn *a, hipStream_t st);    // the sequences' (few) and the prefixes' (not gmany)
hipError_t oh_launch_pattn_many(const oh_pattn *a, hipStream_t st);   // the sequences' (many) and the prefixes' (gmany)
hipError_t oh_launch_pattn_f32(const oh_pattn *a, hipStream_t st);    // the same for f32 rows
hipError_t oh_pattn_many_rows(const oh_pattn *a, int *rows);          // of a block, at most, for a's types
hipError_t oh_launch_pattn_join(const oh_pattn *a, hipStream_t st);
}
