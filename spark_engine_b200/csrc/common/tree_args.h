// Arguments of the kernels for drafted trees over paged caches (tree_rows.cu, tree_attn.cu), shared with the bindings that fill them.
#pragma once
#include <stdint.h>

namespace spark {

// This file as a number (given by the build): the bindings launch only kernels that were compiled from the same one.
#ifndef SPARK_TREE_LAYOUT
#define SPARK_TREE_LAYOUT 0u
#endif

constexpr int TREE_PAGE = 64;

struct BlockTables {
  const int* lengths;                    // [S] tokens a request needs room for; negative: the request is left as it is
  int *tables, *held;                    // [S, ld] pages in position order, -1 behind the held ones; [S]
  int *free, *n_free;                    // stack of free pages: free[0 .. n_free)
  int *room, *status;                    // [S] tokens a request has room for afterwards
  int S, ld, cap;                        // cap: entries of `free`
};

struct SlotMaps {
  const int *lengths, *counts, *tables, *slots, *parents;    // slots (optional): a request's row of the tables; parents (trees): [R]
  int *starts, *slot, *index, *pos, *anc;                    // [S + 1], [R] each, [R, words]
  long long* cache_row;                                      // [R]
  int* status;
  int S, R, ld, n_slots, nodes, words;
};

struct PathConv {
  const void* x; const float* w; const void* tail;           // [R, ldx]; [taps, C]; [slots, taps - 1, C]
  void *q, *k, *v;                                           // q [R, nq]
  const int *slot, *index, *parents;                         // parents null: chains
  const long long* cache_row;
  int* status;
  long long k_page, k_tok, v_page, v_tok, cache_rows;        // strides in elements
  int ldx, R, C, taps, nq, nk, n_slots;
};

struct CommitJob {
  char* base;                            // a cache, or the tail of a convolution
  const char* x;                         // null: a cache; else the rows behind the tail
  long long page, tok;                   // bytes: strides of a cache's pages and tokens, or of a slot's entries (tok) and of x's rows (page)
  int bytes, kept;                       // bytes of a row (multiple of 16); a slot's entries
};
constexpr int COMMIT_JOBS = 128;
struct CommitPaths {
  CommitJob job[COMMIT_JOBS];
  const int *path, *n_path, *starts, *lengths, *slots, *tables;
  int* status;
  int S, P, ld, n_slots, pages;          // pages: of the caches of the whole call, the fewest (-1: it has none)
};

struct TreeAttn {
  const void *q, *k, *v;                 // q [R, H, D] (rows ldq, heads hq apart); caches of pages of 64 tokens of G heads
  void* out;                             // [R, H, V] (rows ldo, heads ho apart)
  const int *starts, *lengths, *slots, *pos, *pages;
  const uint32_t* anc;                   // [R, words] (null: rows see the rows before them)
  const float *bias, *slopes, *sink;     // [H, bias_n], [H], [H]
  const void* gate;                      // [R, H], rows ldg apart
  float *part_o, *part_ml;               // [ctas][2][V / 8][bm][8], [ctas][2][bm][2]: of a tile begun before the CTA, of one that goes on behind it
  int* split;                            // [ctas]: the item that begins in this CTA and ends in another, see ta_split
  int* status;
  long long k_page, k_tok, v_page, v_tok;                    // strides in elements
  int S, R, words, page_ld, n_slots, n_pages, H, G, D, V, ldq, hq, ldo, ho, ldg, bias_n, window, chunk, chunk_shift, bm_log, sms, ctas, extra, zero_rest;
  unsigned chunk_mul;
  float scale, cap, out_scale;
};

}  // namespace spark
