// What the entry points of steps over token trees share with the host: structures that a program fills once and keeps (ops/tree.py), so that a
// call of a few microseconds does not hand over thirty numbers one by one.
#pragma once
#include "common.cuh"

constexpr int kTreePage = 16, kTreeNodes = 64, kTreeRequests = 1024;

struct B2TreeStep {
  int* block_table;             // [requests][max_blocks]
  const int* tree_table;        // [requests][tree_blocks]
  int *lengths, *row_start, *row_req, *row_pos, *slots, *parents;
  unsigned long long* masks;
  int* status;
  int requests, max_blocks, tree_blocks, max_rows, max_nodes, num_pages;
};

struct B2TreePool {
  int *free, *n_free, *held;
  int capacity;
};

struct B2TreeCache {
  CUtensorMap map_k, map_v;     // bf16: rows of D in boxes of 16 x 64 (b2_tree_cache)
  void *k, *v;
  float *k_scale, *v_scale;     // null: bf16
  long long layer_bytes, layer_scales;      // from layer to layer
  int layers, pages, heads, d;
};

struct B2TreeAccepted {
  int *path, *count, *next_token, *lengths;
};
