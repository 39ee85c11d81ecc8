// What csrc/host/draft_ops.cpp packs for the launchers of the operators of a step that verifies drafted tokens: included by both sides.
#pragma once
#include <vector_types.h>

struct StArgs {                       // aie_step_tables
    const int *cached, *counts, *held_in, *tables_in, *free_pages, *free_count;      // [R], [R], [R], [R, W], [F], [1]
    int* out;                         // tables [R, W], held [R], free_left [1], q_start [R], q_len [R], then positions, token_req, slots [capacity]
    unsigned* err;
    int R, W, F, P, num_pages, capacity;      // num_pages * P fits 31 bits
};

struct CwArgs {                       // aie_write_kv_slots
    const void *k, *v;                // [T, K, d], elements k_token / k_head (v_token / v_head) apart between tokens and heads
    void *k_pages, *v_pages;
    const int* slots;
    unsigned* err;
    long long k_token, k_head, v_token, v_head;
    int row_dtype, cache_dtype, T, num_pages, P, K, d;      // num_pages * P and 2 * K * d fit 31 bits
};

struct VdArgs {                       // aie_verify_drafts
    const float* target;              // rows of V floats, target_row apart
    const int *q_start, *draft_tokens, *draft_len;      // [R], [R, N], [R] or null: N each
    const float* draft_probs;         // row i of request r at r * draft_req + i * draft_place, or null
    const float *accept_draws, *token_draws;            // [R, N], [R]
    int *tokens, *emitted;            // [R, N + 1], [R]
    unsigned* err;
    long long target_row, draft_req, draft_place;
    int T, V, R, N;
};

struct ChCall {                       // aie_attention_chunks_*
    const void* q;                    // [T, H, d], elements q_token / q_head apart
    const void* k_pages;              // [num_pages, K, P, d]
    const void* v_pages;
    void* out;                        // [T, H, d]
    const int *q_start, *q_len, *ctx_len, *table;
    float* part_o;                    // [2 * blocks][M][D]
    float* part_ml;                   // [2 * blocks][M][2]
    int4* meta;                       // [blocks] of the item that a block began and did not finish: key head, first row, rows and 2^16 parts (0: none), first token
    long long q_token, q_head;
    int R, W, T, num_pages, P, H, K, G, d, window;
    float scale2;                     // scale * log2 e: exponentials are powers of two
    unsigned* err;
    int blocks;                       // that share the line, and that the three above are made for; 0: clusters, which need none
};
