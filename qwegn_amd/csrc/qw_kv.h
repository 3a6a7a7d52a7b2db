// The paged MXFP4 cache, shared by the door that fills it and the attention that reads it: where a piece (one page of one head) keeps its planes.
#pragma once
#include "qw_mxfp4.h"

struct qw_kv_geometry {
    uint32_t page_log2;     // tokens of a page
    uint32_t piece;         // bytes of a page of one head
    uint32_t k_scales, v_codes, v_scales;   // byte offsets in a piece; the keys' codes are at 0
};
static inline qw_kv_geometry qw_kv_geometry_of(const qwhip_kv_cache* c) {
    const uint32_t codes = c->page_size * c->head_dim / 2u, scales = c->page_size * c->head_dim / 32u;
    return {(uint32_t)__builtin_ctz(c->page_size), 2u * (codes + scales), codes, codes + scales, 2u * codes + scales};
}
