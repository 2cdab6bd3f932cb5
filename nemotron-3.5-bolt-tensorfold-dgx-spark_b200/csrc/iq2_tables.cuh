// The ggml IQ2_XXS tables, for the kernels that decode IQ2_XXS weights.
#pragma once
#include <cstdint>

// The ggml tables are taken from the reference's own table file by path at build time (B200Q_IQ2_TABLES), never
// re-typed: kmask_iq2xs[8], ksigns_iq2xs[128], ksigns64[128], iq2xxs_grid[256] (engine/iq2_tables.inc:1-117).
#define GGML_TABLE_BEGIN(type, name, size) static __device__ const type name[size] = {
#define GGML_TABLE_END() };
#include B200Q_IQ2_TABLES
#undef GGML_TABLE_BEGIN
#undef GGML_TABLE_END
