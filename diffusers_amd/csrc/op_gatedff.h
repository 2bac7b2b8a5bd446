// op_gatedff.h — argument block and launchers of the gated feed-forward's products.
#pragma once
#include "ops.h"

enum GffEpi { GFF_FWD, GFF_BWD, GFF_STORE, GFF_PART };                      // h; [da dg]; the product; the product of a part of the contraction, fp32
enum GffWhat { GFF_X_WT_FWD, GFF_X_WT_BWD, GFF_DAG_W, GFF_DAGT_X };         // x W^T with either epilogue, [da dg] W, [da dg]^T x
struct GffDev {
    const char* A; const char* B;       // first element of row / contraction 0
    long long ldA, ldB;                 // bytes
    int rowsA, rowsB, Kc;               // rows of the output, columns of the output, contraction length
    long long gate;                     // FWD / BWD: byte offset of the gate rows in B
    int F;
    const void* bias; int bias_f32;
    char* out; long long ld_out;        // elements
    const char* dh; long long ld_dh;    // BWD
    float* colsum;                      // BWD: [row parts][2F], or null
    float* part;                        // PART: [splits][rowsA][rowsB]
    int splits, nbm, nbn;
};
// cfg: 0 = 256 x 256, 1 = 128 x 128, 2 = 64 x 64 tiles; each leaves two row parts of column sums to a row of tiles
void gff_launch_f16(const OpCtx& c, const GffDev& d, int what, int act, int cfg);
void gff_launch_bf16(const OpCtx& c, const GffDev& d, int what, int act, int cfg);
void gff_launch_f32(const OpCtx& c, const GffDev& d, int what, int act, int cfg);
