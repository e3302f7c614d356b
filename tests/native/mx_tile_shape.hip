// Compiles where the shape's stages and scale buffers wait for each other, and fails on Tile's assertion where not.
#include "mxfp4_gemm.hip"

int main() { return tb::ntg::mx::Tile<SHAPE>::LDS_BYTES == 0; }
