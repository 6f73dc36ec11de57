// CPU-side entry points for the host+device math headers, so that the 3x3
// rotation fit can be checked against LAPACK without a GPU.  Built by
// visual_odometry_amd.build.build_host_checks(); only the host half is ever run.
#include "../visual_odometry_amd/csrc/vo_packed.h"
#include "../visual_odometry_amd/csrc/vo_svd3.h"

// Where every row tile of packed sequences lies: out (tiles, 6) = any, first row, q0, Lq, k0, Lk; returns the tiles.
extern "C" int64_t host_row_tiles(const int* q_off, const int* k_off, int sequences, int64_t q_tokens, int64_t k_tokens,
                                  int rows_per_token, int rows_per_tile, int64_t* out) {
    const int64_t n = vo_tiles_bound(q_tokens, sequences, rows_per_token, rows_per_tile);
    for (int64_t t = 0; out && t < n; ++t) {
        const vo_place p = vo_find_tile(q_off, k_off, sequences, q_tokens, k_tokens, (unsigned)t, rows_per_token, rows_per_tile);
        const int64_t row[6] = {p.any, p.row, p.q0, p.Lq, p.k0, p.Lk};
        for (int i = 0; i < 6; ++i) out[6 * t + i] = row[i];
    }
    return n;
}

extern "C" void host_rotation_from_covariance(const double* H9, double* R9) {
    double H[3][3], R[3][3];
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j) H[i][j] = H9[3 * i + j];
    rotation_from_covariance(H, R);
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j) R9[3 * i + j] = R[i][j];
}
