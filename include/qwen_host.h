/* qwen_host — deterministic host math of the DiT path (reference
 * qwen_host.h:1-111): sigma schedule, Euler step, RoPE tables, latent grid
 * and the seeded PCG32 + Box-Muller RNG used for synthetic inputs. Same
 * names, constants and semantics as the reference; own implementation. */
#ifndef QWEN_HOST_H
#define QWEN_HOST_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QWEN_TRAIN_TIMESTEPS 1000.0
#define QWEN_SCHED_BASE_SEQ_LEN 256
#define QWEN_SCHED_MAX_SEQ_LEN 8192
#define QWEN_SCHED_BASE_SHIFT 0.5
#define QWEN_SCHED_MAX_SHIFT 0.9
#define QWEN_SCHED_SHIFT_TERMINAL 0.02
#define QWEN_MAX_STEPS 1000

#define QWEN_VAE_SPATIAL_RATIO 16
#define QWEN_Z_DIM 64
#define QWEN_HIDDEN 4096
#define QWEN_HEADS 32
#define QWEN_HEAD_DIM 128
#define QWEN_DIT_LAYERS 32
#define QWEN_MLP_RATIO 3
#define QWEN_MLP_HIDDEN (QWEN_HIDDEN * QWEN_MLP_RATIO)
#define QWEN_TEXT_HIDDEN 4096
#define QWEN_EPS 1e-6f

#define QWEN_ROPE_AXES 3
#define QWEN_ROPE_THETA 10000.0
#define QWEN_ROPE_POS_ROWS 8192
#define QWEN_ROPE_NEG_ROWS 1024
#define QWEN_ROPE_ROWS (QWEN_ROPE_POS_ROWS + QWEN_ROPE_NEG_ROWS)

/* reference qwen_host.h:50 */
int qw_latent_grid(int width, int height, int *latent_w, int *latent_h);
/* reference qwen_host.h:55 */
double qw_calculate_shift(int image_seq_len);

typedef struct {
    int steps;
    float sigma[QWEN_MAX_STEPS + 1];
} qw_sigma_schedule;

/* reference qwen_host.h:66 */
int qw_schedule_build(int steps, int image_seq_len, qw_sigma_schedule *schedule);
/* reference qwen_host.h:70-71 */
int qw_schedule_from_sigmas(const float *sigmas, int steps,
                            qw_sigma_schedule *schedule);
/* reference qwen_host.h:75-76: sample += (sigma - sigma_next) * velocity */
void qw_euler_velocity_step(float *sample, const float *velocity,
                            size_t count, float sigma, float sigma_next);

typedef struct {
    int axes;
    int axis_dim[QWEN_ROPE_AXES];
    float *cos;
    float *sin;
} qw_rope_tables;

/* reference qwen_host.h:90-97 */
int qw_rope_build(const int *axis_dim, int axes, qw_rope_tables *tables);
void qw_rope_free(qw_rope_tables *tables);
int qw_rope_row(int coordinate);

/* Rotary frequencies of a text model, for qw_gpu_rotary_bf16. No counterpart
 * in the reference, whose tables are the image model's. Pair i of n / 2 (n =
 * rotary_dim) turns by f_i = base^(-2 i / n) radians a position, stretched for
 * contexts past the original length L by
 *   LINEAR    f / factor
 *   NTK       base * factor^(n / (n - 2)) in place of base
 *   BY_PARTS  f (k + (1 - k) / factor), k = clamp((L f / 2 pi - low) / (high -
 *             low)): pairs of more than `high` turns over L stay, of fewer
 *             than `low` are divided
 *   YARN      the same with k by the pair's index: 1 up to the pair of `high`
 *             turns over L (rounded down), 0 from that of `low` turns (rounded
 *             up) on, linear between; attention factor 0.1 ln(factor) + 1
 * rotary_dim is even, 2 to 256; base > 1; factor >= 1; original_length > 0 and
 * 0 < low < high where they are used. */
enum { QW_ROPE_PLAIN = 0, QW_ROPE_LINEAR = 1, QW_ROPE_NTK = 2, QW_ROPE_BY_PARTS = 3, QW_ROPE_YARN = 4 };
typedef struct {
    uint32_t rotary_dim;
    int scaling; /* QW_ROPE_* */
    double base, factor, original_length, low, high;
} qw_rope_config;
/* turns[i][0], [1]: the high and low half of f_i / 2 pi modulo 1 as a 64-bit
 * fraction (rounded to nearest; up to the 53 bits of a double below its first
 * one bit), so that position * turns is exact modulo a turn. attention_factor
 * (NULL: not wanted): what the rotated part is multiplied by, 1 but for YARN.
 * 0 and a message for a config outside the ranges above. */
int qw_rope_turns(const qw_rope_config *config, uint32_t *turns, float *attention_factor,
                  char *error, size_t error_size);

typedef struct {
    uint64_t state;
    uint64_t increment;
    float spare;
    int has_spare;
} qw_rng;

/* reference qwen_host.h:106-109 */
void qw_rng_seed(qw_rng *rng, uint64_t seed);
uint32_t qw_rng_u32(qw_rng *rng);
float qw_rng_normal(qw_rng *rng);
void qw_rng_fill_normal(qw_rng *rng, float *values, size_t count);

#ifdef __cplusplus
}
#endif
#endif
