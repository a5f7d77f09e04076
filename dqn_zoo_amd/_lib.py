"""ctypes binding of libdqnzoo_hip.so (the C ABI declared in include/dqnzoo_hip.h).

The product path has NO CPU fallback: if the shared library is missing or does
not export a symbol, importing/using it raises immediately (task rule: "the
product path must fail loudly when the HIP extension is missing").
"""

import ctypes
import os

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, 'libdqnzoo_hip.so')

DZ_OK = 0
DZ_ERR_INVALID_ARG = -1
DZ_ERR_HIP = -2
DZ_ERR_UNSUPPORTED = -3

ACT_FAILED = -2           # DZ_ACT_FAILED: the 'action' of a one-launch decision whose seams timed out
ACT_FAILED_MARKER = 2.0   # DZ_ACT_FAILED_MARKER (dz_dense_act)

ST_BAD_VALUE = 1
ST_BAD_TARGET = 2
ST_BAD_INDEX = 4
ST_ZERO_ROOT = 8
ST_NONFINITE_WEIGHT = 16
ST_CHAIN_TIMEOUT = 32

MAX_FIELDS = 8

c_vp = ctypes.c_void_p
c_i64 = ctypes.c_int64
c_int = ctypes.c_int
c_f64 = ctypes.c_double
c_f32 = ctypes.c_float


class FieldDesc(ctypes.Structure):
  _fields_ = [('src', c_vp), ('dst', c_vp), ('row_bytes', c_i64)]


class InsertField(ctypes.Structure):
  """dz_insert_field_t."""
  _fields_ = [('dst', c_vp), ('src_row', c_vp), ('row_bytes', c_i64),
              ('imm', ctypes.c_uint64)]


class PrioSampleArgs(ctypes.Structure):
  _fields_ = [
      ('node', c_vp), ('cap_pow2', c_i64), ('capacity', c_i64),
      ('size', c_i64), ('t', c_i64), ('pos', c_vp), ('u_target', c_vp),
      ('u_mix', c_vp), ('usp', c_f64), ('one_minus_usp', c_f64),
      ('usp_times_up', c_f64), ('uniform_prob', c_f64), ('beta', c_f64),
      ('normalize', c_int), ('compute_weights', c_int),
      ('assume_nonzero_root', c_int),
  ]


c_i32 = ctypes.c_int32


class RainbowLayout(ctypes.Structure):
  _fields_ = (
      [('num_actions', c_i32), ('num_atoms', c_i32), ('batch', c_i32),
       ('groups', c_i32), ('adv2_ld', c_i32), ('val2_ld', c_i32), ('fc1_ld', c_i32), ('pad0_', c_i32),
       ('param_count', c_i64), ('param_count_ref', c_i64),
       ('conv_w', c_i64 * 3), ('conv_b', c_i64 * 3)] +
      [(n, c_i64) for n in (
          'fc1_mu_w', 'fc1_mu_b', 'fc1_sig_w', 'fc1_sig_b', 'adv2_mu_w',
          'adv2_sig_w', 'val2_mu_w', 'val2_sig_w', 'fc2_sig_b', 'noise_stride',
          'n_adv1_in', 'n_val1_in', 'n_fc1_out', 'n_adv2_in', 'n_val2_in',
          'n_fc2_out', 'ws_count', 'ws_act1', 'ws_act2', 'ws_feat',
          'ws_fc1_part', 'ws_h1', 'ws_fc2_part', 'ws_fc2_out', 'ws_dout2',
          'ws_dh1', 'ws_dfeat_part', 'ws_dfeat', 'ws_dact2', 'ws_dact1',
          'ws_wgrad_part', 'ws_norm_part', 'ws_scalars', 'ws_q_sel',
          'ws_target_probs', 'ws_colsum_part', 'ws_act_seams')])


class RainbowArgs(ctypes.Structure):
  _fields_ = [
      ('num_actions', c_i32), ('num_atoms', c_i32), ('batch', c_i32),
      ('online', c_vp), ('target', c_vp), ('grad', c_vp), ('adam_m', c_vp),
      ('adam_v', c_vp), ('adam_count', c_vp), ('s_tm1', c_vp), ('s_t', c_vp),
      ('a_tm1', c_vp), ('r_t', c_vp), ('discount_t', c_vp), ('weights', c_vp),
      ('support', c_vp), ('noise', c_vp), ('ws', c_vp), ('losses', c_vp),
      ('priorities', c_vp), ('lr', c_f32), ('b1', c_f32), ('b2', c_f32),
      ('eps', c_f32), ('max_norm', c_f32), ('resample_noise', c_i32),
      ('noise_seed', ctypes.c_uint64),
      ('prio_node', c_vp), ('prio_cap_pow2', c_i64), ('prio_capacity', c_i64),
      ('prio_ids', c_vp), ('prio_exponent', c_f64), ('prio_max_seen', c_vp),
      ('prio_status', c_vp), ('keep_all_grads', c_i32), ('separate_launches', c_i32),
      ('next_sample', c_vp),
  ]


class NextSample(ctypes.Structure):
  """dz_next_sample_t: the arguments of dz_prioritized_sample_gather, carried by a
  learner step (RainbowArgs.next_sample)."""
  _fields_ = [
      ('args', PrioSampleArgs), ('pos_h', c_vp), ('u_target_h', c_vp), ('u_mix_h', c_vp),
      ('fields', c_vp), ('num_fields', c_i32), ('n', c_i32), ('ids_out', c_vp),
      ('probs_out', c_vp), ('weights_out', c_vp), ('weights32_out', c_vp),
      ('status', c_vp),
  ]


class DenseLayout(ctypes.Structure):
  _fields_ = (
      [('num_outputs', c_i32), ('shared_bias', c_i32), ('batch', c_i32),
       ('groups', c_i32), ('fc1_ld', c_i32), ('fc2_ld', c_i32),
       ('param_count', c_i64), ('param_count_ref', c_i64),
       ('conv_w', c_i64 * 3), ('conv_b', c_i64 * 3)] +
      [(n, c_i64) for n in (
          'fc1_w', 'fc1_b', 'fc2_w', 'fc2_b', 'ws_count', 'ws_act1', 'ws_act2',
          'ws_feat', 'ws_fc1_part', 'ws_h1', 'ws_fc2_part', 'ws_out', 'ws_dout',
          'ws_dh1', 'ws_dfeat_part', 'ws_dfeat', 'ws_dact2', 'ws_dact1',
          'ws_wgrad_part', 'ws_norm_part', 'ws_scalars', 'ws_zeros', 'ws_act_seams')])


class DenseArgs(ctypes.Structure):
  _fields_ = [
      ('loss', c_i32), ('optimizer', c_i32), ('num_actions', c_i32),
      ('num_outputs', c_i32), ('batch', c_i32), ('shared_bias', c_i32),
      ('num_atoms', c_i32), ('online', c_vp), ('target', c_vp), ('grad', c_vp),
      ('opt_m', c_vp), ('opt_v', c_vp), ('opt_count', c_vp), ('s_tm1', c_vp),
      ('s_t', c_vp), ('a_tm1', c_vp), ('r_t', c_vp), ('discount_t', c_vp),
      ('weights', c_vp), ('aux', c_vp), ('ws', c_vp), ('losses', c_vp),
      ('priorities', c_vp), ('lr', c_f32), ('decay_or_b1', c_f32), ('b2', c_f32),
      ('eps', c_f32), ('max_norm', c_f32), ('grad_error_bound', c_f32),
      ('huber', c_f32),
      ('prio_node', c_vp), ('prio_cap_pow2', c_i64), ('prio_capacity', c_i64),
      ('prio_ids', c_vp), ('prio_exponent', c_f64), ('prio_max_seen', c_vp),
      ('prio_status', c_vp), ('next_sample', c_vp),
      ('keep_all_grads', c_i32), ('pad2_', c_i32),
  ]


class IqnLayout(ctypes.Structure):
  """dz_iqn_layout_t."""
  _fields_ = [
      ('num_actions', c_i32), ('latent_dim', c_i32), ('batch', c_i32),
      ('samples', c_i32 * 3), ('emb_ld', c_i32), ('fc1_ld', c_i32),
      ('fc2_ld', c_i32), ('pad_', c_i32),
      ('conv_w', c_i64 * 3), ('conv_b', c_i64 * 3),
      ('emb_w', c_i64), ('emb_b', c_i64), ('fc1_w', c_i64), ('fc1_b', c_i64),
      ('fc2_w', c_i64), ('fc2_b', c_i64),
      ('param_count', c_i64), ('param_count_ref', c_i64), ('ws_count', c_i64),
      ('ws_act1', c_i64), ('ws_act2', c_i64), ('ws_feat', c_i64),
      ('ws_cos', c_i64), ('ws_hin', c_i64), ('ws_temb', c_i64),
      ('ws_h1', c_i64), ('ws_out', c_i64), ('ws_dout', c_i64),
      ('ws_dh1', c_i64), ('ws_dhin', c_i64), ('ws_dfeat', c_i64),
      ('ws_dact2', c_i64), ('ws_dact1', c_i64), ('ws_wgrad_part', c_i64),
      ('ws_fc2w_part', c_i64), ('ws_embw_part', c_i64),
      ('ws_bias_part', c_i64), ('ws_norm_part', c_i64), ('ws_scalars', c_i64),
      ('ws_zeros', c_i64), ('ws_act_seams', c_i64),
  ]


class IqnArgs(ctypes.Structure):
  """dz_iqn_args_t."""
  _fields_ = [
      ('num_actions', c_i32), ('latent_dim', c_i32), ('batch', c_i32),
      ('samples', c_i32 * 3),
      ('online', c_vp), ('target', c_vp), ('grad', c_vp), ('opt_m', c_vp),
      ('opt_v', c_vp), ('opt_count', c_vp), ('s_tm1', c_vp), ('s_t', c_vp),
      ('a_tm1', c_vp), ('r_t', c_vp), ('discount_t', c_vp), ('tau_tm1', c_vp),
      ('tau_sel', c_vp), ('tau_t', c_vp), ('ws', c_vp), ('losses', c_vp),
      ('lr', c_f32), ('b1', c_f32), ('b2', c_f32), ('eps', c_f32),
      ('max_norm', c_f32), ('huber', c_f32),
  ]


LOSS_Q, LOSS_DOUBLE_Q, LOSS_CATEGORICAL, LOSS_QUANTILE = 0, 1, 2, 3
OPT_RMSPROP, OPT_ADAM = 0, 1
SC_GNORM, SC_LOSS, SC_BC1, SC_BC2, SC_CLIP = 0, 1, 2, 3, 4
SC_CHAIN_FAIL = 6
PHASE_FORWARD, PHASE_BACKWARD, PHASE_OPTIMIZER, PHASE_ALL = 1, 2, 4, 7
PHASE_FWD_NETS, PHASE_FWD_LOSS = 8, 16   # the two halves of PHASE_FORWARD

class ReplayInsertArgs(ctypes.Structure):
  """dz_replay_insert_args_t."""
  _fields_ = [('fields', ctypes.POINTER(InsertField)), ('num_fields', c_i32), ('reserved', c_i32),
              ('t', c_i64), ('capacity', c_i64), ('node', c_vp), ('cap_pow2', c_i64),
              ('priority_h', c_f64), ('priority_d', c_vp), ('exponent', c_f64), ('status', c_vp)]


class RainbowActArgs(ctypes.Structure):
  """dz_rainbow_act_args_t."""
  _fields_ = [('num_actions', c_i32), ('num_atoms', c_i32), ('batch', c_i32), ('reserved', c_i32),
              ('params', c_vp), ('states', c_vp), ('noise', c_vp),
              ('noise_seed', ctypes.c_uint64), ('noise_counter', ctypes.c_uint64),
              ('step_counter', c_vp), ('support', c_vp), ('ws', c_vp), ('q_values_out', c_vp),
              ('greedy_out', c_vp), ('vmax_out', c_vp)]


class AdamWTensor(ctypes.Structure):
  """dz_adamw_tensor_t."""
  _fields_ = [('p', c_vp), ('n', c_i64), ('offset', c_i64), ('decay', c_f32), ('reserved', c_i32)]


class AdamWArgs(ctypes.Structure):
  """dz_adamw_args_t."""
  _fields_ = [('param_dtype', c_i32), ('grad_dtype', c_i32), ('state_bits', c_i32),
              ('num_chunks', c_i32), ('tensors', c_vp), ('chunks', c_vp), ('grads', c_vp),
              ('master', c_vp), ('m', c_vp), ('v', c_vp), ('m_scale', c_vp), ('v_scale', c_vp),
              ('count', c_vp), ('lr', c_vp), ('scalars', c_vp), ('partials', c_vp),
              ('b1', c_f64), ('b2', c_f64), ('eps', c_f32), ('max_norm', c_f32),
              ('grad_scale', c_f32), ('reserved', c_i32), ('seed', ctypes.c_uint64)]


class PolicyLossArgs(ctypes.Structure):
  """dz_policy_loss_args_t."""
  _fields_ = [('dtype', c_i32), ('reserved', c_i32), ('rows', c_i64), ('classes', c_i64),
              ('logits', c_vp), ('ld', c_i64), ('actions', c_vp), ('advantages', c_vp),
              ('old_logp', c_vp), ('ref_logp', c_vp), ('weights', c_vp), ('dlogits', c_vp),
              ('ldg', c_i64), ('loss', c_vp), ('logp', c_vp), ('entropy', c_vp),
              ('status', c_vp), ('ws', c_vp), ('ws_bytes', c_i64), ('clip_low', c_f64),
              ('clip_high', c_f64), ('kl_coef', c_f64), ('entropy_coef', c_f64),
              ('normalizer', c_f64), ('grad_scale', c_f32), ('reserved2', c_i32)]


class LinearArgs(ctypes.Structure):
  """dz_linear_args_t."""
  _fields_ = [('dtype', c_i32), ('activation', c_i32), ('m', c_i64), ('k', c_i64), ('n', c_i64),
              ('x', c_vp), ('ldx', c_i64), ('w', c_vp), ('ldw', c_i64), ('w_transposed', c_i32),
              ('bias_f32', c_i32), ('bias', c_vp), ('residual', c_vp), ('ldr', c_i64),
              ('y', c_vp), ('ldy', c_i64), ('preact', c_vp), ('ldz', c_i64), ('dy', c_vp),
              ('lddy', c_i64), ('dx', c_vp), ('lddx', c_i64), ('dw', c_vp), ('lddw', c_i64),
              ('db', c_vp), ('grads_f32', c_i32), ('reserved', c_i32), ('ws', c_vp),
              ('ws_bytes', c_i64)]


# element types of the size-generic operators (DZ_F32 / DZ_BF16 / DZ_F16)
F32, BF16, F16 = 0, 1, 2
ADAMW_STATE_BLOCK, ADAMW_CHUNK = 256, 4096

STRUCT_IDS = {0: FieldDesc, 1: PrioSampleArgs, 2: RainbowLayout, 3: RainbowArgs,
              4: DenseLayout, 5: DenseArgs, 6: IqnLayout, 7: IqnArgs,
              8: InsertField, 9: NextSample, 10: ReplayInsertArgs, 11: RainbowActArgs,
              12: AdamWTensor, 13: AdamWArgs, 14: PolicyLossArgs,
              15: LinearArgs}

# name -> (restype, argtypes).  tests/test_abi.py checks this table against
# the prototypes in include/dqnzoo_hip.h and against the built library.
SIGNATURES = {
    'dz_version': (ctypes.c_char_p, []),
    'dz_last_hip_error': (c_int, []),
    'dz_built_arch': (ctypes.c_char_p, []),
    'dz_struct_size': (c_int, [c_int]),
    'dz_rainbow_layout': (c_int, [c_int, c_int, c_int,
                                  ctypes.POINTER(RainbowLayout)]),
    'dz_rainbow_learn': (c_int, [ctypes.POINTER(RainbowArgs), c_int, c_vp]),
    'dz_rainbow_apply': (c_int, [c_int, c_int, c_int, c_vp, c_vp, c_vp, c_vp,
                                 c_vp, c_vp, c_vp, c_vp, c_vp]),
    'dz_rainbow_act': (c_int, [c_int, c_int, c_int, c_vp, c_vp, c_vp, ctypes.c_uint64,
                               ctypes.c_uint64, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp]),
    'dz_rainbow_graph_capture': (c_int, [ctypes.POINTER(RainbowArgs), c_int, c_vp,
                                         ctypes.POINTER(c_vp)]),
    'dz_atari_observation': (c_int, [c_vp, c_int, c_int, c_int, c_int, c_int, c_vp, c_vp, c_int,
                                     c_vp, c_vp, c_int, c_int, c_int, c_vp, c_int, c_int,
                                     c_int, c_vp, c_vp]),
    'dz_graph_capture_begin': (c_int, [c_vp]),
    'dz_graph_capture_end': (c_int, [c_vp, c_int, ctypes.POINTER(c_vp)]),
    'dz_graph_launch': (c_int, [c_vp, c_vp]),
    'dz_graph_destroy': (c_int, [c_vp]),
    'dz_dense_layout': (c_int, [c_int, c_int, c_int, c_int,
                                ctypes.POINTER(DenseLayout)]),
    'dz_dense_learn': (c_int, [ctypes.POINTER(DenseArgs), c_int, c_vp]),
    'dz_dense_apply': (c_int, [c_int, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_vp,
                               c_vp, c_vp, c_vp, c_vp]),
    'dz_dense_act': (c_int, [c_int, c_int, c_vp, c_vp, c_vp, c_vp, c_vp]),
    'dz_act_debug_spin_limit': (c_int, [c_int]),
    'dz_iqn_layout': (c_int, [c_int, c_int, c_int, c_int, c_int, c_int,
                              ctypes.POINTER(IqnLayout)]),
    'dz_iqn_learn': (c_int, [ctypes.POINTER(IqnArgs), c_int, c_vp]),
    'dz_iqn_apply': (c_int, [c_int, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_vp,
                             c_vp, c_vp, c_vp, c_vp, c_vp]),
    'dz_iqn_act': (c_int, [c_int, c_int, c_int, c_vp, c_vp, ctypes.c_uint64, ctypes.c_uint64, c_vp,
                           c_vp, c_vp, c_vp]),
    'dz_uniform_fill': (c_int, [c_vp, c_i64, ctypes.c_uint64, ctypes.c_uint64,
                                c_vp, c_vp]),
    'dz_noise_fill': (c_int, [c_vp, c_i64, ctypes.c_uint64, ctypes.c_uint64,
                              c_vp]),
    'dz_param_copy': (c_int, [c_vp, c_vp, c_i64, c_vp]),
    'dz_prof_enable': (c_int, [c_int]),
    'dz_prof_read': (c_int, [c_int, c_vp, c_vp]),
    'dz_prof_read_replay': (c_int, [c_vp]),
    'dz_replay_gather': (c_int, [ctypes.POINTER(FieldDesc), c_int, c_vp, c_int,
                                 c_i64, c_vp]),
    'dz_replay_sample_uniform': (c_int, [ctypes.POINTER(FieldDesc), c_int, c_vp, c_int,
                                         c_i64, c_i64, c_i64, c_vp, c_vp]),
    'dz_replay_insert': (c_int, [ctypes.POINTER(InsertField), c_int, c_i64, c_i64,
                                 c_vp, c_i64, c_f64, c_vp, c_f64, c_vp, c_vp]),
    'dz_replay_insert_v': (c_int, [ctypes.POINTER(ReplayInsertArgs), c_vp]),
    'dz_sample_gather_desc': (c_int, [ctypes.POINTER(NextSample), c_vp]),
    'dz_rainbow_act_v': (c_int, [ctypes.POINTER(RainbowActArgs), c_vp]),
    'dz_uniform_pos_to_id': (c_int, [c_vp, c_int, c_i64, c_i64, c_i64, c_vp,
                                     c_vp]),
    'dz_sumtree_set': (c_int, [c_vp, c_i64, c_i64, c_vp, c_vp, c_int, c_vp,
                               c_vp]),
    'dz_sumtree_get': (c_int, [c_vp, c_i64, c_i64, c_vp, c_int, c_vp, c_vp,
                               c_vp]),
    'dz_sumtree_rebuild': (c_int, [c_vp, c_i64, c_i64, c_vp]),
    'dz_sumtree_query': (c_int, [c_vp, c_i64, c_vp, c_int, c_vp, c_vp, c_vp]),
    'dz_prioritized_sample': (c_int, [ctypes.POINTER(PrioSampleArgs), c_int,
                                      c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                      c_vp]),
    'dz_prioritized_sample_host_draws': (c_int, [ctypes.POINTER(PrioSampleArgs), c_int,
                                                 c_vp, c_vp, c_vp, c_vp, c_vp, c_vp,
                                                 c_vp, c_vp, c_vp, c_vp]),
    'dz_prioritized_sample_gather': (c_int, [ctypes.POINTER(PrioSampleArgs), c_int, c_vp, c_vp,
                                             c_vp, ctypes.POINTER(FieldDesc), c_int, c_vp,
                                             c_vp, c_vp, c_vp, c_vp, c_vp]),
    'dz_prioritized_update': (c_int, [c_vp, c_i64, c_i64, c_i64, c_i64, c_vp,
                                      c_vp, c_int, c_f64, c_int, c_vp, c_vp,
                                      c_vp]),
    'dz_adamw_bind': (c_int, [c_vp, c_int, c_vp, c_vp]),
    'dz_adamw_step': (c_int, [ctypes.POINTER(AdamWArgs), c_vp]),
    'dz_adamw_moments': (c_int, [c_vp, c_vp, c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c_vp]),
    'dz_linear_workspace': (c_int, [ctypes.POINTER(LinearArgs), c_int, ctypes.POINTER(c_i64)]),
    'dz_linear': (c_int, [ctypes.POINTER(LinearArgs), c_vp]),
    'dz_linear_backward': (c_int, [ctypes.POINTER(LinearArgs), c_vp]),
    'dz_policy_loss_workspace': (c_int, [c_int, c_i64, c_i64, ctypes.POINTER(c_i64)]),
    'dz_policy_loss': (c_int, [ctypes.POINTER(PolicyLossArgs), c_vp]),
    'dz_prioritized_add': (c_int, [c_vp, c_i64, c_i64, c_i64, c_int, c_f64,
                                   c_vp, c_f64, c_vp, c_vp]),
}


class HipLibraryError(RuntimeError):
  pass


_lib = None


def load():
  """Loads the library once; raises HipLibraryError if it is unusable."""
  global _lib
  if _lib is not None:
    return _lib
  if not os.path.exists(LIB_PATH):
    raise HipLibraryError(
        'libdqnzoo_hip.so is not built (%s). Run `python -m dqn_zoo_amd.build` '
        '(hipcc, --offload-arch=gfx950). There is no CPU fallback.' % LIB_PATH)
  # PyTorch-ROCm bundles its own libamdhip64.so; it must be mapped BEFORE this
  # library so that both resolve to ONE HIP runtime instance (streams and
  # device pointers are shared between them).
  import torch  # noqa: F401  pylint: disable=unused-import,import-outside-toplevel
  try:
    lib = ctypes.CDLL(LIB_PATH)
  except OSError as e:
    raise HipLibraryError('cannot load %s: %s' % (LIB_PATH, e)) from e
  for name, (res, args) in SIGNATURES.items():
    try:
      fn = getattr(lib, name)
    except AttributeError as e:
      raise HipLibraryError('%s does not export %s' % (LIB_PATH, name)) from e
    fn.restype = res
    fn.argtypes = args
  for which, cls in STRUCT_IDS.items():
    if lib.dz_struct_size(which) != ctypes.sizeof(cls):
      raise HipLibraryError(
          'ABI mismatch: struct %s is %d bytes in the library, %d in _lib.py' %
          (cls.__name__, lib.dz_struct_size(which), ctypes.sizeof(cls)))
  _check_single_hip_runtime()
  _lib = lib
  return lib


def _check_single_hip_runtime():
  try:
    with open('/proc/self/maps') as f:
      paths = {line.split()[-1] for line in f if 'libamdhip64' in line}
  except OSError:
    return
  real = {os.path.realpath(p) for p in paths}
  if len(real) > 1:
    raise HipLibraryError(
        'two HIP runtimes are mapped in this process (%s): import torch before '
        'loading libdqnzoo_hip.so' % sorted(real))


def check(code, what):
  """Maps a DZ_ERR_* return code to a Python exception."""
  if code == DZ_OK:
    return
  if code == DZ_ERR_INVALID_ARG:
    raise ValueError('%s: invalid argument' % what)
  if code == DZ_ERR_HIP:
    raise HipLibraryError('%s: HIP error %d' % (what, load().dz_last_hip_error()))
  if code == DZ_ERR_UNSUPPORTED:
    raise NotImplementedError('%s: unsupported configuration' % what)
  raise HipLibraryError('%s: unknown error code %d' % (what, code))


def capture_graph(stream, enqueue):
  """Runs `enqueue()` (calls into this library on `stream`) under hipGraph
  capture and returns the executable graph handle."""
  lib = load()
  if not stream:
    raise RuntimeError('hipGraph capture needs a non-default stream: run under '
                       '`torch.cuda.stream(torch.cuda.Stream())`')
  # (refused -- ValueError -- while the event profiler is on: its marks are
  # event records between the kernels and cannot live inside a graph)
  global _raw_capture
  check(lib.dz_graph_capture_begin(stream), 'dz_graph_capture_begin')
  h = ctypes.c_void_p()
  _raw_capture = True
  try:
    enqueue()
  except BaseException:
    lib.dz_graph_capture_end(stream, 1, ctypes.byref(h))
    raise
  finally:
    _raw_capture = False
  check(lib.dz_graph_capture_end(stream, 0, ctypes.byref(h)), 'dz_graph_capture_end')
  return h


def ptr(t):
  """Device pointer of a torch tensor (or 0 for None)."""
  if t is None:
    return None
  return t.data_ptr()


_dtype_codes = {}


def dtype_code(dtype):
  """DZ_F32 / DZ_BF16 / DZ_F16 of a torch dtype; None for any other."""
  if not _dtype_codes:
    import torch
    _dtype_codes.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16})
  return _dtype_codes.get(dtype)


def gpu_index(name, t):
  """The device index of a GPU tensor; a TypeError or HipLibraryError for anything else (there
  is no CPU path)."""
  import torch
  if not isinstance(t, torch.Tensor):
    raise TypeError('%s must be a tensor, got %s' % (name, type(t).__name__))
  if not t.is_cuda:
    raise HipLibraryError('%s is on %s: the operators run on an AMD GPU; no CPU fallback' %
                          (name, t.device))
  return t.get_device()


# set while `capture_graph` records: torch's allocator does not know of such a capture, and would
# hand memory that the graph uses to somebody else
_raw_capture = False


def scratch(nbytes, device, workspace):
  """An operator's workspace: the caller's `workspace` (a contiguous uint8 tensor, checked) or a
  block of torch's allocator on the current stream."""
  import torch
  if workspace is None:
    if _raw_capture:
      raise RuntimeError('inside capture_graph the operators need the caller\'s workspace= and '
                         'output buffers: they must live as long as the graph')
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)
  if gpu_index('workspace', workspace) != device.index:
    raise ValueError('workspace is on another device')
  if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
    raise TypeError('workspace must be a contiguous uint8 tensor')
  if workspace.numel() < nbytes or workspace.data_ptr() % 16:
    raise ValueError('workspace needs %d bytes, 16-byte aligned; got %d' % (nbytes, workspace.numel()))
  return workspace


def new_output(shape, dtype, device):
  """torch.empty, refused inside capture_graph (see `scratch`)."""
  import torch
  if _raw_capture:
    raise RuntimeError('inside capture_graph the operators need the caller\'s workspace= and '
                       'output buffers: they must live as long as the graph')
  return torch.empty(shape, dtype=dtype, device=device)


def new_like(t, shape):
  """`new_output` of t's type and device (half the host's time of a torch.empty with keywords)."""
  if _raw_capture:
    return new_output(shape, t.dtype, t.device)
  import torch
  return torch.empty_like(t) if t.shape == shape and t.is_contiguous() else t.new_empty(shape)


def span(t):
  """(first, last + 1) byte of a tensor, whatever lies between its rows."""
  start = t.data_ptr()
  if t.is_contiguous():
    return start, start + t.numel() * t.element_size()
  return start, start + t.element_size() * (1 + sum((s - 1) * d for s, d in zip(t.shape, t.stride())))


class _NoGuard:

  def __enter__(self):
    return self

  def __exit__(self, *exc):
    return False


_no_guard = _NoGuard()


def device_guard(index):
  """Makes `index` the current device for a `with` block (free if it already is): launches go to
  the tensors' device, whichever is current."""
  import torch
  if torch.cuda.current_device() == index:
    return _no_guard
  return torch.cuda.device(index)


def current_stream_ptr():
  import torch
  return torch.cuda.current_stream().cuda_stream


# torch.cuda.current_stream() builds a Stream object through three Python layers
# (~4 us; the agent loop asked for it 3-4 times per frame).  The raw handle of torch's
# CURRENT stream comes from one C call; Stream objects (needed by Event.record) are
# cached per raw handle.
_stream_objects = {}


def _device_index(device):
  import torch
  idx = getattr(device, 'index', device)
  return torch.cuda.current_device() if idx is None else idx


def stream_ptr(device=None):
  """hipStream_t of torch's current stream on `device`, as an integer."""
  import torch
  raw = getattr(torch._C, '_cuda_getCurrentRawStream', None)
  if raw is None:
    return torch.cuda.current_stream(device).cuda_stream
  return raw(_device_index(device))


def current_stream(device=None):
  """torch's current stream on `device` as a (cached) torch.cuda.Stream object."""
  import torch
  idx = _device_index(device)
  key = (idx, stream_ptr(idx))
  s = _stream_objects.get(key)
  if s is None:
    s = torch.cuda.current_stream(idx)
    _stream_objects[key] = s
  return s
