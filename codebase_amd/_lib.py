"""ctypes binding of libmarlhip.so (include/marlhip.h).  No fallbacks: if the library is not
built, importing this module raises; if a call fails, MarlHipError carries marlhip_last_error()."""
import ctypes
import os
from ctypes import POINTER, c_char_p, c_double, c_float, c_int32, c_int64, c_uint8, c_uint32, c_uint64, c_void_p

_HERE = os.path.dirname(os.path.abspath(__file__))
# MARLHIP_LIB: an experiment build of the same library (scripts/build_variants.py); the product path is the in-tree default
LIB_PATH = os.environ.get("MARLHIP_LIB") or os.path.join(_HERE, "csrc", "libmarlhip.so")


class MarlHipError(RuntimeError):
    pass


class LbfConfig(ctypes.Structure):
    _fields_ = [
        ("n_envs", c_int32), ("n_agents", c_int32), ("n_food", c_int32), ("rows", c_int32), ("cols", c_int32),
        ("sight", c_int32), ("max_episode_steps", c_int32), ("time_limit", c_int32), ("force_coop", c_int32),
        ("min_player_level", c_int32), ("max_player_level", c_int32), ("min_food_level", c_int32),
        ("max_food_level", c_int32), ("normalize_reward", c_int32), ("cooperative", c_int32),
        ("penalty", c_double), ("seed", c_uint64), ("reward_stats", c_void_p), ("observe_id", c_int32),
    ]


class RwareConfig(ctypes.Structure):
    _fields_ = [
        ("n_envs", c_int32), ("n_agents", c_int32), ("shelf_rows", c_int32), ("shelf_columns", c_int32),
        ("column_height", c_int32), ("request_queue_size", c_int32), ("max_steps", c_int32),
        ("max_inactivity_steps", c_int32), ("time_limit", c_int32), ("reward_type", c_int32), ("cooperative", c_int32),
        ("observe_id", c_int32), ("seed", c_uint64), ("reward_stats", c_void_p),
    ]


class LbfBuffers(ctypes.Structure):
    _fields_ = [("state", c_void_p), ("episode", c_void_p), ("ep_return", c_void_p), ("ep_length", c_void_p)]


class NetShape(ctypes.Structure):
    _fields_ = [("n_agents", c_int32), ("obs_dim", c_int32), ("hidden", c_int32), ("n_actions", c_int32),
                ("n_networks", c_int32), ("net_of", c_int32 * 16), ("n_hidden", c_int32)]


class ReplayShape(ctypes.Structure):
    _fields_ = [("capacity", c_int32), ("n_agents", c_int32), ("obs_dim", c_int32), ("max_len", c_int32)]


class ReplayBuffers(ctypes.Structure):
    _fields_ = [("obs", c_void_p), ("act", c_void_p), ("rew", c_void_p), ("done", c_void_p), ("filled", c_void_p)]


class BatchStruct(ctypes.Structure):
    _fields_ = [("obss", c_void_p), ("actions", c_void_p), ("rewards", c_void_p), ("dones", c_void_p),
                ("filled", c_void_p), ("max_len", c_int32), ("batch", c_int32),
                ("obs_agent_stride", c_int64), ("obs_row_stride", c_int64), ("act_agent_stride", c_int64),
                ("act_row_stride", c_int64), ("action_mask", c_void_p)]


class QmixMixer(ctypes.Structure):
    _fields_ = [("mixer", c_void_p), ("target_mixer", c_void_p), ("mixer_grad", c_void_p), ("embed_dim", c_int32),
                ("hypernet_layers", c_int32), ("hypernet_embed", c_int32), ("ret_stats", c_void_p), ("l1_fp16", c_int32)]


class AcConfig(ctypes.Structure):
    _fields_ = [("n_steps", c_int32), ("entropy_coef", c_float), ("value_loss_coef", c_float), ("ppo_clip", c_float),
                ("gamma", c_double), ("ret_mean", c_void_p), ("ret_var", c_void_p), ("ret_count", c_void_p),
                ("centralised_critic", c_int32), ("side_stream", c_void_p),
                ("ret_exchange", c_void_p), ("ret_exchange_ctx", c_void_p), ("ret_moments", c_void_p),
                ("critic_n_networks", c_int32), ("critic_net_of", c_int32 * 16), ("actor_forward_kept", c_int32),
                ("defer_critic_backward", c_int32), ("critic_n_hidden", c_int32)]


class RetStatsStruct(ctypes.Structure):
    _fields_ = [("mean", c_void_p), ("var", c_void_p), ("count", c_void_p), ("columns", c_int32),
                ("exchange", c_void_p), ("exchange_ctx", c_void_p), ("moments", c_void_p)]


class SsmShape(ctypes.Structure):
    _fields_ = [("n_agents", c_int32), ("steps", c_int32), ("batch", c_int32), ("channels", c_int32), ("state", c_int32), ("groups", c_int32),
                ("dtype", c_int32), ("n_networks", c_int32), ("net_of", c_int32 * 16)]


class SsmSeq(ctypes.Structure):
    _fields_ = [("data", c_void_p), ("agent_stride", c_int64), ("step_stride", c_int64), ("row_stride", c_int64)]


class SsmConvArgs(ctypes.Structure):
    _fields_ = [("x", SsmSeq), ("dy", SsmSeq), ("weight", c_void_p), ("bias", c_void_p), ("silu", c_int32), ("state", c_void_p),
                ("reset", c_void_p), ("lengths", c_void_p), ("y", c_void_p), ("state_out", c_void_p), ("dstate_out", c_void_p), ("dx", c_void_p),
                ("dstate", c_void_p), ("dweight", c_void_p), ("dbias", c_void_p)]


class SsmScanArgs(ctypes.Structure):
    _fields_ = [("x", SsmSeq), ("delta", SsmSeq), ("B", SsmSeq), ("C", SsmSeq), ("z", SsmSeq), ("dy", SsmSeq),
                ("A", c_void_p), ("D", c_void_p), ("delta_bias", c_void_p), ("softplus", c_int32), ("h_in", c_void_p), ("reset", c_void_p),
                ("lengths", c_void_p), ("y", c_void_p), ("h_out", c_void_p), ("record", c_void_p), ("dh_out", c_void_p), ("dx", c_void_p),
                ("ddelta", c_void_p), ("dB", c_void_p), ("dC", c_void_p), ("dz", c_void_p), ("dA", c_void_p), ("dD", c_void_p),
                ("ddelta_bias", c_void_p), ("dh_in", c_void_p)]


class TensorStruct(ctypes.Structure):
    _fields_ = [("data", c_void_p), ("out", c_void_p), ("n", c_int64), ("dtype", c_int32)]


class IdqnLearner(ctypes.Structure):
    _fields_ = [("net", NetShape), ("rs", ReplayShape), ("rb", ReplayBuffers),
                ("params", c_void_p), ("target", c_void_p), ("exp_avg", c_void_p), ("exp_avg_sq", c_void_p),
                ("grad", c_void_p), ("loss", c_void_p), ("scratch", c_void_p), ("gnorm", c_void_p),
                ("workspace", c_void_p), ("workspace_bytes", c_int64),
                ("obss", c_void_p), ("actions", c_void_p), ("rewards", c_void_p), ("dones", c_void_p), ("filled", c_void_p),
                ("idx", c_void_p), ("batch", c_int32), ("double_q", c_int32), ("mode", c_int32), ("materialise_batch", c_int32),
                ("gamma", c_float), ("max_norm", c_float), ("lr", c_double), ("beta1", c_double), ("beta2", c_double),
                ("eps", c_double), ("target_update_interval_or_tau", c_double)]


class QmixLearner(ctypes.Structure):
    _fields_ = [("base", IdqnLearner), ("mixer", QmixMixer), ("mixer_rw", c_void_p), ("target_mixer_rw", c_void_p),
                ("mixer_exp_avg", c_void_p), ("mixer_exp_avg_sq", c_void_p), ("mixer_scratch", c_void_p), ("optimizer", c_int32)]


# every symbol include/marlhip.h declares: name -> (restype, argtypes)
PROTOTYPES = {
    "marlhip_version": (c_int32, []),
    "marlhip_last_error": (c_char_p, []),
    "marlhip_device_available": (c_int32, []),
    "marlhip_lbf_state_stride": (c_int32, [POINTER(LbfConfig)]),
    "marlhip_lbf_obs_dim": (c_int32, [POINTER(LbfConfig)]),
    "marlhip_lbf_reset": (c_int32, [POINTER(LbfConfig), POINTER(LbfBuffers), c_void_p, c_void_p, c_void_p]),
    "marlhip_lbf_observe": (c_int32, [POINTER(LbfConfig), POINTER(LbfBuffers), c_void_p, c_void_p]),
    "marlhip_lbf_step": (c_int32, [POINTER(LbfConfig), POINTER(LbfBuffers), c_void_p, c_void_p, c_void_p, c_void_p,
                                   c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p]),
    "marlhip_rware_state_stride": (c_int32, [POINTER(RwareConfig)]),
    "marlhip_rware_obs_dim": (c_int32, [POINTER(RwareConfig)]),
    "marlhip_rware_grid": (c_int32, [POINTER(RwareConfig), POINTER(c_int32), POINTER(c_int32), POINTER(c_int32)]),
    "marlhip_rware_reset": (c_int32, [POINTER(RwareConfig), POINTER(LbfBuffers), c_void_p, c_void_p, c_void_p]),
    "marlhip_rware_observe": (c_int32, [POINTER(RwareConfig), POINTER(LbfBuffers), c_void_p, c_void_p]),
    "marlhip_rware_step": (c_int32, [POINTER(RwareConfig), POINTER(LbfBuffers), c_void_p, c_void_p, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p]),
    "marlhip_rware_idqn_collect": (c_int32, [POINTER(RwareConfig), POINTER(NetShape), c_void_p, c_float, c_uint32,
                                             POINTER(ReplayShape), POINTER(ReplayBuffers), c_int32, c_int32, c_int32, c_int32,
                                             c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_rware_ac_collect": (c_int32, [POINTER(RwareConfig), POINTER(NetShape), c_void_p, c_uint32, c_int32, c_int32, c_void_p,
                                           c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                           c_void_p]),
    "marlhip_gru_nparams": (c_int32, [POINTER(NetShape)]),
    "marlhip_gru_forward_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_gru_record_floats": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_gru_forward": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p,
                                      c_void_p, c_int64, c_void_p]),
    "marlhip_gru_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_gru_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32, c_int32, c_void_p,
                                        c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_gru_loss_grad_std": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32, POINTER(RetStatsStruct),
                                            c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_gru_qmix_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_gru_qmix_workspace_bytes_mx": (c_int64, [POINTER(NetShape), POINTER(QmixMixer), c_int32, c_int32]),
    "marlhip_gru_qmix_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(QmixMixer), POINTER(BatchStruct), c_float, c_int32,
                                             c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_wide_qmix_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(QmixMixer), POINTER(BatchStruct), c_float, c_int32,
                                             c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_wide_qmix_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_wide_qmix_workspace_bytes_mx": (c_int64, [POINTER(NetShape), POINTER(QmixMixer), c_int32, c_int32]),
    "marlhip_gru_ac_critic_nparams": (c_int32, [POINTER(NetShape), c_int32]),
    "marlhip_gru_ac_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32]),
    "marlhip_gru_ac_workspace_bytes_lc": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32, c_int32]),
    "marlhip_gru_a2c_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                            c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_gru_ppo_prepare": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                          c_void_p, c_int64, c_void_p]),
    "marlhip_gru_ppo_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                            c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_gru_ac_forward": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, c_int64, c_int64, c_int32, c_int32, c_void_p,
                                         c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_sample_from_logits": (c_int32, [c_int32, c_int32, c_int32, c_void_p, c_uint64, c_void_p, c_int32, c_void_p, c_void_p]),
    "marlhip_act_from_q": (c_int32, [c_int32, c_int32, c_int32, c_void_p, c_float, c_uint64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_net_nparams": (c_int32, [POINTER(NetShape)]),
    "marlhip_wide_nparams": (c_int32, [POINTER(NetShape), c_int32]),
    "marlhip_wide_forward_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32]),
    "marlhip_wide_forward": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, c_int64, c_int64, c_int32, c_void_p, c_void_p, c_int64,
                                       c_void_p]),
    "marlhip_wide_dqn_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_wide_dqn_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32, c_int32, c_void_p,
                                             c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_wide_dqn_loss_grad_std": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32,
                                                 POINTER(RetStatsStruct), c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_act": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_int32, c_float, c_void_p, c_void_p, c_uint64,
                                  c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_replay_init_episode": (c_int32, [POINTER(ReplayShape), POINTER(ReplayBuffers), c_void_p, c_void_p, c_void_p,
                                              c_int32, c_void_p]),
    "marlhip_replay_add_step": (c_int32, [POINTER(ReplayShape), POINTER(ReplayBuffers), c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                          c_void_p, c_void_p, c_void_p, c_int32, c_void_p]),
    "marlhip_replay_add": (c_int32, [POINTER(ReplayShape), POINTER(ReplayBuffers), c_void_p, c_void_p, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_int32, c_void_p]),
    "marlhip_replay_sample": (c_int32, [POINTER(ReplayShape), POINTER(ReplayBuffers), c_void_p, c_int32, c_int32, c_uint64,
                                        c_uint32, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_dqn_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32,
                                        c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_loss_grad_replay": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(ReplayShape),
                                               POINTER(ReplayBuffers), c_void_p, c_int32, c_int32, c_uint64, c_uint32, c_void_p,
                                               c_float, c_int32, c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_loss_grad_std": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32, c_int32,
                                            POINTER(RetStatsStruct), c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_loss_grad_std_replay": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(ReplayShape),
                                                   POINTER(ReplayBuffers), c_void_p, c_int32, c_int32, c_uint64, c_uint32, c_void_p,
                                                   c_float, c_int32, c_int32, POINTER(RetStatsStruct), c_void_p, c_int64, c_void_p, c_void_p,
                                                   c_void_p]),
    "marlhip_qmix_nparams": (c_int32, [POINTER(NetShape), c_int32, c_int32, c_int32]),
    "marlhip_qmix_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32]),
    "marlhip_qmix_workspace_bytes_mx": (c_int64, [POINTER(NetShape), POINTER(QmixMixer), c_int32, c_int32]),
    "marlhip_qmix_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(QmixMixer), POINTER(BatchStruct), c_float,
                                         c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_qmix_loss_grad_replay": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(QmixMixer), POINTER(ReplayShape),
                                                POINTER(ReplayBuffers), c_void_p, c_int32, c_int32, c_uint64, c_uint32, c_void_p,
                                                c_float, c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_ac_critic_nparams": (c_int32, [POINTER(NetShape), c_int32]),
    "marlhip_ac_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32]),
    "marlhip_ac_workspace_bytes_lc": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32, c_int32]),
    "marlhip_ac_forward_rows": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, c_int64, c_int64, c_int32, c_void_p,
                                          c_void_p, c_int64, c_void_p]),
    "marlhip_a2c_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                        c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_mixed_ac_workspace_bytes": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32]),
    "marlhip_mixed_ac_workspace_bytes_lc": (c_int64, [POINTER(NetShape), c_int32, c_int32, c_int32, c_int32]),
    "marlhip_mixed_a2c_loss_grad": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                              c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_mixed_ppo_prepare": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                            c_void_p, c_int64, c_void_p]),
    "marlhip_mixed_ppo_loss_grad": (c_int32, [POINTER(NetShape), c_int32, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                              c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_ppo_prepare": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                      c_void_p, c_int64, c_void_p]),
    "marlhip_ppo_loss_grad": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), POINTER(AcConfig),
                                        c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "marlhip_dqn_clip_adam": (c_int32, [c_int64, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_double,
                                        c_double, c_double, c_double, c_float, c_float, c_int32, c_float, c_void_p,
                                        c_void_p, c_void_p]),
    "marlhip_dqn_clip_step": (c_int32, [c_int32, c_int64, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_double, c_float, c_float,
                                        c_int32, c_float, c_void_p, c_void_p, c_void_p]),
    "marlhip_ac_collect": (c_int32, [POINTER(LbfConfig), POINTER(NetShape), c_void_p, c_uint32, c_int32, c_int32, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_stream_create_cu_share": (c_int32, [c_int32, c_int32, POINTER(c_void_p)]),
    "marlhip_stream_destroy": (c_int32, [c_void_p]),
    "marlhip_ac_collect_keep": (c_int32, [POINTER(LbfConfig), POINTER(NetShape), c_void_p, c_uint32, c_int32, c_int32, c_void_p,
                                          c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_void_p,
                                          c_int64, c_void_p]),
    "marlhip_rware_ac_collect_keep": (c_int32, [POINTER(RwareConfig), POINTER(NetShape), c_void_p, c_uint32, c_int32, c_int32, c_void_p,
                                                c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32,
                                                c_void_p, c_int64, c_void_p]),
    "marlhip_ac_store_step": (c_int32, [c_int32, c_int32, c_int32, c_int32, c_int32] + [c_void_p] * 16 + [c_int32, c_void_p, c_void_p, c_void_p]),
    "marlhip_ac_collect_later_episodes": (c_int32, [c_void_p, POINTER(NetShape), c_void_p, c_uint32, c_int32, c_void_p, c_void_p, c_int32, c_int32,
                                                    c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_rware_ac_collect_later_episodes": (c_int32, [c_void_p, POINTER(NetShape), c_void_p, c_uint32, c_int32, c_void_p, c_void_p, c_int32,
                                                          c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_idqn_update_n": (c_int32, [POINTER(IdqnLearner), c_int32, c_int32, c_uint64, c_uint32, POINTER(c_int64),
                                        POINTER(c_int64), POINTER(c_int64), c_void_p]),
    "marlhip_update_plan": (c_int32, [POINTER(ReplayShape), POINTER(ReplayBuffers), c_int32, c_int32, c_int32, c_uint64, c_uint32, c_int32, c_void_p,
                                      c_int64, c_void_p, c_void_p, c_void_p]),
    "marlhip_idqn_update_n_dist": (c_int32, [POINTER(IdqnLearner), c_int32, c_int32, c_uint64, c_uint32, POINTER(c_int64),
                                             POINTER(c_int64), POINTER(c_int64), c_void_p, c_void_p, c_int32, c_void_p]),
    "marlhip_qmix_update_n": (c_int32, [POINTER(QmixLearner), c_int32, c_int32, c_uint64, c_uint32, POINTER(c_int64), POINTER(c_int64),
                                        POINTER(c_int64), c_void_p, c_void_p, c_int32, c_void_p]),
    "marlhip_p2p_handle_bytes": (c_int32, []),
    "marlhip_p2p_create": (c_int32, [c_int32, c_int32, c_int64, POINTER(c_void_p), c_void_p]),
    "marlhip_p2p_connect": (c_int32, [c_void_p, c_void_p]),
    "marlhip_p2p_allreduce": (c_int32, [c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_p2p_allreduce_wave64": (c_int32, [c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_p2p_status": (c_int32, [c_void_p]),
    "marlhip_p2p_destroy": (c_int32, [c_void_p]),
    "marlhip_dqn_loss_grad_split16": (c_int32, [POINTER(NetShape), c_void_p, c_void_p, POINTER(BatchStruct), c_float, c_int32, c_void_p, c_int64,
                                                c_void_p, c_void_p, c_void_p]),
    "marlhip_idqn_update_n_split16": (c_int32, [POINTER(IdqnLearner), c_int32, c_int32, c_uint64, c_uint32, POINTER(c_int64),
                                                POINTER(c_int64), POINTER(c_int64), c_void_p]),
    # (shape and argument structs as packed bytes or byref of the classes above; marlhip_tensor arrays by address: hip.py)
    "marlhip_ssm_conv": (c_int32, [c_void_p, c_void_p, c_void_p]),
    "marlhip_ssm_conv_grad_workspace_bytes": (c_int64, [c_void_p]),
    "marlhip_ssm_conv_grad": (c_int32, [c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_ssm_scan_record_floats": (c_int64, [c_void_p]),
    "marlhip_ssm_scan_workspace_bytes": (c_int64, [c_void_p]),
    "marlhip_ssm_scan": (c_int32, [c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_ssm_scan_grad_workspace_bytes": (c_int64, [c_void_p]),
    "marlhip_ssm_scan_grad": (c_int32, [c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_tensors_apart": (c_int32, [c_void_p, c_int32]),
    "marlhip_grad_norm_workspace_bytes": (c_int64, [c_void_p, c_int32]),
    "marlhip_grad_norm": (c_int32, [c_void_p, c_int32, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_clip_grad_norm": (c_int32, [c_void_p, c_int32, c_float, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_timing_enable": (c_int32, [c_int32]),
    "marlhip_timing_read": (c_int32, [c_int32, POINTER(c_int64), POINTER(c_double)]),
    "marlhip_idqn_collect": (c_int32, [POINTER(LbfConfig), POINTER(NetShape), c_void_p, c_float, c_uint32,
                                       POINTER(ReplayShape), POINTER(ReplayBuffers), c_int32, c_int32, c_int32, c_int32,
                                       c_void_p, c_void_p, c_void_p, c_int64, c_void_p]),
    "marlhip_forward_workspace_bytes": (c_int64, [POINTER(NetShape)]),
}

if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} is missing: build the HIP library first (python -m codebase_amd.build). "
        "There is no CPU fallback for the marlhip hot path.")

lib = ctypes.CDLL(LIB_PATH)
for _name, (_res, _args) in PROTOTYPES.items():
    _fn = getattr(lib, _name)  # AttributeError here = header and library out of sync
    _fn.restype = _res
    _fn.argtypes = _args


def last_error():
    return lib.marlhip_last_error().decode()


def check(rc, what=""):
    if rc < 0:
        raise MarlHipError(f"{what}: {last_error()}" if what else last_error())
    return rc
