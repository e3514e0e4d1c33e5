"""ctypes declarations of the C ABI (include/nuka_b200.h).  The native library is mandatory: there is no
Python or CPU fallback for the step."""
import ctypes
import os

from . import _build

OK, INVALID_ARG, NULL_HANDLE, CUDA_ERROR, FILE_NOT_FOUND, PARSE_ERROR, OUT_OF_MEMORY, NOT_SUPPORTED, INTERNAL = 0, 1, 2, 3, 4, 5, 6, 7, 100


class DeviceDesc(ctypes.Structure):
    _fields_ = [("gpu_index", ctypes.c_uint32), ("cuda_stream", ctypes.c_void_p), ("backend_selection_layer_enabled", ctypes.c_uint8)]


class WorldDesc(ctypes.Structure):
    _fields_ = [
        ("scene_path", ctypes.c_char_p), ("env_count", ctypes.c_uint32), ("fixed_dt", ctypes.c_float),
        ("determinism", ctypes.c_uint8), ("control_mode", ctypes.c_uint8), ("osc_task_link", ctypes.c_uint32),
        ("terrain_step_height", ctypes.c_float), ("terrain_step_width", ctypes.c_float), ("terrain_platform_width", ctypes.c_float),
        ("terrain_grid_width", ctypes.c_float), ("terrain_grid_height_max", ctypes.c_float),
        ("instance_count", ctypes.c_uint32), ("instance_spacing", ctypes.c_float), ("contact_family", ctypes.c_uint32),
        ("heightfield_terrain_type", ctypes.c_uint32), ("heightfield_nrow", ctypes.c_uint32), ("heightfield_ncol", ctypes.c_uint32),
        ("heightfield_cell", ctypes.c_float), ("heightfield_image_path", ctypes.c_char_p),
        ("heightfield_radius_x", ctypes.c_float), ("heightfield_radius_y", ctypes.c_float),
        ("heightfield_elevation_z", ctypes.c_float), ("heightfield_base_z", ctypes.c_float),
        ("gravity_x", ctypes.c_float), ("gravity_y", ctypes.c_float), ("gravity_z", ctypes.c_float),
        ("curric_levels", ctypes.c_uint32), ("curric_types", ctypes.c_uint32), ("terrain_feature_cell", ctypes.c_float),
        ("solver_vel_iters", ctypes.c_uint32), ("solver_pos_iters", ctypes.c_uint32), ("solver_contact_margin", ctypes.c_float),
        ("solver_max_pairs", ctypes.c_uint32), ("solver_baumgarte_max_velocity", ctypes.c_float), ("cloth_integrator", ctypes.c_uint32),
        ("ogc_contact_capacity", ctypes.c_uint32), ("solver_overlap_recovery_velocity", ctypes.c_float),
        ("solver_substeps", ctypes.c_uint32), ("contact_detection_substeps", ctypes.c_uint32),
    ]


class BufferView(ctypes.Structure):
    _fields_ = [("device_ptr", ctypes.c_void_p), ("element_count", ctypes.c_size_t), ("element_stride_bytes", ctypes.c_uint32), ("dtype", ctypes.c_uint8)]


class WorldInfo(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("env_count", "links_per_env", "bodies_per_env", "dofs_per_env", "contact_slots_per_env",
                                                "shared_bytes_per_env", "warps_per_block")] + [("fixed_dt", ctypes.c_float)]


class ObservationDesc(ctypes.Structure):
    _fields_ = [("command", ctypes.c_void_p), ("command_stride", ctypes.c_uint32), ("last_action", ctypes.c_void_p),
                ("default_position", ctypes.c_void_p), ("joint_order", ctypes.c_void_p), ("reward", ctypes.c_void_p),
                ("lin_vel_scale", ctypes.c_float), ("ang_vel_scale", ctypes.c_float), ("dof_pos_scale", ctypes.c_float),
                ("dof_vel_scale", ctypes.c_float), ("command_scale", ctypes.c_float * 3), ("clip", ctypes.c_float),
                ("row_stride", ctypes.c_uint32)]


class EpisodeDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("actions", "last_action", "default_position", "joint_order", "default_targets", "command",
                                               "episode_steps", "reward", "terminated", "truncated", "done", "done_mask")] + \
               [(n, ctypes.c_float) for n in ("action_scale", "action_clip", "termination_height", "min_up")] + [("max_episode_length", ctypes.c_int32)]


class CookOptions(ctypes.Structure):
    _fields_ = [("dt", ctypes.c_float), ("velocity_iterations", ctypes.c_uint32), ("position_iterations", ctypes.c_uint32),
                ("default_kp", ctypes.c_float), ("default_kd", ctypes.c_float), ("add_default_ground", ctypes.c_uint32),
                ("ground_height", ctypes.c_float), ("ground_mu", ctypes.c_float), ("self_collision", ctypes.c_uint32),
                ("scene_filters", ctypes.c_uint32), ("max_contacts", ctypes.c_uint32), ("max_points", ctypes.c_uint32)]


class EpisodesDesc(ctypes.Structure):
    _fields_ = [("first", ctypes.c_void_p), ("end", ctypes.c_void_p), ("link", ctypes.c_void_p), ("tail", ctypes.c_void_p), ("tokens", ctypes.c_int64), ("rows", ctypes.c_int64), ("length", ctypes.c_int64)]


class RecurrenceDesc(ctypes.Structure):
    _fields_ = [("plan", ctypes.POINTER(EpisodesDesc)), ("dtype", ctypes.c_uint32), ("channels", ctypes.c_int64), ("x", ctypes.c_void_p), ("gate", ctypes.c_void_p),
                ("x_stride", ctypes.c_int64), ("gate_stride", ctypes.c_int64), ("initial", ctypes.c_void_p), ("h", ctypes.c_void_p), ("state", ctypes.c_void_p),
                ("dh", ctypes.c_void_p), ("dstate", ctypes.c_void_p), ("dx", ctypes.c_void_p), ("dgate", ctypes.c_void_p), ("dinitial", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class ConvolutionDesc(ctypes.Structure):
    _fields_ = [("plan", ctypes.POINTER(EpisodesDesc)), ("dtype", ctypes.c_uint32), ("silu", ctypes.c_uint32), ("channels", ctypes.c_int64), ("width", ctypes.c_int64),
                ("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("initial", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("state", ctypes.c_void_p), ("dy", ctypes.c_void_p), ("dstate", ctypes.c_void_p), ("dx", ctypes.c_void_p), ("dinitial", ctypes.c_void_p),
                ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class ConvolutionStepDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("silu", ctypes.c_uint32), ("envs", ctypes.c_int64), ("channels", ctypes.c_int64), ("width", ctypes.c_int64), ("x", ctypes.c_void_p),
                ("x_stride", ctypes.c_int64), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("fresh", ctypes.c_void_p), ("state", ctypes.c_void_p), ("y", ctypes.c_void_p)]


class ScanDesc(ctypes.Structure):
    _fields_ = [("plan", ctypes.POINTER(EpisodesDesc)), ("dtype", ctypes.c_uint32), ("channels", ctypes.c_int64), ("states", ctypes.c_int64), ("x", ctypes.c_void_p),
                ("delta", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("b", ctypes.c_void_p), ("c", ctypes.c_void_p), ("x_stride", ctypes.c_int64),
                ("delta_stride", ctypes.c_int64), ("gate_stride", ctypes.c_int64), ("b_stride", ctypes.c_int64), ("c_stride", ctypes.c_int64), ("decay", ctypes.c_void_p),
                ("skip", ctypes.c_void_p), ("delta_bias", ctypes.c_void_p), ("initial", ctypes.c_void_p), ("y", ctypes.c_void_p), ("state", ctypes.c_void_p),
                ("kept", ctypes.c_void_p), ("kept_bytes", ctypes.c_uint64), ("dy", ctypes.c_void_p), ("dstate", ctypes.c_void_p), ("dx", ctypes.c_void_p),
                ("ddelta", ctypes.c_void_p), ("dgate", ctypes.c_void_p), ("db", ctypes.c_void_p), ("dc", ctypes.c_void_p), ("ddecay", ctypes.c_void_p), ("dskip", ctypes.c_void_p),
                ("ddelta_bias", ctypes.c_void_p), ("dinitial", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class ScanStepDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("envs", ctypes.c_int64), ("channels", ctypes.c_int64), ("states", ctypes.c_int64), ("x", ctypes.c_void_p), ("delta", ctypes.c_void_p),
                ("gate", ctypes.c_void_p), ("b", ctypes.c_void_p), ("c", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("delta_stride", ctypes.c_int64),
                ("gate_stride", ctypes.c_int64), ("b_stride", ctypes.c_int64), ("c_stride", ctypes.c_int64), ("decay", ctypes.c_void_p), ("skip", ctypes.c_void_p),
                ("delta_bias", ctypes.c_void_p), ("fresh", ctypes.c_void_p), ("state", ctypes.c_void_p), ("y", ctypes.c_void_p)]


EXACT_ANGLES = 0x80000000                # added to HeadsDesc.interleaved


class HeadsDesc(ctypes.Structure):
    _fields_ = [("first", ctypes.c_void_p), ("positions", ctypes.c_void_p), ("frequencies", ctypes.c_void_p), ("dtype", ctypes.c_uint32), ("interleaved", ctypes.c_uint32),
                ("tokens", ctypes.c_int64), ("heads_q", ctypes.c_int64), ("heads_k", ctypes.c_int64), ("dim", ctypes.c_int64), ("turned", ctypes.c_int64),
                ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64), ("k_stride", ctypes.c_int64),
                ("k_head_stride", ctypes.c_int64), ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p), ("eps", ctypes.c_float),
                ("q_out", ctypes.c_void_p), ("k_out", ctypes.c_void_p), ("dq_out", ctypes.c_void_p), ("dk_out", ctypes.c_void_p), ("dq", ctypes.c_void_p), ("dk", ctypes.c_void_p),
                ("dq_weight", ctypes.c_void_p), ("dk_weight", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


class AttentionDesc(ctypes.Structure):
    _fields_ = [("plan", ctypes.POINTER(EpisodesDesc)), ("dtype", ctypes.c_uint32), ("heads_q", ctypes.c_int64), ("heads_k", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("window", ctypes.c_int64), ("scale", ctypes.c_float), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64), ("k_stride", ctypes.c_int64), ("k_head_stride", ctypes.c_int64),
                ("v_stride", ctypes.c_int64), ("v_head_stride", ctypes.c_int64), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("dout", ctypes.c_void_p),
                ("delta", ctypes.c_void_p), ("dq", ctypes.c_void_p), ("dk", ctypes.c_void_p), ("dv", ctypes.c_void_p)]


class HistoryDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_uint32), ("envs", ctypes.c_int64), ("capacity", ctypes.c_int64), ("heads_q", ctypes.c_int64), ("heads_k", ctypes.c_int64), ("dim", ctypes.c_int64),
                ("scale", ctypes.c_float), ("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("q_head_stride", ctypes.c_int64),
                ("k_stride", ctypes.c_int64), ("k_head_stride", ctypes.c_int64), ("v_stride", ctypes.c_int64), ("v_head_stride", ctypes.c_int64), ("keys", ctypes.c_void_p),
                ("values", ctypes.c_void_p), ("position", ctypes.c_void_p), ("out", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64)]


EXPORTS = [
    "nuka_get_version", "nuka_result_message", "nuka_last_error_message", "nuka_device_create", "nuka_device_destroy",
    "nuka_world_create_from_scene", "nuka_world_destroy", "nuka_world_step", "nuka_world_step_n", "nuka_world_set_execution_mode",
    "nuka_world_set_gravity_z", "nuka_world_set_velocity_iterations", "nuka_world_get_velocity_iterations", "nuka_world_synchronize",
    "nuka_world_reset", "nuka_world_reset_envs", "nuka_world_forward_kinematics", "nuka_world_get_stream", "nuka_world_record_event",
    "nuka_world_get_buffer_view", "nuka_world_upload_field", "nuka_world_download_field", "nuka_world_create_from_template",
    "nuka_b200_world_info", "nuka_b200_world_run_stage", "nuka_b200_world_launch_count", "nuka_b200_world_reset_envs_static", "nuka_b200_world_download_host", "nuka_b200_host_release",
    "nuka_b200_world_pack_observations", "nuka_b200_observation_desc_defaults", "nuka_b200_world_reset_envs_masked", "nuka_b200_world_episode_step",
    "nuka_b200_world_set_contact_readout", "nuka_b200_world_set_broadphase", "nuka_b200_template_check", "nuka_b200_cook_options_defaults", "nuka_b200_scene_cook", "nuka_world_checkpoint_capture", "nuka_world_checkpoint_restore", "nuka_checkpoint_destroy",
    "nuka_checkpoint_write", "nuka_world_checkpoint_read", "nuka_checkpoint_byte_size", "nuka_checkpoint_equal", "nuka_world_state_hash",
    "nuka_world_get_dof_name", "nuka_b200_episodes_from_offsets", "nuka_b200_episodes_from_done", "nuka_b200_recurrence_workspace", "nuka_b200_recurrence",
    "nuka_b200_recurrence_backward", "nuka_b200_recurrence_step", "nuka_b200_heads_workspace", "nuka_b200_heads", "nuka_b200_heads_backward",
    "nuka_b200_attention_pitch", "nuka_b200_attention", "nuka_b200_attention_backward",
    "nuka_b200_history_workspace", "nuka_b200_history", "nuka_b200_history_advance",
    "nuka_b200_convolution_workspace", "nuka_b200_convolution", "nuka_b200_convolution_backward", "nuka_b200_convolution_step",
    "nuka_b200_attention_sinks", "nuka_b200_attention_sinks_workspace", "nuka_b200_attention_sinks_backward", "nuka_b200_history_sinks", "nuka_b200_scan_kept", "nuka_b200_scan_workspace", "nuka_b200_scan", "nuka_b200_scan_backward", "nuka_b200_scan_step",
]

_LIB = None


def lib():
    """Loads libnuka_b200.so (building it first when the sources are newer)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    path = os.environ.get("NUKA_B200_LIBRARY") or _build.LIB_PATH       # the variable selects an alternative build of the library
    if not os.path.exists(path):
        path = _build.build_native()
    L = ctypes.CDLL(path)
    vp, u32, sz = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_size_t
    L.nuka_result_message.restype = ctypes.c_char_p
    L.nuka_result_message.argtypes = [ctypes.c_int]
    L.nuka_last_error_message.restype = ctypes.c_char_p
    L.nuka_device_create.argtypes = [ctypes.POINTER(DeviceDesc), ctypes.POINTER(vp)]
    L.nuka_device_destroy.argtypes = [vp]
    L.nuka_device_destroy.restype = None
    L.nuka_world_create_from_scene.argtypes = [vp, ctypes.POINTER(WorldDesc), ctypes.POINTER(vp)]
    L.nuka_world_create_from_template.argtypes = [vp, ctypes.POINTER(WorldDesc), ctypes.c_char_p, sz, ctypes.POINTER(vp)]
    L.nuka_world_destroy.argtypes = [vp]
    L.nuka_world_destroy.restype = None
    L.nuka_world_step.argtypes = [vp]
    L.nuka_world_step_n.argtypes = [vp, u32]
    L.nuka_world_set_execution_mode.argtypes = [vp, ctypes.c_int]
    L.nuka_world_set_gravity_z.argtypes = [vp, ctypes.c_float]
    L.nuka_world_set_velocity_iterations.argtypes = [vp, u32]
    L.nuka_world_get_velocity_iterations.argtypes = [vp, ctypes.POINTER(u32)]
    L.nuka_world_synchronize.argtypes = [vp]
    L.nuka_world_reset.argtypes = [vp]
    L.nuka_world_reset_envs.argtypes = [vp, ctypes.POINTER(u32), u32]
    L.nuka_b200_world_reset_envs_static.argtypes = [vp, ctypes.POINTER(u32), u32]
    L.nuka_b200_world_pack_observations.argtypes = [vp, ctypes.POINTER(ObservationDesc), vp, sz, ctypes.POINTER(u32)]
    L.nuka_b200_observation_desc_defaults.argtypes = [ctypes.POINTER(ObservationDesc)]
    L.nuka_b200_observation_desc_defaults.restype = None
    L.nuka_b200_world_reset_envs_masked.argtypes = [vp, vp]
    L.nuka_b200_world_episode_step.argtypes = [vp, ctypes.POINTER(EpisodeDesc), ctypes.POINTER(ObservationDesc), u32, vp, vp, sz]
    L.nuka_b200_cook_options_defaults.argtypes = [ctypes.POINTER(CookOptions)]
    L.nuka_b200_cook_options_defaults.restype = None
    L.nuka_b200_scene_cook.argtypes = [ctypes.c_char_p, sz, ctypes.POINTER(CookOptions), vp, sz, ctypes.POINTER(sz)]
    L.nuka_b200_world_set_contact_readout.argtypes = [vp, u32]
    L.nuka_b200_world_set_broadphase.argtypes = [vp, u32]
    L.nuka_world_forward_kinematics.argtypes = [vp]
    L.nuka_world_get_stream.argtypes = [vp, ctypes.POINTER(vp)]
    L.nuka_world_record_event.argtypes = [vp, vp]
    L.nuka_world_get_buffer_view.argtypes = [vp, ctypes.c_int, ctypes.POINTER(BufferView)]
    L.nuka_world_get_dof_name.argtypes = [vp, ctypes.c_uint32, ctypes.c_char_p, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)]
    L.nuka_world_upload_field.argtypes = [vp, ctypes.c_int, vp, sz, sz]
    L.nuka_world_download_field.argtypes = [vp, ctypes.c_int, vp, sz, sz]
    L.nuka_b200_world_download_host.argtypes = [vp, ctypes.c_int, ctypes.POINTER(vp), ctypes.POINTER(sz)]
    L.nuka_b200_host_release.argtypes = [vp]
    L.nuka_b200_host_release.restype = None
    L.nuka_b200_world_info.argtypes = [vp, ctypes.POINTER(WorldInfo)]
    L.nuka_b200_world_run_stage.argtypes = [vp, u32]
    L.nuka_b200_world_launch_count.argtypes = [vp, ctypes.POINTER(ctypes.c_uint64)]
    L.nuka_world_checkpoint_capture.argtypes = [vp, ctypes.POINTER(vp)]
    L.nuka_world_checkpoint_restore.argtypes = [vp, vp]
    L.nuka_checkpoint_destroy.argtypes = [vp]
    L.nuka_checkpoint_destroy.restype = None
    L.nuka_checkpoint_write.argtypes = [vp, ctypes.c_char_p]
    L.nuka_world_checkpoint_read.argtypes = [vp, ctypes.c_char_p, ctypes.POINTER(vp)]
    L.nuka_checkpoint_byte_size.argtypes = [vp, ctypes.POINTER(ctypes.c_uint64)]
    L.nuka_checkpoint_equal.argtypes = [vp, vp, ctypes.POINTER(u32)]
    L.nuka_world_state_hash.argtypes = [vp, ctypes.POINTER(ctypes.c_uint64)]
    i64, u64 = ctypes.c_int64, ctypes.c_uint64
    L.nuka_b200_episodes_from_offsets.argtypes = [ctypes.POINTER(EpisodesDesc), vp, vp]
    L.nuka_b200_episodes_from_done.argtypes = [ctypes.POINTER(EpisodesDesc), vp, vp]
    L.nuka_b200_recurrence_workspace.argtypes = [ctypes.POINTER(EpisodesDesc), i64]
    L.nuka_b200_recurrence_workspace.restype = u64
    L.nuka_b200_recurrence.argtypes = [ctypes.POINTER(RecurrenceDesc), vp]
    L.nuka_b200_recurrence_backward.argtypes = [ctypes.POINTER(RecurrenceDesc), vp]
    L.nuka_b200_recurrence_step.argtypes = [u32, i64, i64, vp, i64, vp, i64, vp, vp, vp, vp]
    L.nuka_b200_heads_workspace.argtypes = [i64, i64]
    L.nuka_b200_heads_workspace.restype = u64
    L.nuka_b200_heads.argtypes = [ctypes.POINTER(HeadsDesc), vp]
    L.nuka_b200_heads_backward.argtypes = [ctypes.POINTER(HeadsDesc), vp]
    L.nuka_b200_attention_pitch.argtypes = [i64]
    L.nuka_b200_attention_pitch.restype = i64
    L.nuka_b200_attention.argtypes = [ctypes.POINTER(AttentionDesc), vp]
    L.nuka_b200_attention_backward.argtypes = [ctypes.POINTER(AttentionDesc), vp]
    L.nuka_b200_history_workspace.argtypes = [ctypes.POINTER(HistoryDesc)]
    L.nuka_b200_history_workspace.restype = u64
    L.nuka_b200_history.argtypes = [ctypes.POINTER(HistoryDesc), vp]
    L.nuka_b200_history_advance.argtypes = [vp, vp, i64, vp]
    L.nuka_b200_convolution_workspace.argtypes = [ctypes.POINTER(EpisodesDesc), i64, i64]
    L.nuka_b200_convolution_workspace.restype = u64
    L.nuka_b200_convolution.argtypes = [ctypes.POINTER(ConvolutionDesc), vp]
    L.nuka_b200_convolution_backward.argtypes = [ctypes.POINTER(ConvolutionDesc), vp]
    L.nuka_b200_convolution_step.argtypes = [ctypes.POINTER(ConvolutionStepDesc), vp]
    L.nuka_b200_attention_sinks.argtypes = [ctypes.POINTER(AttentionDesc), i64, vp]
    L.nuka_b200_attention_sinks_workspace.argtypes = [ctypes.POINTER(AttentionDesc), i64]
    L.nuka_b200_attention_sinks_workspace.restype = u64
    L.nuka_b200_attention_sinks_backward.argtypes = [ctypes.POINTER(AttentionDesc), i64, vp, u64, vp]
    L.nuka_b200_history_sinks.argtypes = [ctypes.POINTER(HistoryDesc), i64, vp]
    L.nuka_b200_scan_kept.argtypes = [ctypes.POINTER(EpisodesDesc), i64, i64]
    L.nuka_b200_scan_kept.restype = u64
    L.nuka_b200_scan_workspace.argtypes = [ctypes.POINTER(EpisodesDesc), i64, i64, u32]
    L.nuka_b200_scan_workspace.restype = u64
    L.nuka_b200_scan.argtypes = [ctypes.POINTER(ScanDesc), vp]
    L.nuka_b200_scan_backward.argtypes = [ctypes.POINTER(ScanDesc), vp]
    L.nuka_b200_scan_step.argtypes = [ctypes.POINTER(ScanStepDesc), vp]
    _LIB = L
    return L
