"""MI355X-native Graph U-Net forward path: HIP kernels behind the reference's layer API.

Layout mirrors the reference modules that lie on the path:
    layers.hybrid_gnn   GeoQuadrantGCN, GraphDownsamplingBlock, GraphUpsamplingBlock,
                        GraphUpsampling2x2, graph_pooling_2x2, remove_duplicate_edges
    layers.graph_ops    get_sender_receiver
    data.data_utils     sample_quadrant_subgraphs, DIR_TO_EDGE, QUADRANT_IDS
    models.graph_unet   GraphUNet
Beside them, without a counterpart in the reference:
    layers.expert_ops   expert_plan, expert_dispatch, expert_combine and their gradients
    layers.mxfp4        Mxfp4Tensor, mxfp4_quantize, mxfp4_dequantize, mxfp4_dense, mxfp4_expert_dense, Mxfp4Dense
"""
from . import _lib                                   # raises if libgunet_hip.so is missing
from ._lib import GunetError, LIB_PATH, set_matmul_mode, get_matmul_mode, set_kernel_choice
from . import plan
from . import layers
from .layers import hybrid_gnn, graph_ops, expert_ops, mxfp4
from .layers.expert_ops import (ExpertPlan, expert_plan, expert_dispatch, expert_dispatch_grad, expert_combine,
                                expert_combine_grad)
from .layers.mxfp4 import Mxfp4Tensor, Mxfp4Dense, mxfp4_quantize, mxfp4_dequantize, mxfp4_dense, mxfp4_expert_dense
from .data import data_utils
from .models import graph_unet, base_model
from . import evaluation, submission
from .capture import CapturedForward
from .models.graph_unet import GraphUNet

__all__ = ['GunetError', 'LIB_PATH', 'set_matmul_mode', 'get_matmul_mode', 'plan', 'layers', 'hybrid_gnn', 'graph_ops', 'data_utils',
           'graph_unet', 'GraphUNet', 'expert_ops', 'mxfp4', 'ExpertPlan', 'expert_plan', 'expert_dispatch',
           'expert_dispatch_grad', 'expert_combine', 'expert_combine_grad', 'Mxfp4Tensor', 'Mxfp4Dense', 'mxfp4_quantize',
           'mxfp4_dequantize', 'mxfp4_dense', 'mxfp4_expert_dense']
