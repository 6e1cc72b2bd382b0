"""Model family: cell-embedding + convolutional frame head, streaming LSTM + causal-attention action model."""
from .frame_head import CellEmbed, DownsampleBlock, FrameHead
from .blocks import AttentionBlock, Embedding, GatedMlp, Mean, MlpBlock, RmsNorm, LayerNorm, Linear, FullMhaAttention, TokenEmbedding
from .attention_decoder import AttentionDecoder, PagedCache, WindowBlock
from .recurrent_decoder import RecurrentBlock, RecurrentDecoder
from .streaming_lstm import StreamingLstm
from .action_model import ActionModel
from .fbam import FbamModel, model_dtype, checkpoint_name_map

__all__ = ["AttentionDecoder", "PagedCache", "WindowBlock", "RecurrentDecoder", "RecurrentBlock", "GatedMlp", "TokenEmbedding", "Embedding", "Mean", "CellEmbed", "DownsampleBlock", "FrameHead", "AttentionBlock", "MlpBlock", "RmsNorm", "LayerNorm",
           "Linear", "FullMhaAttention", "StreamingLstm", "ActionModel", "FbamModel", "model_dtype",
           "checkpoint_name_map"]
