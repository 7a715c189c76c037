"""Model zoo + ``build_model`` factory (the reference's TODO "# build_model",
`/root/reference/train_pascal.py:6`)."""
from __future__ import annotations

import torch.nn as nn

from ..ops import convert_group_norm, convert_sync_batchnorm, freeze_batchnorm
from .danet import DANet
from .deeplab import ASPP, Decoder, DeepLabV3Plus
from .fcn import FCN
from .resnet import ResNet
from .xception import AlignedXception

MODEL_NAMES = (
    "fcn_resnet18", "fcn_resnet50", "fcn_resnet101",
    "deeplabv3plus_resnet18", "deeplabv3plus_resnet50", "deeplabv3plus_resnet101",
    "deeplabv3plus_xception65", "danet_resnet50", "danet_resnet101",
)

_ALIASES = {
    "deeplabv3plus_r101": "deeplabv3plus_resnet101",
    "deeplabv3plus_r50": "deeplabv3plus_resnet50",
    "deeplabv3plus_x65": "deeplabv3plus_xception65",
    "deeplabv3plus_xception": "deeplabv3plus_xception65",
    "fcn_r18": "fcn_resnet18",
    "danet": "danet_resnet101",
}


def build_model(name: str = "deeplabv3plus_resnet101", num_classes: int = 21, output_stride: int | None = None,
                sync_bn: bool = False, freeze_bn: bool = False, in_channels: int = 3,
                process_group=None, norm: str = "batch", decoder_attention: bool = False) -> nn.Module:
    """Construct a segmentation network by name.

    ``sync_bn`` / ``freeze_bn`` mirror the knobs of the reference's commented DeepLab constructor
    (`/root/reference/train_pascal.py:85`).  ``norm``: ``'batch'``, or ``'group'`` for group norm in every layer's place
    (statistics of one image: training at a few images per GPU; ResNet backbones).  ``decoder_attention``: DeepLabv3+
    with cross attention from the decoder's positions to the encoder's map (``models.deeplab.DecoderAttention``)."""
    name = _ALIASES.get(name, name)
    head, _, backbone = name.partition("_")
    if norm not in ("batch", "group"):
        raise ValueError(f"norm must be 'batch' or 'group', got {norm!r}")
    if norm == "group" and (sync_bn or freeze_bn):
        raise ValueError("sync_bn / freeze_bn are about batch statistics: group norm has none")
    if norm == "group" and backbone.startswith("xception"):
        raise NotImplementedError("Xception's middle flow is stored wider than it is: its zero channels would enter a group's "
                                  "statistics (norm='group' takes the ResNet backbones)")
    if decoder_attention and head != "deeplabv3plus":
        raise ValueError("decoder_attention: DeepLabv3+ models")
    if head == "fcn":
        model = FCN(num_classes, backbone, output_stride or 32, in_channels)
    elif head == "deeplabv3plus":
        model = DeepLabV3Plus(num_classes, backbone, output_stride or 16, in_channels, decoder_attention)
    elif head == "danet":
        model = DANet(num_classes, backbone, in_channels, output_stride or 8)
    else:
        raise ValueError(f"unknown model '{name}'; choose from {MODEL_NAMES}")
    if norm == "group":
        convert_group_norm(model)
    if sync_bn:
        convert_sync_batchnorm(model, process_group)
    if freeze_bn:
        freeze_batchnorm(model)
    return model


__all__ = ["build_model", "MODEL_NAMES", "DeepLabV3Plus", "FCN", "DANet", "ResNet", "AlignedXception",
           "ASPP", "Decoder"]
