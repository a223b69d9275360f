package sampler

// uncompiled: no Go toolchain in the build environment of this file; it is written against
// include/born_sampler.h and the loaders of cgo.go / purego.go.

import (
	"runtime"
	"unsafe"
)

// Beam search and the output head, over device memory (asynchronous on `stream`, nothing is
// allocated per call).  The reference has neither; the head is its Linear layer with the activations
// that its modules probe for (internal/nn/linear.go:78-107, internal/nn/activation.go:7-20).

const (
	MaxBeams   = 16
	MaxStops   = 8
	MaxReorder = 128

	BeamKeepSlots = 1 // the best child of a beam stays in the beam's own row
	BeamEarlyStop = 2 // a group is done as soon as its pool is full

	RowDead = 8 // the row's score is -inf: it has no candidates

	ActNone    = 0
	ActReLU    = 1
	ActSigmoid = 2
	ActTanh    = 3 // Scale * tanh(y / Scale)
	ActGELU    = 4
	ActSiLU    = 5
)

// BeamArgs is born_beam_args, field for field.
type BeamArgs struct {
	StructSize      uint32
	Memory          uint32
	Groups          int32
	Beams           int32
	Vocab           int32
	LogitsDType     int32
	LogitsRowStride int64
	Logits          uintptr
	Mask            uintptr
	MaskRowStride   int64
	History         uintptr
	HistoryLen      uintptr
	HistoryStride   int32
	Flags           uint32
	Params          RowParams
	Scores          uintptr
	StopIDs         [MaxStops]int32
	NStop           int32
	Step            int32
	OutParent       uintptr
	OutToken        uintptr
	OutScore        uintptr
	OutStatus       uintptr
	OutEndParent    uintptr
	OutEndToken     uintptr
	OutEndScore     uintptr
	PoolScore       uintptr
	PoolStep        uintptr
	PoolParent      uintptr
	PoolToken       uintptr
	Done            uintptr
	LengthPenalty   float32
	Reserved        int32
}

// ReorderArgs is born_reorder_args; Buffers is the address of a host array of device addresses.
type ReorderArgs struct {
	StructSize    uint32
	Memory        uint32
	Groups        int32
	Beams         int32
	NBuffers      int32
	Planes        int32
	Buffers       uintptr
	RowStride     int64
	PlaneStride   int64
	PositionBytes int64
	Positions     int64
	Parents       uintptr
	Lens          uintptr
}

// SequencesArgs is born_sequences_args.
type SequencesArgs struct {
	StructSize  uint32
	Memory      uint32
	Groups      int32
	Beams       int32
	Steps       int32
	Hypotheses  int32
	TableStride int64
	Tokens      uintptr
	Parents     uintptr
	EndStep     uintptr
	EndParent   uintptr
	EndToken    uintptr
	OutTokens   uintptr
	OutStride   int64
	OutLens     uintptr
	Pad         int32
	Reserved    int32
}

// LinearArgs is born_linear_args.
type LinearArgs struct {
	StructSize        uint32
	Memory            uint32
	Rows              int32
	Hidden            int32
	Features          int32
	OutDType          int32
	Activation        int32
	Scale             float32
	X                 uintptr
	Weight            uintptr
	Bias              uintptr
	Residual          uintptr
	Out               uintptr
	XRowStride        int64
	WeightRowStride   int64
	ResidualRowStride int64
	OutRowStride      int64
}

// BeamStep picks the beams that go on: one step of a search over groups*beams rows of logits.
func (s *CUDASampler) BeamStep(a *BeamArgs, stream uintptr) error {
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	return check(s.b.beamStep(s.h, a, stream), s.msg)
}

// BeamNext is BeamStep over the device-resident history (HistoryCreate, a row per beam): a.History
// must be 0; the kernel moves the histories after the beams and appends their tokens.
func (s *CUDASampler) BeamNext(a *BeamArgs, stream uintptr) error {
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	return check(s.b.beamNext(s.h, a, stream), s.msg)
}

// BeamPoolReset empties the pool that `a` points to.
func (s *CUDASampler) BeamPoolReset(a *BeamArgs, stream uintptr) error {
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	return check(s.b.beamPoolReset(s.h, a, stream), s.msg)
}

// BeamReorder moves the rows of per-beam states (device addresses, all of one layout) after the
// beams, in place.
func (s *CUDASampler) BeamReorder(buffers []uintptr, a *ReorderArgs, stream uintptr) error {
	if len(buffers) == 0 {
		panic("sampler: BeamReorder: no buffers")
	}
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	var pin runtime.Pinner // the args struct holds a Go pointer: pinned for the duration of the call
	defer pin.Unpin()
	pin.Pin(&buffers[0])
	a.NBuffers, a.Buffers = int32(len(buffers)), uintptr(unsafe.Pointer(&buffers[0]))
	return check(s.b.beamReorder(s.h, a, stream), s.msg)
}

// BeamSequences reads the token sequences of hypotheses out of the tables that the steps wrote.
func (s *CUDASampler) BeamSequences(a *SequencesArgs, stream uintptr) error {
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	return check(s.b.beamSequences(s.h, a, stream), s.msg)
}

// Linear is the output head: act(x weight^T + bias) + residual, bfloat16 operands.
func (s *CUDASampler) Linear(a *LinearArgs, stream uintptr) error {
	a.StructSize, a.Memory = uint32(unsafe.Sizeof(*a)), MemDevice
	return check(s.b.linear(s.h, a, stream), s.msg)
}
